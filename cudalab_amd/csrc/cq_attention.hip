// Attention over the quantized paged key/value cache (gfx950).
//
//   s_j = scale * (q . kcode_j) * kscale_j, p = softmax(s) over what the row
//   sees, out_d = sum_j p_j * vscale_j * vcode_jd
//
// One pass over the keys with the running maximum and sum: a wave keeps
// (m, l, o) = (max s, sum e^(s - m), sum e^(s - m) v) and rescales l and o
// when m grows; partial triples of disjoint key ranges join the same way.

#include "cq_attn.h"
#include "cq_elem.h"

namespace cq {
namespace {

constexpr int kBlock = 256;
constexpr float kNegInf = -__builtin_inff();

// One workgroup per row (sequence, new token, query head); its four waves
// take every fourth key, a lane E dims.
template <class T, int BITS, int D>
__global__ __launch_bounds__(kBlock) void row_kernel(cq_kv_cache_t c, cq_attention_t a) {
    constexpr int E = D / 64;
    constexpr int R = BITS == 8 ? D : D / 2;
    __shared__ float part[4][D + 2];
    const int hq = blockIdx.x % a.q_heads;
    const int64_t bt = blockIdx.x / a.q_heads;
    const int b = (int)(bt / a.tokens), t = (int)(bt % a.tokens);
    const int h = hq / (a.q_heads / c.heads);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const T* q = static_cast<const T*>(a.q) + b * a.q_batch_stride + t * a.q_token_stride +
                 hq * a.q_head_stride;
    float qf[E], o[E] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) qf[e] = (float)q[lane * E + e];
    int count = a.tokens;
    if (a.counts != nullptr) count = min(count, a.counts[b]);
    float m = kNegInf, l = 0.f;
    auto walk = [&](const int32_t* table, int64_t cols, int64_t n) {
        n = min(n, cols * c.page_size);
        for (int64_t j = wave; j < n; j += 4) {
            const int64_t page = page_in(table[j / c.page_size], c.pages);
            if (page < 0) continue;
            const int64_t ph = page * c.heads + h;
            const int in = (int)(j % c.page_size);
            const uint8_t* kr = static_cast<const uint8_t*>(c.k) + (ph * c.page_size + in) * R;
            const uint8_t* vr = static_cast<const uint8_t*>(c.v) +
                                (ph * (c.page_size / 16) + in / 16) * R * 16 + in % 16;
            auto code = [&](const uint8_t* p, int step, int d) {
                if (BITS == 8) return (float)(int8_t)p[d * step];
                return (float)((int)((uint32_t)p[(d / 2) * step] << (28 - 4 * (d & 1))) >> 28);
            };
            const float* sc = c.scales + ph * 2 * c.page_size + in;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s = __builtin_fmaf(qf[e], code(kr, 1, lane * E + e), s);
            s = lanes_sum<64>(s) * (sc[0] * a.softmax_scale);
            const float top = fmaxf(m, s);
            const float ref = top == kNegInf ? 0.f : top;
            const float keep = __expf(m - ref), p = __expf(s - ref);
            m = top;
            l = l * keep + p;
            const float pv = p * sc[c.page_size];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = o[e] * keep + pv * code(vr, 16, lane * E + e);
        }
    };
    if (t < count) {
        if (a.prefix_len > 0) walk(a.prefix_table, a.prefix_cols, a.prefix_len);
        walk(a.table + b * a.table_stride, a.table_cols, (int64_t)a.lengths[b] - count + t + 1);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) part[wave][lane * E + e] = o[e];
    if (lane == 0) part[wave][D] = m, part[wave][D + 1] = l;
    __syncthreads();
    float top = kNegInf;
    for (int w = 0; w < 4; ++w) top = fmaxf(top, part[w][D]);
    const float ref = top == kNegInf ? 0.f : top;
    for (int d = threadIdx.x; d < D; d += kBlock) {
        float sum = 0.f, out = 0.f;
        for (int w = 0; w < 4; ++w) {
            const float keep = __expf(part[w][D] - ref);
            sum += part[w][D + 1] * keep;
            out += part[w][d] * keep;
        }
        static_cast<T*>(a.out)[(int64_t)blockIdx.x * D + d] = (T)(sum == 0.f ? 0.f : out / sum);
    }
}

}  // namespace

int64_t attention_workspace(const cq_kv_cache_t&, const cq_attention_t&) { return 0; }

hipError_t launch_attention(const cq_kv_cache_t& c, const cq_attention_t& a,
                            hipStream_t stream) {
    const int64_t grid = (int64_t)a.batch * a.tokens * a.q_heads;
    if (grid > kMaxGrid) return hipErrorInvalidValue;
    auto go = [&](auto* kernel) {
        kernel<<<dim3((unsigned)grid), dim3(kBlock), 0, stream>>>(c, a);
        return hipGetLastError();
    };
    auto typed = [&](auto elem) {
        using T = decltype(elem);
        if (c.bits == 8)
            return c.head_dim == 64 ? go(&row_kernel<T, 8, 64>)
                   : c.head_dim == 128 ? go(&row_kernel<T, 8, 128>) : go(&row_kernel<T, 8, 256>);
        return c.head_dim == 64 ? go(&row_kernel<T, 4, 64>)
               : c.head_dim == 128 ? go(&row_kernel<T, 4, 128>) : go(&row_kernel<T, 4, 256>);
    };
    return a.dtype == CQ_DTYPE_F16 ? typed(_Float16{}) : typed(__bf16{});
}

}  // namespace cq
