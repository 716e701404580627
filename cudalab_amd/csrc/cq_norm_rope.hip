// Per-head RMS norm of queries and keys with the position rotation in the
// same pass (gfx950).
//
//   n = x * (1 / sqrt(mean(x^2) + eps)) * weight
//   a' = a cos - b sin, b' = b cos + a sin  for the pairs the rotation turns
//
// in FP32, rounded once.  Rounding the normed value to the element type before
// the rotation, as a chain of separate calls would, is left out: one rounding
// is closer to the formula.
//
// Bound by memory: each element is read and written once, past the caches, and
// the tables' rows of a token serve all its heads; by the launch at one token.
// LANES lanes take a head, C elements of each end of its pairs each: the lane
// that holds a holds its b too, so the rotation needs no exchange, and the only
// one is the sum of squares.

#include "cq_attn.h"
#include "cq_elem.h"

namespace cq {
namespace {

constexpr int kBlock = 256;

__device__ __forceinline__ float load_weight(const void* p, int dtype, int i) {
    if (dtype == CQ_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
    if (dtype == CQ_DTYPE_BF16) return (float)static_cast<const __bf16*>(p)[i];
    return static_cast<const float*>(p)[i];
}

// C weights from i, a multiple of C (all at once where `wide`).
template <int C>
__device__ __forceinline__ void load_weights(const void* p, int dtype, int i, bool wide,
                                             float (&w)[C]) {
    if (wide && dtype != CQ_DTYPE_F32) {
        const Vec<uint16_t, C> v =
            *reinterpret_cast<const Vec<uint16_t, C>*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const uint16_t bits = v[j];      // (a cast of v[j] itself takes v[0])
            w[j] = dtype == CQ_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, bits)
                                         : __uint_as_float((uint32_t)bits << 16);
        }
    } else {
#pragma unroll
        for (int j = 0; j < C; ++j) w[j] = load_weight(p, dtype, i + j);
    }
}

// Row of the cos/sin tables of a token, or -1 for a position outside them.
__device__ __forceinline__ int64_t table_row(const cq_norm_rope_t& a, int64_t token) {
    const int64_t p = a.positions_64 ? static_cast<const int64_t*>(a.positions)[token]
                                     : static_cast<const int32_t*>(a.positions)[token];
    return p >= 0 && p < a.table_rows ? p : -1;
}

// One head's place: heads count through q's, then k's.
template <class T>
struct Head {
    const T* src;
    T* dst;
    bool is_q;
    __device__ __forceinline__ Head(const cq_norm_rope_t& a, int64_t token, int h) {
        is_q = h < a.q_heads;
        if (is_q) {
            src = static_cast<const T*>(a.q) + token * a.q_token_stride + h * a.q_head_stride;
            dst = static_cast<T*>(a.q_out) + token * a.q_out_token_stride +
                  h * a.q_out_head_stride;
        } else {
            h -= a.q_heads;
            src = static_cast<const T*>(a.k) + token * a.k_token_stride + h * a.k_head_stride;
            dst = static_cast<T*>(a.k_out) + token * a.k_out_token_stride +
                  h * a.k_out_head_stride;
        }
    }
};

// Vector kernel: head_dim and rot_dim multiples of 2 C, head_dim <= 2 C * LANES,
// rows aligned to C elements, tables to 16 bytes.  A group of LANES lanes takes
// heads part, part + parts, ... of one token, BATCH loads of each end in
// flight; lane l holds elements e0..e0+C-1 and e1..e1+C-1, in the half style
// the two ends of pairs Cl..Cl+C-1, else 2 C neighbours.  `first` is the
// launch's first workgroup.
template <class T, bool PAIRS, int C, int LANES, int BATCH>
__global__ __launch_bounds__(kBlock) void norm_rope_kernel(cq_norm_rope_t a, uint32_t parts,
                                                           uint32_t iters, bool wide,
                                                           uint32_t first) {
    using V = Vec<T, C>;
    const int lane = threadIdx.x % LANES;
    const uint32_t group = (first + blockIdx.x) * (kBlock / LANES) + threadIdx.x / LANES;
    const int heads = a.q_heads + a.k_heads;
    // groups past the last token repeat it and store nothing
    const bool live = group / parts < a.tokens;
    const int64_t token = live ? group / parts : a.tokens - 1;
    const uint32_t part = group % parts;
    const bool active = 2 * C * lane < a.head_dim;
    const bool turn = a.cos_table != nullptr && 2 * C * lane < a.rot_dim;
    const bool halves = turn && !PAIRS;
    const int e0 = !active ? 0 : halves ? C * lane : 2 * C * lane;
    const int e1 = !active ? C : halves ? a.rot_dim / 2 + C * lane : 2 * C * lane + C;

    V x0[BATCH], x1[BATCH];
    auto load = [&](uint32_t it) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int h = (int)min(part + (it + u) * parts, (uint32_t)heads - 1);
            const Head<T> head(a, token, h);
            x0[u] = __builtin_nontemporal_load(reinterpret_cast<const V*>(head.src + e0));
            x1[u] = __builtin_nontemporal_load(reinterpret_cast<const V*>(head.src + e1));
        }
    };
    load(0);
    float w[2][2][C];           // of q and k, at e0 and e1
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const void* p = i == 0 ? a.q_weight : a.k_weight;
#pragma unroll
        for (int j = 0; j < C; ++j) w[i][0][j] = w[i][1][j] = 1.f;
        if (p != nullptr) {
            load_weights(p, a.weight_dtype, e0, wide, w[i][0]);
            load_weights(p, a.weight_dtype, e1, wide, w[i][1]);
        }
    }
    float c[C], s[C];
#pragma unroll
    for (int i = 0; i < C; ++i) c[i] = 1.f, s[i] = 0.f;
    if (turn) {
        const int64_t row = table_row(a, token);
        if (row >= 0) {
            const int64_t at = row * (a.rot_dim / 2) + C * lane;
#pragma unroll
            for (int i = 0; i < C; i += 4) {
                const Vec<float, 4> cv =
                    *reinterpret_cast<const Vec<float, 4>*>(a.cos_table + at + i);
                const Vec<float, 4> sv =
                    *reinterpret_cast<const Vec<float, 4>*>(a.sin_table + at + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) c[i + j] = cv[j], s[i + j] = sv[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i) c[i] = s[i] = __builtin_nanf("");
        }
    }
    const bool norm = a.q_weight != nullptr || a.k_weight != nullptr;
    const float mean = 1.f / (float)a.head_dim;

    for (uint32_t it = 0;;) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const uint32_t h = part + (it + u) * parts;
            const Head<T> head(a, token, (int)min(h, (uint32_t)heads - 1));
            float f[2 * C];
#pragma unroll
            for (int i = 0; i < C; ++i) f[i] = (float)x0[u][i], f[C + i] = (float)x1[u][i];
            if (norm) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * C; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
                ss = lanes_sum<LANES>(active ? ss : 0.f);
                const bool has = head.is_q ? a.q_weight != nullptr : a.k_weight != nullptr;
                const float r = has ? 1.f / sqrtf(ss * mean + a.eps) : 1.f;
#pragma unroll
                for (int i = 0; i < 2 * C; ++i)
                    f[i] = f[i] * r * (head.is_q ? w[0][i / C][i % C] : w[1][i / C][i % C]);
            }
            if (turn) {
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    float& p = f[PAIRS ? 2 * i : i];
                    float& q = f[PAIRS ? 2 * i + 1 : C + i];
                    const float t = p * c[i] - q * s[i];
                    q = q * c[i] + p * s[i];
                    p = t;
                }
            }
            V y0, y1;
#pragma unroll
            for (int i = 0; i < C; ++i) y0[i] = (T)f[i], y1[i] = (T)f[C + i];
            if (live && active && h < (uint32_t)heads) {
                __builtin_nontemporal_store(y0, reinterpret_cast<V*>(head.dst + e0));
                __builtin_nontemporal_store(y1, reinterpret_cast<V*>(head.dst + e1));
            }
        }
        it += BATCH;
        if (it >= iters) break;
        load(it);
    }
}

// Element kernel (any even dims, any alignment): one wave per head, pairs
// lane, lane + 64, ... held between the sum and the rotation.
constexpr int kMaxPairs = 8;      // head_dim <= 1024

template <class T>
__global__ __launch_bounds__(kBlock) void norm_rope_any_kernel(cq_norm_rope_t a,
                                                               uint32_t first) {
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)(first + blockIdx.x) * (kBlock / 64) + (threadIdx.x >> 6);
    const int heads = a.q_heads + a.k_heads;
    const int64_t token = unit / heads;
    if (token >= a.tokens) return;                 // uniform over the wave
    const Head<T> head(a, token, (int)(unit % heads));
    const void* weight = head.is_q ? a.q_weight : a.k_weight;
    const int half = a.cos_table != nullptr ? a.rot_dim / 2 : 0;
    const int64_t row = half > 0 ? table_row(a, token) : 0;
    float p[kMaxPairs], q[kMaxPairs];
    float ss = 0.f;
    auto places = [&](int pair, int& e0, int& e1) {
        const bool halves = pair < half && !a.interleaved;
        e0 = halves ? pair : 2 * pair;
        e1 = halves ? pair + half : 2 * pair + 1;
    };
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        const int pair = lane + 64 * i;
        p[i] = q[i] = 0.f;
        if (2 * pair < a.head_dim) {
            int e0, e1;
            places(pair, e0, e1);
            p[i] = (float)head.src[e0];
            q[i] = (float)head.src[e1];
            ss = __builtin_fmaf(p[i], p[i], ss);
            ss = __builtin_fmaf(q[i], q[i], ss);
        }
    }
    ss = lanes_sum<64>(ss);
    const float r = weight != nullptr ? 1.f / sqrtf(ss * (1.f / (float)a.head_dim) + a.eps) : 1.f;
#pragma unroll
    for (int i = 0; i < kMaxPairs; ++i) {
        const int pair = lane + 64 * i;
        if (2 * pair >= a.head_dim) continue;
        int e0, e1;
        places(pair, e0, e1);
        float x = p[i], y = q[i];
        if (weight != nullptr) {
            x = x * r * load_weight(weight, a.weight_dtype, e0);
            y = y * r * load_weight(weight, a.weight_dtype, e1);
        }
        if (pair < half) {
            const float c = row >= 0 ? a.cos_table[row * half + pair] : __builtin_nanf("");
            const float s = row >= 0 ? a.sin_table[row * half + pair] : __builtin_nanf("");
            const float t = x * c - y * s;
            y = y * c + x * s;
            x = t;
        }
        head.dst[e0] = (T)x;
        head.dst[e1] = (T)y;
    }
}

bool multiple(int64_t v, int64_t m) { return v % m == 0; }

// Whether the vector kernel may run with C elements at a time: everything it
// reads or writes so starts at a multiple of them.
bool vector_ok(const cq_norm_rope_t& a, int64_t elem, int c) {
    const int64_t bytes = c * elem;
    auto rows_ok = [&](const void* p, int64_t ts, int64_t hs) {
        return multiple((int64_t)(uintptr_t)p, bytes) && multiple(ts * elem, bytes) &&
               multiple(hs * elem, bytes);
    };
    if (a.head_dim % (2 * c) != 0 || a.head_dim > 512) return false;
    if (a.cos_table != nullptr &&
        (a.rot_dim % (2 * c) != 0 || !multiple((int64_t)(uintptr_t)a.cos_table, 16) ||
         !multiple((int64_t)(uintptr_t)a.sin_table, 16)))
        return false;
    if (a.q_heads > 0 && !(rows_ok(a.q, a.q_token_stride, a.q_head_stride) &&
                           rows_ok(a.q_out, a.q_out_token_stride, a.q_out_head_stride)))
        return false;
    return a.k_heads == 0 || (rows_ok(a.k, a.k_token_stride, a.k_head_stride) &&
                              rows_ok(a.k_out, a.k_out_token_stride, a.k_out_head_stride));
}

template <class T, bool PAIRS>
hipError_t launch_typed(const cq_norm_rope_t& a, hipStream_t stream) {
    const int64_t heads = (int64_t)a.q_heads + a.k_heads;
    if (!vector_ok(a, sizeof(T), 4)) {
        const int64_t units = a.tokens * heads, grid = (units + kBlock / 64 - 1) / (kBlock / 64);
        if (grid > kMaxGrid) return hipErrorInvalidValue;
        return launch_parts(grid, [&](dim3 blocks, uint32_t first) {
            norm_rope_any_kernel<T><<<blocks, dim3(kBlock), 0, stream>>>(a, first);
        });
    }
    auto go = [&](auto* kernel, int c, int lanes, int64_t iters) {
        const int64_t per = kBlock / lanes;
        const int64_t parts = (heads + iters - 1) / iters, groups = a.tokens * parts;
        if (groups + per > kMaxGrid) return hipErrorInvalidValue;
        auto weight_wide = [&](const void* p) {
            return a.weight_dtype == CQ_DTYPE_F32 || (uintptr_t)p % (2 * c) == 0;
        };
        const bool wide = weight_wide(a.q_weight) && weight_wide(a.k_weight);
        return launch_parts((groups + per - 1) / per, [&](dim3 blocks, uint32_t first) {
            kernel<<<blocks, dim3(kBlock), 0, stream>>>(a, (uint32_t)parts, (uint32_t)iters, wide,
                                                        first);
        });
    };
    // Pieces of 16 bytes of each end, two heads in flight and weights and tables
    // fetched once for several heads, as long as waves enough are left: by how
    // many there are with one head to a group.  Few: one, in pieces of four
    // elements, which is ahead where a call is hardly more than its launch and
    // level then.  fp16 heads of 128, us with one head to a group in pieces of 8 and
    // 16 bytes, then (from where it matters) with two, four and eight:
    //   72 heads     (9 waves)     3.03 3.31
    //   2304         (288)         3.64 3.87
    //   4000         (500)         3.69 3.93
    //   9216         (1152)        4.62 4.53
    //   20480        (2560)        5.79 5.76
    //   16384        (2048)         -    -   5.9  7.6 11.5
    //   65536       (8192)        14.0 12.9  9.8 11.4 14.2
    //   169696      (21212)       33.9 29.5 23.8 23.1 23.1
    //   524288      (65536)       95.9 83.8 68.2 59.5 57.4
    // (FP32 in pieces of 32 bytes is slower: 262144 heads 65 us, of 16 bytes 58.)
    const int lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : a.head_dim <= 256 ? 32 : 64;
    const bool wide_ok = sizeof(T) == 2 && vector_ok(a, sizeof(T), 8);
    const int64_t waves = a.tokens * heads * (wide_ok ? lanes / 2 : lanes) / 64;
    const int64_t each = waves < 4096 ? 1 : waves <= 8192 ? 2 : waves < 32768 ? 4 : 8;
#define CQ_GO(C, L, B) go(&norm_rope_kernel<T, PAIRS, C, L, B>, C, L, each)
    if constexpr (sizeof(T) == 2) {
        if (wide_ok && each > 1) {
            if (a.head_dim <= 64) return CQ_GO(8, 4, 2);
            if (a.head_dim <= 128) return CQ_GO(8, 8, 2);
            if (a.head_dim <= 256) return CQ_GO(8, 16, 2);
            return CQ_GO(8, 32, 2);
        }
    }
    if (lanes == 8) return each > 1 ? CQ_GO(4, 8, 2) : CQ_GO(4, 8, 1);
    if (lanes == 16) return each > 1 ? CQ_GO(4, 16, 2) : CQ_GO(4, 16, 1);
    if (lanes == 32) return each > 1 ? CQ_GO(4, 32, 2) : CQ_GO(4, 32, 1);
    return each > 1 ? CQ_GO(4, 64, 2) : CQ_GO(4, 64, 1);
#undef CQ_GO
}

}  // namespace

hipError_t launch_norm_rope(const cq_norm_rope_t& a, hipStream_t stream) {
    auto go = [&](auto elem) {
        using T = decltype(elem);
        return a.interleaved ? launch_typed<T, true>(a, stream) : launch_typed<T, false>(a, stream);
    };
    if (a.dtype == CQ_DTYPE_F16) return go(_Float16{});
    if (a.dtype == CQ_DTYPE_BF16) return go(__bf16{});
    return go(float{});
}

}  // namespace cq
