// C entry points of the operators of a step of many tokens (declared in
// include/cdnaqgemv.h): the checks that a safe launch needs.  What lies on the
// device (lengths, offsets, slots) the kernels check themselves.

#include <climits>
#include <cmath>
#include <string>

#include "cq_checks.h"
#include "cq_step.h"

using namespace cq::checks;

namespace {

bool stride_ok(int64_t n) { return n >= 0 && n <= (int64_t)1 << 40; }

int check_append_rows(const cq_kv_cache_t& c, int dtype, int64_t tokens, const int64_t* slots,
                      const void* k, cq::KvStrides ks, const void* v, cq::KvStrides vs) {
    const int st = check_cache(c);
    if (st != CQ_OK) return st;
    if (!known_dtype(dtype)) return invalid("unknown dtype");
    if (tokens < 1 || tokens > INT_MAX) return invalid("tokens must be in [1, 2^31-1]");
    if (k == nullptr || v == nullptr || slots == nullptr) return invalid("null pointer argument");
    const int64_t es = elem_bytes(dtype);
    if (!aligned(k, es) || !aligned(v, es) || !aligned(slots, 8))
        return invalid("a pointer is not aligned to its element size");
    for (int64_t n : {ks.token, ks.head, vs.token, vs.head})
        if (!stride_ok(n)) return invalid("strides must be in [0, 2^40]");
    const CacheSpans cs(c);
    for (const Span& in : {strided(k, {{tokens, ks.token}, {c.heads, ks.head}}, c.head_dim, es),
                           strided(v, {{tokens, vs.token}, {c.heads, vs.head}}, c.head_dim, es),
                           Span(slots, static_cast<U>(tokens) * 8)})
        if (cs.meet(in)) return invalid("an input overlaps the cache");
    if (cs.meet_themselves()) return invalid("the cache's tensors overlap");
    return CQ_OK;
}

constexpr int64_t kMostRows = INT_MAX - 511;      // a tile's rows behind them fit an int

int check_prompt(const cq_prompt_t& a) {
    if (a.batch < 1 || a.batch == INT_MAX) return invalid("batch must be in [1, 2^31-2]");
    if (a.q_tokens < 1 || a.q_tokens > kMostRows || a.k_tokens < 0 || a.k_tokens > kMostRows)
        return invalid("q_tokens must be in [1, 2^31-512], k_tokens in [0, 2^31-512]");
    if (a.k_heads < 1 || a.q_heads < 1 || a.q_heads > 65535 || a.q_heads % a.k_heads != 0)
        return invalid("q_heads must be a multiple of k_heads, at most 65535");
    if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256)
        return invalid("head_dim must be 64, 128 or 256");
    if (a.dtype != CQ_DTYPE_F16 && a.dtype != CQ_DTYPE_BF16)
        return invalid("dtype must be CQ_DTYPE_F16 or CQ_DTYPE_BF16");
    if (std::isnan(a.softmax_scale) || std::isinf(a.softmax_scale))
        return invalid("softmax_scale must be finite");
    if (a.q == nullptr || a.out == nullptr || a.q_offsets == nullptr ||
        (a.k_tokens > 0 && (a.k == nullptr || a.v == nullptr)))
        return invalid("null pointer argument");
    if (!aligned(a.q, 16) || !aligned(a.k, 16) || !aligned(a.v, 16) || !aligned(a.out, 16))
        return invalid("q, k, v and out must be 16-byte aligned");
    if (!aligned(a.q_offsets, 4) || !aligned(a.k_offsets, 4))
        return invalid("the offsets must be 4-byte aligned");
    for (int64_t n : {a.q_token_stride, a.q_head_stride, a.k_token_stride, a.k_head_stride,
                      a.v_token_stride, a.v_head_stride})
        if (!stride_ok(n) || n % 8 != 0) return invalid("strides must be multiples of 8 in [0, 2^40]");
    if (a.k_token_stride > 1 << 24 || a.v_token_stride > 1 << 24)
        return invalid("the token strides of k and v must be at most 2^24");
    const Span out[] = {strided(a.out, {{a.q_tokens, (int64_t)a.q_heads * a.head_dim}},
                                (int64_t)a.q_heads * a.head_dim, 2)};
    const Span in[] = {
        strided(a.q, {{a.q_tokens, a.q_token_stride}, {a.q_heads, a.q_head_stride}}, a.head_dim, 2),
        strided(a.k, {{a.k_tokens, a.k_token_stride}, {a.k_heads, a.k_head_stride}}, a.head_dim, 2),
        strided(a.v, {{a.k_tokens, a.v_token_stride}, {a.k_heads, a.v_head_stride}}, a.head_dim, 2),
        Span(a.q_offsets, (static_cast<U>(a.batch) + 1) * 4),
        Span(a.k_offsets, (static_cast<U>(a.batch) + 1) * 4)};
    if (meet(out, in)) return invalid("out overlaps an input");
    return CQ_OK;
}

constexpr int64_t kMostK = 131071;                // of products of 2^14 a sum in 32 bits

int check_quantize(int dtype, const void* x, int64_t x_stride, int64_t tokens, int64_t k,
                   const int8_t* codes, const float* scales) {
    if (!known_dtype(dtype)) return invalid("unknown dtype");
    if (tokens < 1 || tokens > kMostRows) return invalid("tokens must be in [1, 2^31-512]");
    if (k < 1 || k > INT_MAX) return invalid("k must be in [1, 2^31-1]");
    if (x == nullptr || codes == nullptr || scales == nullptr) return invalid("null pointer argument");
    const int64_t es = elem_bytes(dtype);
    if (!aligned(x, es) || !aligned(scales, 4))
        return invalid("a pointer is not aligned to its element size");
    if (!stride_ok(x_stride)) return invalid("strides must be in [0, 2^40]");
    const Span out[] = {Span(codes, static_cast<U>(tokens) * static_cast<U>(k)),
                        Span(scales, static_cast<U>(tokens) * 4)};
    const Span in[] = {strided(x, {{tokens, x_stride}}, k, es)};
    if (meet(out, in)) return invalid("an output overlaps another operand");
    return CQ_OK;
}

int check_qgemm(const cq_qgemm_t& a, bool launching) {
    if (!known_dtype(a.dtype)) return invalid("unknown dtype");
    if (a.tokens < 1 || a.tokens > kMostRows || a.n < 1 || a.n > kMostRows)
        return invalid("tokens and n must be in [1, 2^31-512]");
    if (a.k < 1 || a.k > kMostK) return invalid("k must be in [1, 131071]");
    if (a.x_stride < a.k || a.x_stride > (int64_t)1 << 40)
        return invalid("x_stride must be in [k, 2^40]");
    if (!launching) return CQ_OK;
    if (a.x == nullptr || a.x_scale == nullptr || a.w == nullptr || a.w_scale == nullptr ||
        a.out == nullptr)
        return invalid("null pointer argument");
    if (!aligned(a.x_scale, 4) || !aligned(a.w_scale, 4) || !aligned(a.out, 16))
        return invalid("out must be 16-byte aligned, the scales 4-byte aligned");
    const int64_t need = cq::qgemm_workspace(a);
    if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || !aligned(a.workspace, 16)))
        return cq::set_error(CQ_ERR_BUFFER_TOO_SMALL,
                             "the call needs " + std::to_string(need) +
                                 " bytes of 16-byte aligned workspace, got " +
                                 std::to_string(a.workspace_bytes));
    const U n = static_cast<U>(a.n), tokens = static_cast<U>(a.tokens);
    const Span out[] = {Span(a.out, tokens * n * static_cast<U>(elem_bytes(a.dtype))),
                        Span(need > 0 ? a.workspace : nullptr, static_cast<U>(need > 0 ? need : 0))};
    const Span in[] = {strided(a.x, {{a.tokens, a.x_stride}}, a.k, 1),
                       Span(a.w, n * static_cast<U>(a.k)), Span(a.x_scale, tokens * 4),
                       Span(a.w_scale, n * 4)};
    if (meet(out, in)) return invalid("out or the workspace overlaps an input");
    return CQ_OK;
}

}  // namespace

extern "C" {

int cq_attention_tree(const cq_kv_cache_t* cache, const cq_attention_t* args,
                      const int64_t* seen, void* stream) {
    return guarded([&]() -> int {
        if (cache == nullptr || args == nullptr || seen == nullptr)
            return invalid("null pointer: cache, args or seen");
        const int st =
            cq::check_attention(*cache, *args, true, cq::attention_tree_workspace);
        if (st != CQ_OK) return st;
        if (!aligned(seen, 8)) return invalid("seen must be 8-byte aligned");
        const cq_attention_t& a = *args;
        const Span bits(seen, static_cast<U>(a.batch) * static_cast<U>(a.tokens) *
                                  static_cast<U>((a.tokens + (int64_t)63) / 64) * 8);
        const Span out(a.out, static_cast<U>(a.batch) * static_cast<U>(a.tokens) *
                                  static_cast<U>(a.q_heads) *
                                  static_cast<U>(cache->head_dim * elem_bytes(a.dtype)));
        const int64_t need = cq::attention_tree_workspace(*cache, a);
        if (overlap(out, bits) ||
            overlap(Span(need > 0 ? a.workspace : nullptr, static_cast<U>(need > 0 ? need : 0)), bits))
            return invalid("out or the workspace overlaps an input");
        return hip_status(cq::launch_attention_tree(*cache, a, seen,
                                                    static_cast<hipStream_t>(stream)),
                          "cq_attention_tree");
    });
}

int64_t cq_attention_tree_workspace(const cq_kv_cache_t* cache, const cq_attention_t* args) {
    return guarded([&]() -> int64_t {
        if (cache == nullptr || args == nullptr) return -invalid("null pointer: cache or args");
        const int st = cq::check_attention(*cache, *args, false, cq::attention_tree_workspace);
        if (st != CQ_OK) return -st;
        return cq::attention_tree_workspace(*cache, *args);
    }, -CQ_ERR_HIP);
}

int cq_quantize_tokens(int dtype, const void* x, int64_t x_stride, int64_t tokens, int64_t k,
                       int8_t* codes, float* scales, void* stream) {
    return guarded([&]() -> int {
        const int st = check_quantize(dtype, x, x_stride, tokens, k, codes, scales);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_quantize_tokens(dtype, x, x_stride, tokens, k, codes, scales,
                                                     static_cast<hipStream_t>(stream)),
                          "cq_quantize_tokens");
    });
}

int cq_qgemm(const cq_qgemm_t* args, void* stream) {
    return guarded([&]() -> int {
        if (args == nullptr) return invalid("null pointer: args");
        const int st = check_qgemm(*args, true);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_qgemm(*args, static_cast<hipStream_t>(stream)), "cq_qgemm");
    });
}

int64_t cq_qgemm_workspace(const cq_qgemm_t* args) {
    return guarded([&]() -> int64_t {
        if (args == nullptr) return -invalid("null pointer: args");
        const int st = check_qgemm(*args, false);
        if (st != CQ_OK) return -st;
        return cq::qgemm_workspace(*args);
    }, -CQ_ERR_HIP);
}

int cq_prompt_attention(const cq_prompt_t* args, void* stream) {
    return guarded([&]() -> int {
        if (args == nullptr) return invalid("null pointer: args");
        const int st = check_prompt(*args);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_prompt(*args, static_cast<hipStream_t>(stream)),
                          "cq_prompt_attention");
    });
}

int cq_place(const cq_place_t* args, void* stream) {
    return guarded([&]() -> int {
        if (args == nullptr) return invalid("null pointer: args");
        const int st = check_place(*args, nullptr, nullptr);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_place(*args, static_cast<hipStream_t>(stream)), "cq_place");
    });
}

int cq_kv_append_rows(const cq_kv_cache_t* cache, int dtype, int64_t tokens,
                      const int64_t* slots, const void* k, int64_t k_token_stride,
                      int64_t k_head_stride, const void* v, int64_t v_token_stride,
                      int64_t v_head_stride, void* stream) {
    return guarded([&]() -> int {
        if (cache == nullptr) return invalid("null pointer: cache");
        const cq::KvStrides ks{0, k_token_stride, k_head_stride};
        const cq::KvStrides vs{0, v_token_stride, v_head_stride};
        const int st = check_append_rows(*cache, dtype, tokens, slots, k, ks, v, vs);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_kv_append_rows(*cache, dtype, tokens, slots, k, ks, v, vs,
                                                    static_cast<hipStream_t>(stream)),
                          "cq_kv_append_rows");
    });
}

}  // extern "C"
