// C entry points of the operators around attention (declared in
// include/cdnaqgemv.h): the checks that a safe launch needs.  What lies on the
// device (lengths, positions, page numbers) the kernels check themselves.

#include <climits>
#include <cmath>
#include <initializer_list>
#include <string>

#include "cdnaqgemv.h"
#include "cq_attn.h"

namespace {

using U = unsigned __int128;

int invalid(const char* what) { return cq::set_error(CQ_ERR_INVALID_ARG, what); }

int hip_status(hipError_t e, const char* what) {
    if (e == hipSuccess) return CQ_OK;
    if (e == hipErrorInvalidValue)
        return cq::set_error(CQ_ERR_INVALID_ARG,
                             std::string(what) + ": the call needs more workgroups than a launch holds");
    return cq::set_error(CQ_ERR_HIP, std::string(what) + ": " + hipGetErrorName(e) + " (" +
                                         hipGetErrorString(e) + ")");
}

// Runs an entry point's body; nothing may be thrown through the C interface
// (std::string allocates).
template <class F>
auto guarded(F&& body, decltype(body()) thrown = CQ_ERR_HIP) noexcept -> decltype(body()) {
    try {
        return body();
    } catch (...) {
        return thrown;
    }
}

int64_t elem_bytes(int dtype) { return dtype == CQ_DTYPE_F32 ? 4 : 2; }

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Bytes [lo, hi) of an operand; empty where there is none.
struct Span {
    U lo = 0, hi = 0;
    Span() = default;
    Span(const void* p, U bytes) : lo(reinterpret_cast<uintptr_t>(p)), hi(lo + bytes) {
        if (p == nullptr) lo = hi = 0;
    }
};

bool overlap(const Span& a, const Span& b) {
    return a.lo < a.hi && b.lo < b.hi && a.lo < b.hi && b.lo < a.hi;
}

// An operand of `rows` x `cols` x ... innermost runs: extents and strides in
// elements, strides not negative.
Span strided(const void* p, std::initializer_list<std::pair<int64_t, int64_t>> dims,
             int64_t run, int64_t elem) {
    U last = 0;
    for (const auto& [n, stride] : dims) {
        if (n <= 0) return {};
        last += static_cast<U>(n - 1) * static_cast<U>(stride);
    }
    return Span(p, (last + static_cast<U>(run)) * static_cast<U>(elem));
}

int check_norm_rope(const cq_norm_rope_t& a) {
    if (a.tokens < 1 || a.tokens > INT_MAX) return invalid("tokens must be in [1, 2^31-1]");
    if (a.q_heads < 0 || a.k_heads < 0 || (int64_t)a.q_heads + a.k_heads < 1 ||
        (int64_t)a.q_heads + a.k_heads > 65535)
        return invalid("q_heads and k_heads must be >= 0, 1 to 65535 together");
    if (a.head_dim < 2 || a.head_dim > 1024 || a.head_dim % 2 != 0)
        return invalid("head_dim must be even and in [2, 1024]");
    for (int d : {a.dtype, a.weight_dtype})
        if (d != CQ_DTYPE_F16 && d != CQ_DTYPE_F32 && d != CQ_DTYPE_BF16)
            return invalid("unknown dtype");
    const int64_t es = elem_bytes(a.dtype), ws = elem_bytes(a.weight_dtype);
    const int64_t strides[] = {a.q_token_stride, a.q_head_stride, a.q_out_token_stride,
                               a.q_out_head_stride, a.k_token_stride, a.k_head_stride,
                               a.k_out_token_stride, a.k_out_head_stride};
    for (int i = 0; i < 8; ++i)
        if ((i < 4 ? a.q_heads : a.k_heads) > 0 && (strides[i] < 0 || strides[i] > (int64_t)1 << 40))
            return invalid("strides must be in [0, 2^40]");
    if (a.q_heads > 0 && (a.q == nullptr || a.q_out == nullptr)) return invalid("null pointer: q");
    if (a.k_heads > 0 && (a.k == nullptr || a.k_out == nullptr)) return invalid("null pointer: k");
    if (!aligned(a.q, es) || !aligned(a.k, es) || !aligned(a.q_out, es) || !aligned(a.k_out, es) ||
        !aligned(a.q_weight, ws) || !aligned(a.k_weight, ws))
        return invalid("a pointer is not aligned to its element size");
    if ((a.cos_table == nullptr) != (a.sin_table == nullptr))
        return invalid("cos_table and sin_table come together");
    if (a.cos_table != nullptr) {
        if (a.rot_dim < 2 || a.rot_dim % 2 != 0 || a.rot_dim > a.head_dim)
            return invalid("rot_dim must be even and in [2, head_dim]");
        if (a.positions == nullptr) return invalid("null pointer: positions");
        if (a.table_rows < 1 || a.table_rows > (int64_t)1 << 40)
            return invalid("table_rows must be in [1, 2^40]");
        if (!aligned(a.cos_table, 4) || !aligned(a.sin_table, 4) ||
            !aligned(a.positions, a.positions_64 ? 8 : 4))
            return invalid("a pointer is not aligned to its element size");
    } else if (a.q_weight == nullptr && a.k_weight == nullptr) {
        return invalid("nothing to do: neither weights nor tables");
    }
    if (!(a.eps >= 0.f) || std::isinf(a.eps)) return invalid("eps must be finite and >= 0");

    // An output's heads of a token must not meet each other.
    if ((a.q_heads > 1 && a.q_out_head_stride < a.head_dim) ||
        (a.k_heads > 1 && a.k_out_head_stride < a.head_dim) ||
        (a.tokens > 1 && a.q_heads > 0 &&
         a.q_out_token_stride < (int64_t)(a.q_heads - 1) * a.q_out_head_stride + a.head_dim) ||
        (a.tokens > 1 && a.k_heads > 0 &&
         a.k_out_token_stride < (int64_t)(a.k_heads - 1) * a.k_out_head_stride + a.head_dim))
        return invalid("an output overlaps itself");
    struct Operand {
        const void* p;
        int64_t token, head;
        int32_t n;
        Span all, one;      // every token; the first token
    };
    auto operand = [&](const void* p, int64_t ts, int64_t hs, int32_t n) {
        Operand o{p, ts, hs, n, {}, {}};
        o.all = strided(p, {{a.tokens, ts}, {n, hs}}, a.head_dim, es);
        o.one = strided(p, {{n, hs}}, a.head_dim, es);
        return o;
    };
    const Operand q = operand(a.q, a.q_token_stride, a.q_head_stride, a.q_heads);
    const Operand k = operand(a.k, a.k_token_stride, a.k_head_stride, a.k_heads);
    const Operand qo = operand(a.q_out, a.q_out_token_stride, a.q_out_head_stride, a.q_heads);
    const Operand ko = operand(a.k_out, a.k_out_token_stride, a.k_out_head_stride, a.k_heads);
    auto same = [](const Operand& x, const Operand& y) {
        return x.p == y.p && x.token == y.token && x.head == y.head;
    };
    // Disjoint outright, or interleaved token by token (views of one tensor of
    // q, k and v side by side) with both runs of heads within one stride.
    auto apart = [&](const Operand& x, const Operand& y) {
        if (!overlap(x.all, y.all)) return true;
        if (x.token != y.token || overlap(x.one, y.one)) return false;
        const U lo = x.one.lo < y.one.lo ? x.one.lo : y.one.lo;
        const U hi = x.one.hi > y.one.hi ? x.one.hi : y.one.hi;
        return hi - lo <= static_cast<U>(x.token) * static_cast<U>(es);
    };
    if (!(same(qo, q) || apart(qo, q)) || !(same(ko, k) || apart(ko, k)) || !apart(qo, k) ||
        !apart(ko, q) || !apart(qo, ko))
        return invalid("an output overlaps an operand that it is not");
    const U half = static_cast<U>(a.rot_dim / 2);
    const Span rest[] = {Span(a.q_weight, static_cast<U>(a.head_dim * ws)),
                         Span(a.k_weight, static_cast<U>(a.head_dim * ws)),
                         Span(a.cos_table, static_cast<U>(a.table_rows) * half * 4),
                         Span(a.sin_table, static_cast<U>(a.table_rows) * half * 4),
                         Span(a.cos_table != nullptr ? a.positions : nullptr,
                              static_cast<U>(a.tokens) * (a.positions_64 ? 8 : 4))};
    for (const Span& r : rest)
        if (overlap(qo.all, r) || overlap(ko.all, r))
            return invalid("an output overlaps a weight, a table or the positions");
    return CQ_OK;
}

int check_cache(const cq_kv_cache_t& c) {
    if (c.k == nullptr || c.v == nullptr || c.scales == nullptr) return invalid("null pointer: cache");
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.scales, 16))
        return invalid("the cache's tensors must be 16-byte aligned");
    if (c.pages < 1 || c.pages > INT_MAX) return invalid("pages must be in [1, 2^31-1]");
    if (c.heads < 1 || c.heads > 65535) return invalid("heads must be in [1, 65535]");
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
        return invalid("the cache's head_dim must be 64, 128 or 256");
    if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1)) != 0)
        return invalid("page_size must be 16, 32, 64, 128 or 256");
    if (c.bits != 4 && c.bits != 8) return invalid("bits must be 4 or 8");
    return CQ_OK;
}

struct CacheSpans {
    Span k, v, scales;
    explicit CacheSpans(const cq_kv_cache_t& c) {
        const U tokens = static_cast<U>(c.pages) * static_cast<U>(c.heads) *
                         static_cast<U>(c.page_size);
        const U row = static_cast<U>(c.head_dim * c.bits / 8);
        k = Span(c.k, tokens * row);
        v = Span(c.v, tokens * row);
        scales = Span(c.scales, tokens * 8);
    }
    bool meet(const Span& s) const {
        return overlap(k, s) || overlap(v, s) || overlap(scales, s);
    }
    bool meet_themselves() const {
        return overlap(k, v) || overlap(k, scales) || overlap(v, scales);
    }
};

int check_table(const int32_t* table, int64_t stride, int32_t cols, int32_t batch) {
    if (table == nullptr) return invalid("null pointer: table");
    if (!aligned(table, 4)) return invalid("table must be 4-byte aligned");
    if (cols < 1) return invalid("table_cols must be >= 1");
    if (batch > 1 && (stride < cols || stride > (int64_t)1 << 40))
        return invalid("table_stride must be at least table_cols");
    return CQ_OK;
}

int check_slots(const cq_kv_slots_t& s) {
    if (s.batch < 1 || s.tokens < 1) return invalid("batch and tokens must be >= 1");
    if (s.starts == nullptr) return invalid("null pointer: starts");
    if (!aligned(s.starts, 4) || !aligned(s.counts, 4))
        return invalid("starts and counts must be 4-byte aligned");
    return check_table(s.table, s.table_stride, s.table_cols, s.batch);
}

Span table_span(const int32_t* table, int64_t stride, int32_t cols, int32_t batch) {
    return strided(table, {{batch, stride}}, cols, 4);
}

bool known_dtype(int d) { return d == CQ_DTYPE_F16 || d == CQ_DTYPE_F32 || d == CQ_DTYPE_BF16; }

int check_append(const cq_kv_cache_t& c, const cq_kv_slots_t& s, int dtype, const void* k,
                 cq::KvStrides ks, const void* v, cq::KvStrides vs) {
    int st = check_cache(c);
    if (st != CQ_OK || (st = check_slots(s)) != CQ_OK) return st;
    if (!known_dtype(dtype)) return invalid("unknown dtype");
    if (k == nullptr || v == nullptr) return invalid("null pointer: k or v");
    const int64_t es = elem_bytes(dtype);
    if (!aligned(k, es) || !aligned(v, es)) return invalid("k and v must be aligned to their element size");
    for (const cq::KvStrides& x : {ks, vs})
        for (int64_t n : {x.batch, x.token, x.head})
            if (n < 0 || n > (int64_t)1 << 40) return invalid("strides must be in [0, 2^40]");
    const CacheSpans cs(c);
    const Span inputs[] = {
        strided(k, {{s.batch, ks.batch}, {s.tokens, ks.token}, {c.heads, ks.head}}, c.head_dim, es),
        strided(v, {{s.batch, vs.batch}, {s.tokens, vs.token}, {c.heads, vs.head}}, c.head_dim, es),
        table_span(s.table, s.table_stride, s.table_cols, s.batch),
        Span(s.starts, static_cast<U>(s.batch) * 4), Span(s.counts, static_cast<U>(s.batch) * 4)};
    for (const Span& in : inputs)
        if (cs.meet(in)) return invalid("an input overlaps the cache");
    if (cs.meet_themselves()) return invalid("the cache's tensors overlap");
    return CQ_OK;
}

int check_read(const cq_kv_cache_t& c, const cq_kv_slots_t& s, int dtype, const void* k,
               const void* v) {
    int st = check_cache(c);
    if (st != CQ_OK || (st = check_slots(s)) != CQ_OK) return st;
    if (!known_dtype(dtype)) return invalid("unknown dtype");
    if (k == nullptr || v == nullptr) return invalid("null pointer: k_out or v_out");
    if (!aligned(k, 16) || !aligned(v, 16)) return invalid("k_out and v_out must be 16-byte aligned");
    const U bytes = static_cast<U>(s.batch) * static_cast<U>(s.tokens) * static_cast<U>(c.heads) *
                    static_cast<U>(c.head_dim) * static_cast<U>(elem_bytes(dtype));
    const Span ko(k, bytes), vo(v, bytes);
    const CacheSpans cs(c);
    const Span inputs[] = {table_span(s.table, s.table_stride, s.table_cols, s.batch),
                           Span(s.starts, static_cast<U>(s.batch) * 4),
                           Span(s.counts, static_cast<U>(s.batch) * 4)};
    for (const Span& in : inputs)
        if (overlap(ko, in) || overlap(vo, in)) return invalid("an output overlaps an input");
    if (cs.meet(ko) || cs.meet(vo) || overlap(ko, vo)) return invalid("an output overlaps an input");
    return CQ_OK;
}

int check_attention(const cq_kv_cache_t& c, const cq_attention_t& a, bool launching) {
    int st = check_cache(c);
    if (st != CQ_OK) return st;
    if (a.batch < 1 || a.tokens < 1) return invalid("batch and tokens must be >= 1");
    if (a.q_heads < 1 || a.q_heads > 65535 || a.q_heads % c.heads != 0)
        return invalid("q_heads must be a multiple of the cache's heads, at most 65535");
    if ((int64_t)a.batch * a.tokens > INT_MAX / a.q_heads)
        return invalid("batch * tokens * q_heads must be below 2^31");
    if (a.dtype != CQ_DTYPE_F16 && a.dtype != CQ_DTYPE_BF16)
        return invalid("dtype must be CQ_DTYPE_F16 or CQ_DTYPE_BF16");
    if (a.prefix_len < 0) return invalid("prefix_len must be >= 0");
    if (a.prefix_len > 0 && (a.prefix_cols < 1 || (int64_t)a.prefix_cols * c.page_size < a.prefix_len))
        return invalid("the prefix's pages must hold prefix_len tokens");
    if (a.table_cols < 1) return invalid("table_cols must be >= 1");
    if (std::isnan(a.softmax_scale) || std::isinf(a.softmax_scale))
        return invalid("softmax_scale must be finite");
    const int64_t need = cq::attention_workspace(c, a);
    if (need < 0)
        return invalid("the tables' tokens times batch, rows and heads are too many for one call");
    if (!launching) return CQ_OK;
    if ((st = check_table(a.table, a.table_stride, a.table_cols, a.batch)) != CQ_OK) return st;
    if (a.q == nullptr || a.out == nullptr || a.lengths == nullptr ||
        (a.prefix_len > 0 && a.prefix_table == nullptr))
        return invalid("null pointer argument");
    if (!aligned(a.q, 16) || !aligned(a.out, 16)) return invalid("q and out must be 16-byte aligned");
    if (!aligned(a.lengths, 4) || !aligned(a.counts, 4) || !aligned(a.prefix_table, 4))
        return invalid("lengths, counts and prefix_table must be 4-byte aligned");
    for (int64_t n : {a.q_batch_stride, a.q_token_stride, a.q_head_stride})
        if (n < 0 || n > (int64_t)1 << 40 || n % 8 != 0)
            return invalid("q's strides must be multiples of 8 in [0, 2^40]");
    if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || !aligned(a.workspace, 16)))
        return cq::set_error(CQ_ERR_BUFFER_TOO_SMALL,
                             "the call needs " + std::to_string(need) +
                                 " bytes of 16-byte aligned workspace, got " +
                                 std::to_string(a.workspace_bytes));
    const int64_t es = elem_bytes(a.dtype);
    const Span out(a.out, static_cast<U>(a.batch) * static_cast<U>(a.tokens) *
                              static_cast<U>(a.q_heads) * static_cast<U>(c.head_dim * es));
    const Span ws(need > 0 ? a.workspace : nullptr, static_cast<U>(need > 0 ? need : 0));
    const CacheSpans cs(c);
    const Span inputs[] = {
        strided(a.q, {{a.batch, a.q_batch_stride}, {a.tokens, a.q_token_stride},
                      {a.q_heads, a.q_head_stride}}, c.head_dim, es),
        table_span(a.table, a.table_stride, a.table_cols, a.batch),
        Span(a.lengths, static_cast<U>(a.batch) * 4), Span(a.counts, static_cast<U>(a.batch) * 4),
        Span(a.prefix_len > 0 ? a.prefix_table : nullptr, static_cast<U>(a.prefix_cols) * 4)};
    for (const Span& in : inputs)
        if (overlap(out, in) || overlap(ws, in))
            return invalid("out or the workspace overlaps an input");
    if (cs.meet(out) || cs.meet(ws) || overlap(out, ws))
        return invalid("out or the workspace overlaps an input");
    return CQ_OK;
}

}  // namespace

extern "C" {

int cq_qk_norm_rope(const cq_norm_rope_t* args, void* stream) {
    return guarded([&]() -> int {
        if (args == nullptr) return invalid("null pointer: args");
        const int st = check_norm_rope(*args);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_norm_rope(*args, static_cast<hipStream_t>(stream)),
                          "cq_qk_norm_rope");
    });
}

int cq_kv_append(const cq_kv_cache_t* cache, const cq_kv_slots_t* slots, int dtype,
                 const void* k, int64_t k_batch_stride, int64_t k_token_stride,
                 int64_t k_head_stride, const void* v, int64_t v_batch_stride,
                 int64_t v_token_stride, int64_t v_head_stride, void* stream) {
    return guarded([&]() -> int {
        if (cache == nullptr || slots == nullptr) return invalid("null pointer: cache or slots");
        const cq::KvStrides ks{k_batch_stride, k_token_stride, k_head_stride};
        const cq::KvStrides vs{v_batch_stride, v_token_stride, v_head_stride};
        const int st = check_append(*cache, *slots, dtype, k, ks, v, vs);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_kv_append(*cache, *slots, dtype, k, ks, v, vs,
                                               static_cast<hipStream_t>(stream)),
                          "cq_kv_append");
    });
}

int cq_kv_read(const cq_kv_cache_t* cache, const cq_kv_slots_t* slots, int dtype, void* k_out,
               void* v_out, void* stream) {
    return guarded([&]() -> int {
        if (cache == nullptr || slots == nullptr) return invalid("null pointer: cache or slots");
        const int st = check_read(*cache, *slots, dtype, k_out, v_out);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_kv_read(*cache, *slots, dtype, k_out, v_out,
                                             static_cast<hipStream_t>(stream)),
                          "cq_kv_read");
    });
}

int cq_attention(const cq_kv_cache_t* cache, const cq_attention_t* args, void* stream) {
    return guarded([&]() -> int {
        if (cache == nullptr || args == nullptr) return invalid("null pointer: cache or args");
        const int st = check_attention(*cache, *args, true);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_attention(*cache, *args, static_cast<hipStream_t>(stream)),
                          "cq_attention");
    });
}

int64_t cq_attention_workspace(const cq_kv_cache_t* cache, const cq_attention_t* args) {
    return guarded([&]() -> int64_t {
        if (cache == nullptr || args == nullptr) return -invalid("null pointer: cache or args");
        const int st = check_attention(*cache, *args, false);
        if (st != CQ_OK) return -st;
        return cq::attention_workspace(*cache, *args);
    }, -CQ_ERR_HIP);
}

}  // extern "C"
