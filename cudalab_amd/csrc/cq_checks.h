// What the C entry points check with: spans of memory that must not meet, the
// cache's and the tables' arguments, statuses.  Host code only.
#pragma once

#include <climits>
#include <initializer_list>
#include <string>
#include <utility>

#include "cdnaqgemv.h"
#include "cq_attn.h"

namespace cq::checks {

using U = unsigned __int128;

inline int invalid(const char* what) { return cq::set_error(CQ_ERR_INVALID_ARG, what); }

inline int hip_status(hipError_t e, const char* what) {
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

inline int64_t elem_bytes(int dtype) { return dtype == CQ_DTYPE_F32 ? 4 : 2; }

inline bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Bytes [lo, hi) of an operand; empty where there is none.
struct Span {
    U lo = 0, hi = 0;
    Span() = default;
    Span(const void* p, U bytes) : lo(reinterpret_cast<uintptr_t>(p)), hi(lo + bytes) {
        if (p == nullptr) lo = hi = 0;
    }
};

inline bool overlap(const Span& a, const Span& b) {
    return a.lo < a.hi && b.lo < b.hi && a.lo < b.hi && b.lo < a.hi;
}

// An operand of `rows` x `cols` x ... innermost runs: extents and strides in
// elements, strides not negative.
inline Span strided(const void* p, std::initializer_list<std::pair<int64_t, int64_t>> dims,
                    int64_t run, int64_t elem) {
    U last = 0;
    for (const auto& [n, stride] : dims) {
        if (n <= 0) return {};
        last += static_cast<U>(n - 1) * static_cast<U>(stride);
    }
    return Span(p, (last + static_cast<U>(run)) * static_cast<U>(elem));
}

inline int check_cache(const cq_kv_cache_t& c) {
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

inline int check_table(const int32_t* table, int64_t stride, int32_t cols, int32_t batch) {
    if (table == nullptr) return invalid("null pointer: table");
    if (!aligned(table, 4)) return invalid("table must be 4-byte aligned");
    if (cols < 1) return invalid("table_cols must be >= 1");
    if (batch > 1 && (stride < cols || stride > (int64_t)1 << 40))
        return invalid("table_stride must be at least table_cols");
    return CQ_OK;
}

inline Span table_span(const int32_t* table, int64_t stride, int32_t cols, int32_t batch) {
    return strided(table, {{batch, stride}}, cols, 4);
}

// Whether a span written meets another operand of the call.
template <int N, int M>
bool meet(const Span (&out)[N], const Span (&in)[M]) {
    for (int i = 0; i < N; ++i) {
        for (int j = i + 1; j < N; ++j)
            if (overlap(out[i], out[j])) return true;
        for (const Span& x : in)
            if (overlap(out[i], x)) return true;
    }
    return false;
}

// A call of cq_place, or with counts of held pages (cq_place_held).
inline int check_place(const cq_place_t& a, const int32_t* held_in, const int32_t* held_out) {
    if (a.batch < 1 || a.batch == INT_MAX) return invalid("batch must be in [1, 2^31-2]");
    if (a.tokens < 0 || a.tokens > INT_MAX) return invalid("tokens must be in [0, 2^31-1]");
    if (a.page_size < 16 || a.page_size > 256 || (a.page_size & (a.page_size - 1)) != 0)
        return invalid("page_size must be 16, 32, 64, 128 or 256");
    if (a.free_count < 0 || a.free_count > (int64_t)1 << 40)
        return invalid("free_count must be in [0, 2^40]");
    int st = check_table(a.table, a.table_stride, a.table_cols, a.batch);
    if (st != CQ_OK) return st;
    if ((int64_t)a.table_cols * a.page_size > INT_MAX)
        return invalid("table_cols * page_size must be below 2^31");
    if (a.starts == nullptr || a.counts == nullptr || a.offsets == nullptr ||
        a.lengths == nullptr || a.taken_out == nullptr ||
        (a.free_count > 0 && a.free_pages == nullptr) ||
        (a.tokens > 0 && (a.slots == nullptr || a.positions == nullptr)))
        return invalid("null pointer argument");
    for (const void* p : {(const void*)a.starts, (const void*)a.counts, (const void*)a.free_pages,
                          (const void*)a.taken_in, (const void*)a.positions,
                          (const void*)a.offsets, (const void*)a.lengths,
                          (const void*)a.taken_out, (const void*)held_in, (const void*)held_out})
        if (!aligned(p, 4)) return invalid("a pointer is not aligned to its element size");
    if (!aligned(a.slots, 8)) return invalid("a pointer is not aligned to its element size");
    const U batch = static_cast<U>(a.batch), tokens = static_cast<U>(a.tokens);
    const Span out[] = {table_span(a.table, a.table_stride, a.table_cols, a.batch),
                        Span(a.slots, tokens * 8),
                        Span(a.positions, tokens * 4),
                        Span(a.offsets, (batch + 1) * 4),
                        Span(a.lengths, batch * 4),
                        Span(a.taken_out, 4),
                        Span(held_out, batch * 4)};
    const Span in[] = {Span(a.starts, batch * 4), Span(a.counts, batch * 4),
                       Span(a.free_pages, static_cast<U>(a.free_count) * 4), Span(a.taken_in, 4),
                       Span(held_in, batch * 4)};
    if (meet(out, in)) return invalid("an output overlaps another operand");
    return CQ_OK;
}

inline bool known_dtype(int d) { return d == CQ_DTYPE_F16 || d == CQ_DTYPE_F32 || d == CQ_DTYPE_BF16; }

}  // namespace cq::checks
