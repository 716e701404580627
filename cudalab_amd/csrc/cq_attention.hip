// Attention over the quantized paged cache where the call's own tokens follow one
// another: what it launches.  The arithmetic and the kernels are described in
// cq_attention_kernels.h.

#include "cq_attention_kernels.h"
#include "cq_step.h"

namespace cq {
namespace {

template <class T, int D>
hipError_t join(const Source& own, Shape os, const Source& ahead, hipStream_t stream) {
    // a wave finds out for eight rows at once that they are finished, as most
    // are where rows are many (1024 tokens of 64 heads over 8700 keys: the call 357
    // us with one row, 348 with eight; of four sequences 1376 and 1336); of few
    // rows most have triples to join, one row a wave
    const int64_t all = (int64_t)own.rows * own.a.batch * own.c.heads;
    const int each = own.finish && os.nb == 0 && all >= 32 * kWaves * kCus ? 8 : 1;
    const int64_t places = (int64_t)((own.rows + each - 1) / each) * own.a.batch * own.c.heads;
    // units over more runs than a wave has loads for: four waves to a row, as
    // long as the rows alone do not fill the device (calls of 64 rows, us with one
    // wave and with four: of 19 runs 13.6 13.7, of 64 22.0 20.7, of 256 22.8 18.8;
    // the join of 4096 rows of 18: 12.1 13.6)
    const int64_t runs = own.runs / ((int64_t)own.row_groups * own.a.batch * own.c.heads) +
                         (ahead.rows > 0 ? ahead.runs / ((int64_t)ahead.row_groups * own.c.heads)
                                         : 0);
    const bool four = each == 1 && places <= 4 * kCus && runs > in_flight<D>;
    const int64_t grid = four ? places : (places + kWaves - 1) / kWaves;
    return launch_parts(grid, [&](dim3 blocks, uint32_t first) {
        if (four)
            join_kernel<T, D, kWaves><<<blocks, dim3(kBlock), 0, stream>>>(own, ahead, each, first);
        else
            join_kernel<T, D, 1><<<blocks, dim3(kBlock), 0, stream>>>(own, ahead, each, first);
    });
}

// Bytes that a call's sources take, or -1 where their tables are too long.
int64_t workspace_of(const cq_kv_cache_t& c, const cq_attention_t& a, bool tree) {
    Shape os{}, as{};
    Source own = source_of(c, a, false, &os, tree), ahead{};
    if (a.prefix_len > 0) ahead = source_of(c, a, true, &as);
    if (!own.fits || (ahead.rows > 0 && !ahead.fits)) return -1;
    return lay_out(c, a, &own, &ahead, nullptr);
}

}  // namespace

int64_t attention_workspace(const cq_kv_cache_t& c, const cq_attention_t& a) {
    return workspace_of(c, a, false);
}

int64_t attention_tree_workspace(const cq_kv_cache_t& c, const cq_attention_t& a) {
    return workspace_of(c, a, true);
}

hipError_t launch_attention_ahead(const cq_kv_cache_t& c, const cq_attention_t& a,
                                  hipStream_t stream) {
    if (a.prefix_len == 0) return hipSuccess;
    const Sources s(c, a, true);
    return by_head(c, a, [&](auto elem, auto dim) {
        return launch_source<decltype(elem), decltype(dim)::value, false>(s.ahead, s.as, stream);
    });
}

// A tree's rows are many, and most of their units lie in two runs or three: a wave to
// a row, four triples in flight (49152 rows, us: eight rows to a wave and 16 in flight
// as `join` has it for other calls 50, this 28).
hipError_t launch_attention_tree_join(const cq_kv_cache_t& c, const cq_attention_t& a,
                                      hipStream_t stream) {
    const Sources s(c, a, true);
    return by_head(c, a, [&](auto elem, auto dim) {
        using T = decltype(elem);
        constexpr int D = decltype(dim)::value;
        const int64_t rows = (int64_t)s.own.rows * a.batch * c.heads;
        if (rows < 4 * kWaves * kCus) return join<T, D>(s.own, s.os, s.ahead, stream);
        return launch_parts((rows + kWaves - 1) / kWaves, [&](dim3 blocks, uint32_t first) {
            join_kernel<T, D, 1, 4><<<blocks, dim3(kBlock), 0, stream>>>(s.own, s.ahead, 1, first);
        });
    });
}

hipError_t launch_attention(const cq_kv_cache_t& c, const cq_attention_t& a,
                            hipStream_t stream) {
    const Sources s(c, a, false);
    return by_head(c, a, [&](auto elem, auto dim) {
        using T = decltype(elem);
        constexpr int D = decltype(dim)::value;
        hipError_t e = hipSuccess;
        if (s.ahead.rows > 0) e = launch_source<T, D, false>(s.ahead, s.as, stream);
        if (e == hipSuccess) e = launch_source<T, D, false>(s.own, s.os, stream);
        if (e == hipSuccess) e = join<T, D>(s.own, s.os, s.ahead, stream);
        return e;
    });
}

}  // namespace cq
