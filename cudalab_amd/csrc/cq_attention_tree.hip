// Attention over the quantized paged cache where the call's own tokens form a
// tree: each sees what lies ahead of all of them, and of them those that its bits
// name.  As cq_attention.hip, with one difference: where tiles hold the call's
// tokens a lane takes the 16 bits of its row for its 16 keys from `seen` and masks
// by them.  Tiles ahead cost what they cost there, and the same prefix's kernel
// and join are used.
//
// Bound as there by the softmax and the unpacking between the products, and by the
// joins: 16 sequences of up to 8000 keys, 48 tokens, 64/8 heads of 128, INT8, 194 us
// (100 GFLOP), of which the joins of 49152 rows are 27; 7 of up to 1501, 13 tokens,
// 28/4 heads of 64, 18.3: 12.5 and 5.3 of loads that follow one another.  (Units of
// 384 rows, twelve waves, would unpack a tile once for the large case's rows, but
// leave a wave 168 registers of the 240 that it needs.)

#include "cq_attention_kernels.h"
#include "cq_step.h"

namespace cq {

hipError_t launch_attention_tree(const cq_kv_cache_t& c, const cq_attention_t& a,
                                 const int64_t* seen, hipStream_t stream) {
    Sources s(c, a, true);
    s.own.seen = reinterpret_cast<const uint32_t*>(seen);
    s.own.words = (a.tokens + 63) / 64 * 2;
    hipError_t e = launch_attention_ahead(c, a, stream);
    if (e == hipSuccess)
        e = by_head(c, a, [&](auto elem, auto dim) {
            return launch_source<decltype(elem), decltype(dim)::value, true>(s.own, s.os, stream);
        });
    return e == hipSuccess ? launch_attention_tree_join(c, a, stream) : e;
}

}  // namespace cq
