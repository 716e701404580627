// Attention over the quantized paged cache where the call's own tokens form a
// tree: each sees what lies ahead of all of them, and of them those that its bits
// name.  As cq_attention.hip, with one difference: where tiles hold the call's
// tokens a lane takes the 16 bits of its row for its 16 keys from `seen` and masks
// by them.  Tiles ahead cost what they cost there, and the same prefix's kernel
// and join are used.

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
