// Internal interface of the operators of a step of many tokens: the C entry
// points (cq_step_capi.cpp) check a call's arguments and hand them on unchanged
// to the launchers.
#pragma once

#include "cq_attn.h"

namespace cq {

// Launchers: arguments are checked, sizes are positive.  A launcher that
// finds its grid beyond kMaxGrid returns hipErrorInvalidValue unlaunched.

// cq_place.hip
hipError_t launch_place(const cq_place_t& a, hipStream_t stream);
// With counts of held pages, in and out (either may be null).
hipError_t launch_place_held(const cq_place_t& a, const int32_t* held_in, int32_t* held_out,
                             hipStream_t stream);

// cq_kvcache.hip.  Element strides of k or v [tokens, heads, head_dim] (of
// KvStrides `batch` is not used).
hipError_t launch_kv_append_rows(const cq_kv_cache_t& c, int dtype, int64_t tokens,
                                 const int64_t* slots, const void* k, KvStrides ks, const void* v,
                                 KvStrides vs, hipStream_t stream);

// cq_prompt.hip
hipError_t launch_prompt(const cq_prompt_t& a, hipStream_t stream);

// cq_attention.hip: of a tree's call the workspace (-1 as attention_workspace), the
// prefix's part, and the join of the parts
int64_t attention_tree_workspace(const cq_kv_cache_t& c, const cq_attention_t& a);
hipError_t launch_attention_ahead(const cq_kv_cache_t& c, const cq_attention_t& a,
                                  hipStream_t stream);
hipError_t launch_attention_tree_join(const cq_kv_cache_t& c, const cq_attention_t& a,
                                      hipStream_t stream);
// cq_attention_tree.hip
hipError_t launch_attention_tree(const cq_kv_cache_t& c, const cq_attention_t& a,
                                 const int64_t* seen, hipStream_t stream);

// cq_qgemm.hip
hipError_t launch_quantize_tokens(int dtype, const void* x, int64_t x_stride, int64_t tokens,
                                  int64_t k, int8_t* codes, float* scales, hipStream_t stream);
int64_t qgemm_workspace(const cq_qgemm_t& a);
hipError_t launch_qgemm(const cq_qgemm_t& a, hipStream_t stream);

}  // namespace cq
