// Internal interface of the operators around attention: the C entry points
// (cq_attn_capi.cpp) check a call's arguments and hand them on unchanged to
// the launchers (cq_norm_rope.hip, cq_kvcache.hip, cq_attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>
#include <string>

#include "cdnaqgemv.h"

namespace cq {

// Sets the calling thread's cq_last_error() text and returns `code`
// (cq_capi.cpp).
int set_error(int code, const std::string& msg);

// Workgroups of all of a call's launches (31 bits in the kernels), and those of
// 256 threads that one launch may have: HIP counts a launch's threads in 32 bits.
constexpr int64_t kMaxGrid = 0x7FFFFFFF;
constexpr int64_t kMaxLaunch = 0xFFFFFFFF / 256;

// go(workgroups, first) for each launch of a call of `grid` workgroups.
template <class Go>
hipError_t launch_parts(int64_t grid, Go&& go) {
    hipError_t e = hipSuccess;
    for (int64_t first = 0; first < grid && e == hipSuccess; first += kMaxLaunch) {
        go(dim3((unsigned)std::min(grid - first, kMaxLaunch)), (uint32_t)first);
        e = hipGetLastError();
    }
    return e;
}

// Launchers: arguments are checked, sizes are positive.  A launcher that
// finds its grid beyond kMaxGrid returns hipErrorInvalidValue unlaunched.
hipError_t launch_norm_rope(const cq_norm_rope_t& a, hipStream_t stream);
// Element strides of k or v [batch, tokens, heads, head_dim].
struct KvStrides {
    int64_t batch, token, head;
};
hipError_t launch_kv_append(const cq_kv_cache_t& c, const cq_kv_slots_t& s, int dtype,
                            const void* k, KvStrides ks, const void* v, KvStrides vs,
                            hipStream_t stream);
hipError_t launch_kv_read(const cq_kv_cache_t& c, const cq_kv_slots_t& s, int dtype,
                          void* k_out, void* v_out, hipStream_t stream);

// The checks of an attention call (cq_attn_capi.cpp) whose workspace is that many
// bytes (-1: its tables are too long); `launching`: those of its addresses too.
int check_attention(const cq_kv_cache_t& c, const cq_attention_t& a, bool launching,
                    int64_t (*workspace)(const cq_kv_cache_t&, const cq_attention_t&));

// Bytes, or -1 for a call whose tables span more tiles than 31 bits count.
int64_t attention_workspace(const cq_kv_cache_t& c, const cq_attention_t& a);
hipError_t launch_attention(const cq_kv_cache_t& c, const cq_attention_t& a,
                            hipStream_t stream);

}  // namespace cq
