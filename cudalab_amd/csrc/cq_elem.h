// Element types and lane reductions shared by the kernels around attention.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace cq {

template <class T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

// DPP within rows of 16 lanes (every lane of the row active).
template <int CTRL>
__device__ __forceinline__ uint32_t row_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float row_dpp(float v) {
    return __uint_as_float(row_dpp<CTRL>(__float_as_uint(v)));
}

// Sum over LANES (a power of two up to 64) adjacent lanes, in every one of
// them; rows of 16 by rotations, wider groups by lane exchanges.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (LANES == 4 || LANES == 8) {
        v += row_dpp<0xB1>(v);                      // quad_perm 1 0 3 2
        v += row_dpp<0x4E>(v);                      // quad_perm 2 3 0 1
        if (LANES == 8) v += row_dpp<0x141>(v);     // the row's halves mirrored
    } else if constexpr (LANES >= 16) {
        v += row_dpp<0x128>(v);
        v += row_dpp<0x124>(v);
        v += row_dpp<0x122>(v);
        v += row_dpp<0x121>(v);
        for (int off = 16; off < LANES; off <<= 1) v += __shfl_xor(v, off);
    }
    return v;
}

// Page of a table entry, or -1 for one outside the cache.
__device__ __forceinline__ int64_t page_in(int32_t entry, int64_t pages) {
    return entry >= 0 && entry < pages ? (int64_t)entry : -1;
}

}  // namespace cq
