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

// Scale of a vector and the reciprocal that its codes are rounded with, from the
// bits of its largest |x|: 0 for a vector of tiny numbers (the scale or its
// reciprocal would leave FP32's normal range), NaN for one with NaN or Inf.
template <int BITS>
__device__ __forceinline__ void scale_of(uint32_t amax_bits, float& scale, float& inv) {
    constexpr float rcp = 1.0f / (BITS == 8 ? 127.0f : 7.0f);
    const float amax = __uint_as_float(amax_bits);
    scale = amax * rcp;
    inv = 1.0f / scale;
    if (amax < 0x1p-100f) scale = inv = 0.f;
    if (amax_bits >= 0x7F800000u) {
        scale = __builtin_nanf("");
        inv = 0.f;
    }
}

// The upper half of the wave's a changes places with the lower half of its b.
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

// `bytes` from base on as a buffer: a load past them gives 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000);
}

// 16 bytes a lane from base + at (0 where that passes `bytes`; both the wave's)
// straight to LDS, lane after lane from `to` (the wave's, 16-byte aligned).
__device__ __forceinline__ void load_to_lds(void* to, const void* base, int bytes, int at) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        buffer_of(base, bytes), (__attribute__((address_space(3))) void*)to, 16, at, 0, 0, 0);
}

// Page of a table entry, or -1 for one outside the cache.
__device__ __forceinline__ int64_t page_in(int32_t entry, int64_t pages) {
    return entry >= 0 && entry < pages ? (int64_t)entry : -1;
}

}  // namespace cq
