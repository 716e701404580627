// INT8 products of many tokens (gfx950): activations quantized with a scale for
// each token, multiplied with the weights of the INT8 GEMV.
//
//   codes:  scale = amax * fl(1 / 127), code = rint(x * fl(1 / scale))
//   out[t, n] = (sum_k x[t, k] w[n, k]) * x_scale[t] * w_scale[n]
//
// The sums are whole numbers in 32 bits (v_mfma_i32_*_i8), so neither the order
// nor the way the work is split changes a result; scales multiply in FP32, and
// the result is rounded once.

#include <algorithm>
#include <type_traits>

#include "cq_elem.h"
#include "cq_step.h"

namespace cq {
namespace {

using i4 = Vec<int, 4>;
using i16v = Vec<int, 16>;
using u4 = Vec<uint32_t, 4>;

// -------------------------------------------------------------- activations
constexpr int kBlock = 256;

// |x| as FP32 bits: NaN above Inf above every number.
template <class T>
__device__ __forceinline__ uint32_t magnitude(T x) {
    return __float_as_uint((float)x) & 0x7FFFFFFFu;
}

// One workgroup to a token; what it holds of the row (HOLD pieces of 8 elements a
// thread) is read once, the rest again.  Codes need no clamp: x * inv lies within
// 127 (1 + 2^-21).
template <class T, int HOLD>
__global__ __launch_bounds__(kBlock) void quantize_kernel(const T* x, int64_t stride, int64_t k,
                                                          int8_t* codes, float* scales, bool wide,
                                                          uint32_t first) {
    __shared__ uint32_t most[kBlock / 64];
    const int64_t row = (int64_t)first + blockIdx.x;
    const T* p = x + row * stride;
    int8_t* to = codes + row * k;
    constexpr int N = 8;
    Vec<T, N> held[HOLD];
    uint32_t m = 0;
    auto get = [&](int64_t at) {
        Vec<T, N> v = {};
        if (wide && at + N <= k) {
            if constexpr (sizeof(T) == 4) {
                const Vec<T, 4> a = *reinterpret_cast<const Vec<T, 4>*>(p + at);
                const Vec<T, 4> b = *reinterpret_cast<const Vec<T, 4>*>(p + at + 4);
                v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                v = *reinterpret_cast<const Vec<T, N>*>(p + at);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < k) v[i] = p[at + i];
        }
        return v;
    };
    auto most_of = [&](const Vec<T, N>& v) {
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, magnitude(v[i]));
    };
    const int64_t mine = (int64_t)threadIdx.x * N;
#pragma unroll
    for (int j = 0; j < HOLD; ++j) held[j] = get(mine + j * kBlock * N);
#pragma unroll
    for (int j = 0; j < HOLD; ++j) most_of(held[j]);
    for (int64_t at = mine + HOLD * kBlock * N; at < k; at += kBlock * N) most_of(get(at));
    m = max(m, row_dpp<0x128>(m));
    m = max(m, row_dpp<0x124>(m));
    m = max(m, row_dpp<0x122>(m));
    m = max(m, row_dpp<0x121>(m));
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBlock / 64; ++i) m = max(m, most[i]);
    float scale, inv;
    scale_of<8>(m, scale, inv);
    if (threadIdx.x == 0) scales[row] = scale;
    const bool whole = (reinterpret_cast<uintptr_t>(to) & 7) == 0;
    auto put = [&](int64_t at, const Vec<T, N>& v) {
        if (at >= k) return;
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                c[j] = __float_as_uint((float)v[4 * i + j] * inv + 0x1.8p23f);
            w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0C0C0400u),
                                         __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u),
                                         0x05040100u);
            // inv 0 stands for a row of zeros, whose x may be NaN or Inf
            if (inv == 0.f) w[i] = 0;
        }
        if (whole && at + N <= k) {
            *reinterpret_cast<Vec<uint32_t, 2>*>(to + at) = Vec<uint32_t, 2>{w[0], w[1]};
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (at + i < k) to[at + i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
        }
    };
#pragma unroll
    for (int j = 0; j < HOLD; ++j) put(mine + j * kBlock * N, held[j]);
    for (int64_t at = mine + HOLD * kBlock * N; at < k; at += kBlock * N) put(at, get(at));
}

// ------------------------------------------------------------------ products
// 16 bytes of a row of codes from byte `at` on, where the row is not aligned to
// words: the words around them that hold any, shifted.  `end` bytes belong to
// the operand; what lies behind comes as 0.
__device__ __forceinline__ u4 unaligned16(const int8_t* base, int64_t at, int64_t end) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(base) + at;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(p & ~(uintptr_t)3);
    const uint32_t shift = p & 3;
    uint32_t w[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = at + 4 * i - (int64_t)shift < end ? words[i] : 0;
    u4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_alignbyte(w[i + 1], w[i], shift);
    return r;
}

// The bytes of 16 from `at` on that lie below k, the others 0.
__device__ __forceinline__ u4 below(u4 v, int64_t at, int64_t k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t left = k - at - 4 * i;
        if (left < 4) v[i] &= left <= 0 ? 0u : (1u << (8 * left)) - 1;
    }
    return v;
}

template <class T, int N>
__device__ __forceinline__ void store_scaled(T* p, const int* sums, float xs, const float* ws,
                                             int n, bool whole) {
    Vec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float y = (float)sums[i] * xs * ws[i];
        // the last product is rounded to FP32 (not in one with the conversion)
        asm("" : "+v"(y));
        v[i] = (T)y;
    }
    if (whole) {
        *reinterpret_cast<Vec<T, N>*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = v[i];
    }
}

constexpr int kDeep = 128;             // bytes of k of a tile

// A workgroup computes BN channels of BM tokens; its WM x WN waves share tiles of
// 128 codes of their rows, two in turn: the next comes from memory straight to
// LDS while one is multiplied.  Pieces of 16 bytes lie at places turned by the
// row, so that 16 rows' same piece meets every bank once.
// WORDS: rows start at words and the loads need no shifting.
template <class T, int BM, int BN, int WM, int WN, bool WORDS>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_kernel(cq_qgemm_t a, uint32_t m_tiles,
                                                            uint32_t n_tiles) {
    constexpr int W = WM * WN;
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int kTileBytes = (BM + BN) * kDeep;
    constexpr int kXLoads = BM / 8 / W, kWLoads = BN / 8 / W;       // 8 rows each
    static_assert(kXLoads * 8 * W == BM && kWLoads * 8 * W == BN, "whole loads");
    __shared__ __attribute__((aligned(1024))) uint8_t sm[2 * kTileBytes];
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // neighbours on an XCD take neighbouring tiles, four rows of tiles at a time
    const uint32_t all = m_tiles * n_tiles, xcd = blockIdx.x % 8, each = all / 8, over = all % 8;
    const uint32_t tile = xcd * each + min(xcd, over) + blockIdx.x / 8;
    constexpr uint32_t kBand = 4;
    const uint32_t band = tile / (kBand * n_tiles), first = band * kBand;
    const uint32_t high = min(kBand, m_tiles - first), in = tile - first * n_tiles;
    const int64_t m0 = (int64_t)(first + in % high) * BM, n0 = (int64_t)(in / high) * BN;

    const int8_t* xp = a.x + m0 * a.x_stride;
    const int8_t* wp = a.w + n0 * a.k;
    const int64_t x_end = (std::min<int64_t>(a.tokens - m0, BM) - 1) * a.x_stride + a.k;
    const int64_t w_end = std::min<int64_t>(a.n - n0, BN) * a.k;
    auto turn = [](int row) { return row >> 1 & 7; };
    const int piece = lane & 7;
    auto row_of = [&](int i) { return (wave + W * i) * 8 + (lane >> 3); };
    const int k = (int)a.k, steps = (k + kDeep - 1) / kDeep;
    auto fetch = [&](int step, int buf) {
        uint8_t* to = sm + buf * kTileBytes;
        auto load = [&](uint8_t* dst, const int8_t* base, int64_t end, int64_t stride, int i) {
            const int row = row_of(i), at = (piece ^ turn(row)) * 16;
            if constexpr (WORDS) {
                // past the row's end nothing is loaded: zeros come
                const int64_t from = row * stride + step * kDeep + at;
                const bool some = step * kDeep + at < k && row * stride < end;
                load_to_lds(dst + (wave + W * i) * 1024, base, (int)end,
                            some ? (int)from : 0x7FFFFFFF);
            } else {
                const int64_t from = row * stride + step * kDeep + at;
                u4 v = {};
                if (step * kDeep + at < k && row * stride < end)
                    v = below(unaligned16(base, from, end), step * kDeep + at, k);
                *reinterpret_cast<u4*>(dst + (wave + W * i) * 1024 + lane * 16) = v;
            }
        };
#pragma unroll
        for (int i = 0; i < kXLoads; ++i) load(to, xp, x_end, a.x_stride, i);
#pragma unroll
        for (int i = 0; i < kWLoads; ++i) load(to + BM * kDeep, wp, w_end, a.k, i);
    };
    i16v acc[TN][TM];
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[n][m] = i16v{};
    fetch(0, 0);
    for (int step = 0; step < steps; ++step) {
        __syncthreads();
        uint8_t* buf = sm + (step & 1) * kTileBytes;
        if (WORDS && step == steps - 1 && k % 16 != 0) {
            // a last piece that is a row's in part: the rest of x is made 0
            if ((int)threadIdx.x < BM) {
                const int row = threadIdx.x, p = k % kDeep / 16;
                u4* at = reinterpret_cast<u4*>(buf + row * kDeep + (p ^ turn(row)) * 16);
                *at = below(*at, p * 16, k % kDeep);
            }
            __syncthreads();
        }
        if (step + 1 < steps) fetch(step + 1, (step + 1) & 1);
        const uint8_t* xs = buf + (wm * TM * 32 + col) * kDeep;
        const uint8_t* ws = buf + BM * kDeep + (wn * TN * 32 + col) * kDeep;
#pragma unroll
        for (int u = 0; u < kDeep / 32; ++u) {
            const int at = ((2 * u + half) ^ turn(col)) * 16;
            i4 x[TM], w[TN];
#pragma unroll
            for (int m = 0; m < TM; ++m) x[m] = *reinterpret_cast<const i4*>(xs + m * 32 * kDeep + at);
#pragma unroll
            for (int n = 0; n < TN; ++n) w[n] = *reinterpret_cast<const i4*>(ws + n * 32 * kDeep + at);
#pragma unroll
            for (int n = 0; n < TN; ++n)
#pragma unroll
                for (int m = 0; m < TM; ++m)
                    acc[n][m] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[n], x[m], acc[n][m], 0, 0, 0);
        }
    }
    // acc[n][m][j]: token 32 m + col, channel 32 n + 8 (j / 4) + 4 half + j % 4
    T* out = static_cast<T*>(a.out);
    const bool even = a.n % 4 == 0;
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const int64_t t = m0 + (wm * TM + m) * 32 + col;
        if (t >= a.tokens) continue;
        const float xscale = a.x_scale[t];
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const int64_t c = n0 + (wn * TN + n) * 32 + 2 * j + 4 * half;
                if (c >= a.n) continue;
                const int left = (int)std::min<int64_t>(4, a.n - c);
                float wscale[4];
                int sums[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    wscale[i] = a.w_scale[c + std::min(i, left - 1)];
                    sums[i] = acc[n][m][j + i];
                }
                store_scaled<T, 4>(out + t * a.n + c, sums, xscale, wscale, left, even);
            }
    }
}

// ------------------------------------------------------------------- host
template <class T, int BM, int BN, int WM, int WN>
hipError_t launch_tiles(const cq_qgemm_t& a, hipStream_t stream) {
    const int64_t m = (a.tokens + BM - 1) / BM, n = (a.n + BN - 1) / BN;
    if ((__int128)m * n > kMaxLaunch / 4) return hipErrorInvalidValue;
    const bool words = a.k % 4 == 0 && a.x_stride % 4 == 0 && (uintptr_t)a.x % 4 == 0 &&
                       (uintptr_t)a.w % 4 == 0;
    const dim3 grid((unsigned)(m * n)), block(64 * WM * WN);
    // offsets inside a tile of rows fit 31 bits
    if (words && a.x_stride <= (1 << 22))
        tile_kernel<T, BM, BN, WM, WN, true><<<grid, block, 0, stream>>>(a, (uint32_t)m, (uint32_t)n);
    else
        tile_kernel<T, BM, BN, WM, WN, false><<<grid, block, 0, stream>>>(a, (uint32_t)m, (uint32_t)n);
    return hipGetLastError();
}

template <class T>
hipError_t launch_typed(const cq_qgemm_t& a, hipStream_t stream) {
    const int64_t large = ((a.tokens + 255) / 256) * ((a.n + 255) / 256);
    if (a.tokens > 128 && large >= 192) return launch_tiles<T, 256, 256, 2, 4>(a, stream);
    return launch_tiles<T, 128, 128, 2, 2>(a, stream);
}

template <class T>
hipError_t quantize_typed(const void* x, int64_t stride, int64_t tokens, int64_t k, int8_t* codes,
                          float* scales, hipStream_t stream) {
    const T* p = static_cast<const T*>(x);
    const bool wide = (uintptr_t)x % 16 == 0 && stride % (16 / sizeof(T)) == 0;
    return launch_parts(tokens, [&](dim3 blocks, uint32_t first) {
        auto go = [&](auto hold) {
            quantize_kernel<T, decltype(hold)::value>
                <<<blocks, dim3(kBlock), 0, stream>>>(p, stride, k, codes, scales, wide, first);
        };
        if (k <= 2 * kBlock * 8) go(std::integral_constant<int, 2>{});
        else if (k <= 4 * kBlock * 8) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 8>{});
    });
}

}  // namespace

hipError_t launch_quantize_tokens(int dtype, const void* x, int64_t x_stride, int64_t tokens,
                                  int64_t k, int8_t* codes, float* scales, hipStream_t stream) {
    if (dtype == CQ_DTYPE_F16)
        return quantize_typed<_Float16>(x, x_stride, tokens, k, codes, scales, stream);
    if (dtype == CQ_DTYPE_BF16)
        return quantize_typed<__bf16>(x, x_stride, tokens, k, codes, scales, stream);
    return quantize_typed<float>(x, x_stride, tokens, k, codes, scales, stream);
}

int64_t qgemm_workspace(const cq_qgemm_t&) { return 0; }

hipError_t launch_qgemm(const cq_qgemm_t& a, hipStream_t stream) {
    if (a.dtype == CQ_DTYPE_F16) return launch_typed<_Float16>(a, stream);
    if (a.dtype == CQ_DTYPE_BF16) return launch_typed<__bf16>(a, stream);
    return launch_typed<float>(a, stream);
}

}  // namespace cq
