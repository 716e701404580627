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
using f4 = Vec<float, 4>;

// -------------------------------------------------------------- activations
constexpr int kBlock = 256;

// |x| as FP32 bits: NaN above Inf above every number.
template <class T>
__device__ __forceinline__ uint32_t magnitude(T x) {
    return __float_as_uint((float)x) & 0x7FFFFFFFu;
}

// One workgroup to a token; what it holds of the row (HOLD pieces of 8 elements a
// thread) is read once, the rest again.  Codes need no clamp: x * inv lies within
// 127 (1 + 2^-21).  Bound by memory: 4096 tokens of 8192 in fp16 17.3 us, in fp32 28.8,
// 5.8 TB/s.
template <class T, int HOLD>
__global__ __launch_bounds__(kBlock) void quantize_kernel(const T* x, int64_t stride, int64_t k,
                                                          int8_t* codes, float* scales, uint32_t first) {
    __shared__ uint32_t most[kBlock / 64];
    const int64_t row = (int64_t)first + blockIdx.x;
    const T* p = x + row * stride;
    int8_t* to = codes + row * k;
    constexpr int N = 8;
    Vec<T, N> held[HOLD];
    uint32_t m = 0;
    // (loads and stores of pieces need no alignment but an element's)
    auto get = [&](int64_t at) {
        Vec<T, N> v = {};
        if (at + N <= k) {
            __builtin_memcpy(&v, p + at, sizeof v);
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
        if (at + N <= k) {
            __builtin_memcpy(to + at, w, sizeof w);
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
// A product whose rows start at words, with their distances.
struct Product {
    const int8_t* x;
    const int8_t* w;
    const float* x_scale;
    const float* w_scale;
    void* out;
    int64_t tokens, n;
    int32_t k, x_stride, w_stride;
};

// The bytes of 16 from `at` on that lie below k, the others 0.
__device__ __forceinline__ u4 below(u4 v, int at, int k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = k - at - 4 * i;
        if (left < 4) v[i] &= left <= 0 ? 0u : (1u << (8 * left)) - 1;
    }
    return v;
}

// Rows that start at any byte, to rows of whole pieces of 16 (zeros behind their
// ends).  A piece comes from the words around it that hold any of the row's bytes,
// shifted: nothing else is read.  5003 rows of 4099: 13 us; a product with shifts
// in its loads took 185 us of 777 tokens, this and the product of rows at words 47.
__global__ __launch_bounds__(kBlock) void pack_kernel(const int8_t* from, int64_t stride,
                                                      int64_t rows, int k, int8_t* to, int pieces,
                                                      uint32_t first) {
    const int64_t i = ((int64_t)first + blockIdx.x) * kBlock + threadIdx.x;
    const int64_t row = i / pieces;
    if (row >= rows) return;
    const int at = (int)(i - row * pieces) * 16;
    const uintptr_t p = reinterpret_cast<uintptr_t>(from) + row * stride + at;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(p & ~(uintptr_t)3);
    const int shift = p & 3;
    uint32_t w[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = at + 4 * j - shift < k ? words[j] : 0;
    u4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_alignbyte(w[j + 1], w[j], shift);
    *reinterpret_cast<u4*>(to + i * 16) = below(r, at, k);
}

// Four scaled sums of a token.
template <class T>
__device__ __forceinline__ Vec<T, 4> scaled(const int* sums, float xs, const float* ws) {
    Vec<T, 4> v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float y = (float)sums[i] * xs * ws[i];
        // the last product is rounded to FP32 (not in one with the conversion)
        asm("" : "+v"(y));
        v[i] = (T)y;
    }
    return v;
}

// The first `n` of N values, at any element's place.
template <class T, int N>
__device__ __forceinline__ void store_some(T* p, const Vec<T, N>& v, int64_t n) {
    if (n >= N) {
        __builtin_memcpy(p, &v, sizeof v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = v[i];
    }
}

// A workgroup computes BN channels of BM tokens.  Its waves share tiles of BK codes
// of their rows, STAGES in turn: the next come from memory straight to LDS while
// one is multiplied.  WM x WN of them share the channels and tokens, and KS such
// sets the codes of a tile; the sets' sums are added in LDS at the end.  Pieces of
// 16 bytes lie at places turned by the row, so that 16 rows' same piece meets every
// bank once.
template <class T, int BM, int BN, int WM, int WN, int KS, int BK, int STAGES>
__global__ __launch_bounds__(64 * WM * WN * KS, WM * WN * KS * STAGES > 8 ? 1 : 2) void tile_kernel(
    Product a, uint32_t m_tiles, uint32_t n_tiles) {
    constexpr int W = WM * WN * KS;
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int kTileBytes = (BM + BN) * BK;
    constexpr int kRowPieces = BK / 16, kLoadRows = 64 / kRowPieces;      // rows of a wave's load
    constexpr int kXLoads = BM / kLoadRows / W, kWLoads = BN / kLoadRows / W;
    constexpr int kUnits = BK / 32 / KS;           // products over k of a wave and tile
    static_assert(kXLoads * kLoadRows * W == BM && kWLoads * kLoadRows * W == BN, "whole loads");
    constexpr int kSums = (KS - 1) * BM * BN * 4;
    constexpr int kSpace = std::max(STAGES * kTileBytes, kSums);
    __shared__ __attribute__((aligned(1024))) uint8_t sm[kSpace + (BM + BN) * 4];
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM % WN, wk = wave / (WM * WN);

    // neighbours on an XCD take neighbouring tiles, four rows of tiles at a time
    const uint32_t all = m_tiles * n_tiles, xcd = blockIdx.x % 8, each = all / 8, over = all % 8;
    const uint32_t tile = xcd * each + min(xcd, over) + blockIdx.x / 8;
    constexpr uint32_t kBand = 4;
    const uint32_t band = tile / (kBand * n_tiles), first = band * kBand;
    const uint32_t high = min(kBand, m_tiles - first), in = tile - first * n_tiles;
    const int64_t m0 = (int64_t)(first + in % high) * BM, n0 = (int64_t)(in / high) * BN;

    const int8_t* xp = a.x + m0 * a.x_stride;
    const int8_t* wp = a.w + n0 * a.w_stride;
    const int k = a.k, steps = (k + BK - 1) / BK;
    // (whole words: rows of a k that is none have been packed, with zeros behind)
    const int row = (k + 3) & ~3;
    const int x_end = ((int)std::min<int64_t>(a.tokens - m0, BM) - 1) * a.x_stride + row;
    const int w_end = ((int)std::min<int64_t>(a.n - n0, BN) - 1) * a.w_stride + row;
    // (a row's pieces, as many rows as fill the banks)
    auto turn = [](int row) { return BK == 256 ? row & 15 : row / (256 / BK) & (kRowPieces - 1); };
    const int piece = lane % kRowPieces;
    auto row_of = [&](int i) { return (wave + W * i) * kLoadRows + lane / kRowPieces; };
    // of a lane's loads: the place in the operand's rows (of rows that are not
    // there it lies past the end, and zeros come), and in a row's tile
    int x_at[kXLoads], w_at[kWLoads];
    auto in_tile = [&](int i) { return (piece ^ turn(row_of(i))) * 16; };
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) x_at[i] = row_of(i) * a.x_stride + in_tile(i);
#pragma unroll
    for (int i = 0; i < kWLoads; ++i) w_at[i] = row_of(i) * a.w_stride + in_tile(i);
    auto fetch = [&](int step) {
        uint8_t* to = sm + step % STAGES * kTileBytes + wave * 1024;
        const int from = step * BK;
        const bool whole = from + BK <= k;
        // nor is anything loaded past the row's end
        auto place = [&](int at, int i) { return whole || from + in_tile(i) < k ? at + from : 0x7FFFFFFF; };
#pragma unroll
        for (int i = 0; i < kXLoads; ++i) load_to_lds(to + W * i * 1024, xp, x_end, place(x_at[i], i));
#pragma unroll
        for (int i = 0; i < kWLoads; ++i)
            load_to_lds(to + BM * BK + W * i * 1024, wp, w_end, place(w_at[i], i));
    };
    i16v acc[TN][TM];
#pragma unroll
    for (int n = 0; n < TN; ++n)
#pragma unroll
        for (int m = 0; m < TM; ++m) acc[n][m] = i16v{};
    // the scales, for the end
    float* const sm_x = reinterpret_cast<float*>(sm + kSpace);
    float* const sm_w = sm_x + BM;
    for (int i = threadIdx.x; i < BM; i += 64 * W)
        sm_x[i] = m0 + i < a.tokens ? a.x_scale[m0 + i] : 0.f;
    for (int i = threadIdx.x; i < BN; i += 64 * W)
        sm_w[i] = n0 + i < a.n ? a.w_scale[n0 + i] : 0.f;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);
    for (int step = 0; step < steps; ++step) {
        // the wave's loads of this step have come (those of the STAGES - 2 behind
        // it may be on their way) and its reads and writes of LDS are done, then
        // everybody's
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES - 2) * (kXLoads + kWLoads))
                     : "memory");
        const uint8_t* buf = sm + step % STAGES * kTileBytes;
        fetch(step + STAGES - 1);        // (zeros behind the last step: the count of loads stays)
        const uint8_t* xs = buf + (wm * TM * 32 + col) * BK;
        const uint8_t* ws = buf + BM * BK + (wn * TN * 32 + col) * BK;
        const bool cut = step == steps - 1 && k % 16 != 0;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int p = 2 * (wk * kUnits + u) + half, at = (p ^ turn(col)) * 16;
            i4 x[TM], w[TN];
#pragma unroll
            for (int m = 0; m < TM; ++m) x[m] = *reinterpret_cast<const i4*>(xs + m * 32 * BK + at);
#pragma unroll
            for (int n = 0; n < TN; ++n) w[n] = *reinterpret_cast<const i4*>(ws + n * 32 * BK + at);
            if (cut) {
                // a last piece that is a row's in part: the rest of x counts as 0
#pragma unroll
                for (int m = 0; m < TM; ++m)
                    x[m] = __builtin_bit_cast(
                        i4, below(__builtin_bit_cast(u4, x[m]), step * BK + p * 16, k));
            }
#pragma unroll
            for (int n = 0; n < TN; ++n)
#pragma unroll
                for (int m = 0; m < TM; ++m)
                    acc[n][m] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[n], x[m], acc[n][m], 0, 0, 0);
        }
    }
    if constexpr (KS > 1) {
        // (loads past the last step have come too: nothing but the sums is written)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        int* sums = reinterpret_cast<int*>(sm) + (wn * WM + wm) * TN * TM * 1024 + lane * 4;
        constexpr int kSet = BM * BN;
        if (wk > 0) {
#pragma unroll
            for (int n = 0; n < TN; ++n)
#pragma unroll
                for (int m = 0; m < TM; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<i4*>(sums + (wk - 1) * kSet + ((n * TM + m) * 4 + j) * 256) =
                            i4{acc[n][m][4 * j], acc[n][m][4 * j + 1], acc[n][m][4 * j + 2],
                               acc[n][m][4 * j + 3]};
        }
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int set = 0; set < KS - 1; ++set)
#pragma unroll
            for (int n = 0; n < TN; ++n)
#pragma unroll
                for (int m = 0; m < TM; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const i4 v = *reinterpret_cast<const i4*>(
                            sums + set * kSet + ((n * TM + m) * 4 + j) * 256);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][m][4 * j + i] += v[i];
                    }
    }
    // acc[n][m][j]: token 32 m + col, channel 32 n + 8 (j / 4) + 4 half + j % 4.  Of
    // types of 16 bits the halves of the wave change fours, so that a lane has eight
    // channels side by side (4096 tokens, 11008 x 4096: 213 us with stores of 8
    // bytes, 199 with these).
    T* out = static_cast<T*>(a.out);
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const int row = (wm * TM + m) * 32 + col;
        const bool there = m0 + row < a.tokens;
        const float xscale = sm_x[row];
        T* to = out + (m0 + row) * a.n + n0;
#pragma unroll
        for (int n = 0; n < TN; ++n) {
            const int c0 = (wn * TN + n) * 32;
            Vec<T, 4> v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int sums[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) sums[i] = acc[n][m][4 * j + i];
                v[j] = scaled<T>(sums, xscale, sm_w + c0 + 8 * j + 4 * half);
            }
            if constexpr (sizeof(T) == 2) {
                using u2 = Vec<uint32_t, 2>;
#pragma unroll
                for (int j = 0; j < 4; j += 2) {
                    u2 x = __builtin_bit_cast(u2, v[j]), y = __builtin_bit_cast(u2, v[j + 1]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t p = x[i], q = y[i];
                        swap_halves(p, q);
                        x[i] = p;
                        y[i] = q;
                    }
                    using T8 = Vec<T, 8>;
                    const T8 eight = __builtin_bit_cast(T8, u4{x[0], x[1], y[0], y[1]});
                    const int c = c0 + 8 * j + 8 * half;
                    if (there) store_some<T, 8>(to + c, eight, a.n - n0 - c);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = c0 + 8 * j + 4 * half;
                    if (there) store_some<T, 4>(to + c, v[j], a.n - n0 - c);
                }
            }
        }
    }
}

// ------------------------------------------------------------------- host
template <class T, int BM, int BN, int WM, int WN, int KS, int BK, int STAGES>
hipError_t launch_tiles(const Product& a, hipStream_t stream) {
    const int64_t m = (a.tokens + BM - 1) / BM, n = (a.n + BN - 1) / BN;
    constexpr int kThreads = 64 * WM * WN * KS;
    if ((__int128)m * n > kMaxLaunch * 256 / kThreads) return hipErrorInvalidValue;
    tile_kernel<T, BM, BN, WM, WN, KS, BK, STAGES>
        <<<dim3((unsigned)(m * n)), dim3(kThreads), 0, stream>>>(a, (uint32_t)m, (uint32_t)n);
    return hipGetLastError();
}

// Which tile.  Small ones leave more workgroups, large ones read less: the
// smallest that does not give the 256 CUs more than one workgroup each.  (us, with
// weights from memory, fp16 out:
//   tile                      64x32 64x64 128x64 128x128 128x160 128x192 128x256 256x256
//   35 tokens, 8192 x 8192     16.0  21.1   24.7   35      46      44      53      93
//   256 tokens, 4096 x 4096    14.9  11.6   14.4   19.5    21.5    25.4    28.6    50
//   256 tokens, 8192 x 8192    59    47     33.2   47      49      49      57     102
//   512 tokens, 8192 x 8192   119    85     60     48      53      56      62     105
//   777 tokens, 5003 x 4100    68    58     50     50      30.5    34.1    42      61
//   512 tokens, 11008 x 4096   94    73     50     45      49      32.0    35      59
//   1500 tokens, 5000 x 4096  122    83     65     50      49      54      38.1    60)
// Where even the largest of these is too many, two workgroups of 128 x 128 to a CU, or
// one of 256 x 256: per 128 codes a CU's pair takes 1.34 us (a workgroup alone 0.8),
// the large one 2.07 us, in as many rounds as they need.  (us: 4096 tokens, 11008 x 4096
// 208, 194; 28672 x 8192 965, 888 or 2170 TOP/s, where the library's product of that size
// reaches 2210.)
// By that rule 1 to 64 tokens take, us: 8192 x 8192 15.4 to 18.6, 8192 x 28672 49 to 59
// (64x32, one workgroup to a CU); 16384 x 8192 40 to 46 (64x32, two to a CU, where 65
// tokens take 34 by 128x64); 16448 x 8192 39 to 42 and 28672 x 8192 52 (128x128, 129 and
// 224 workgroups; their weights alone 23 and 39); 1024 x 8192 11 (64x32, 32 workgroups).
template <class T>
hipError_t launch_typed(const Product& a, hipStream_t stream) {
    auto tiles = [&](int64_t m, int64_t n) {
        return ((a.tokens + m - 1) / m) * ((a.n + n - 1) / n);
    };
    constexpr int kCus = 256;
    // (few tokens are bound by memory, and take it up to two workgroups to a CU)
    if (a.tokens <= 64 && tiles(64, 32) <= 2 * kCus)
        return launch_tiles<T, 64, 32, 1, 1, 4, 256, 4>(a, stream);
    if (tiles(64, 64) <= kCus) return launch_tiles<T, 64, 64, 1, 1, 4, 256, 3>(a, stream);
    if (tiles(128, 64) <= kCus) return launch_tiles<T, 128, 64, 2, 1, 4, 256, 3>(a, stream);
    const int64_t middle = tiles(128, 128), large = tiles(256, 256);
    if (middle <= kCus) return launch_tiles<T, 128, 128, 2, 2, 2, 128, 3>(a, stream);
    if (tiles(128, 160) <= kCus) return launch_tiles<T, 128, 160, 4, 1, 2, 256, 2>(a, stream);
    if (tiles(128, 192) <= kCus) return launch_tiles<T, 128, 192, 2, 2, 2, 128, 3>(a, stream);
    if (tiles(128, 256) <= kCus) return launch_tiles<T, 128, 256, 2, 4, 1, 128, 3>(a, stream);
    const int64_t over = middle % (2 * kCus);
    const double pairs = 1.34 * (double)(middle / (2 * kCus)) +
                         (over == 0 ? 0. : over <= kCus ? 0.8 : 1.34);
    if (2.07 * (double)((large + kCus - 1) / kCus) < pairs)
        return launch_tiles<T, 256, 256, 2, 4, 1, 64, 3>(a, stream);
    return launch_tiles<T, 128, 128, 2, 2, 1, 128, 2>(a, stream);
}

template <class T>
hipError_t quantize_typed(const void* x, int64_t stride, int64_t tokens, int64_t k, int8_t* codes,
                          float* scales, hipStream_t stream) {
    const T* p = static_cast<const T*>(x);
    return launch_parts(tokens, [&](dim3 blocks, uint32_t first) {
        auto go = [&](auto hold) {
            quantize_kernel<T, decltype(hold)::value>
                <<<blocks, dim3(kBlock), 0, stream>>>(p, stride, k, codes, scales, first);
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

namespace {
// Which operands need their rows moved to words (or nearer: a tile's offsets fit 31
// bits), and the bytes that takes.
struct Packing {
    bool x, w;
    int64_t row, x_bytes, w_bytes;
    explicit Packing(const cq_qgemm_t& a)
        : x(a.k % 4 != 0 || a.x_stride % 4 != 0 || (uintptr_t)a.x % 4 != 0 ||
            a.x_stride > (1 << 22)),
          w(a.k % 4 != 0 || (uintptr_t)a.w % 4 != 0), row((a.k + 15) / 16 * 16),
          x_bytes(x ? a.tokens * row : 0), w_bytes(w ? a.n * row : 0) {}
};

hipError_t pack(const int8_t* from, int64_t stride, int64_t rows, int64_t k, int8_t* to,
                int64_t row, hipStream_t stream) {
    const int64_t grid = (rows * (row / 16) + kBlock - 1) / kBlock;
    if (grid > kMaxGrid) return hipErrorInvalidValue;
    return launch_parts(grid, [&](dim3 blocks, uint32_t first) {
        pack_kernel<<<blocks, dim3(kBlock), 0, stream>>>(from, stride, rows, (int)k, to,
                                                         (int)(row / 16), first);
    });
}
}  // namespace

int64_t qgemm_workspace(const cq_qgemm_t& a) {
    const Packing p(a);
    return p.x_bytes + p.w_bytes;
}

hipError_t launch_qgemm(const cq_qgemm_t& a, hipStream_t stream) {
    const Packing p(a);
    Product s{a.x, a.w, a.x_scale, a.w_scale, a.out, a.tokens, a.n, (int32_t)a.k,
              (int32_t)a.x_stride, (int32_t)a.k};
    int8_t* space = static_cast<int8_t*>(a.workspace);
    hipError_t e = hipSuccess;
    if (p.x) {
        e = pack(a.x, a.x_stride, a.tokens, a.k, space, p.row, stream);
        s.x = space;
        s.x_stride = (int32_t)p.row;
    }
    if (p.w && e == hipSuccess) {
        e = pack(a.w, a.k, a.n, a.k, space + p.x_bytes, p.row, stream);
        s.w = space + p.x_bytes;
        s.w_stride = (int32_t)p.row;
    }
    if (e != hipSuccess) return e;
    if (a.dtype == CQ_DTYPE_F16) return launch_typed<_Float16>(s, stream);
    if (a.dtype == CQ_DTYPE_BF16) return launch_typed<__bf16>(s, stream);
    return launch_typed<float>(s, stream);
}

}  // namespace cq
