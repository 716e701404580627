// Attention of packed sequences over their own keys and values (gfx950): whole
// prompts, or chunks of them with the keys of earlier chunks ahead.
//
//   o_t = sum_j softmax_j(scale * q_t . k_j) v_j over the keys j that token t
//   sees: all m of its sequence, or (causal) those up to m - n + t, of n tokens
//
// One pass over the keys with a running reference M and sum l of the softmax, in
// matrix form, 64 keys at a time (v_mfma_f32_32x32x16, FP32 sums):
//   S^T [keys x rows] = K [keys x D] Q^T [D x rows]
//   O^T [D x rows]   += V^T [D x keys] P^T [keys x rows]
// with p = 2^(s scale log2(e) - M), M raised when an exponent passes kRaise, so
// that the sums are seldom rescaled.  A wave takes 32 rows of one query head and
// keeps their queries, scores and sums in registers.  S comes out with a row's
// keys in the two lanes row and row + 32, four keys of each eight in a lane,
// which is how P goes in again if V is read in that order: nothing crosses lanes
// but a raise of M and the last sums.  K's rows are read from LDS as they lie, V
// by the transposing read, which gives a lane four keys of one dim.
//
// The waves of a workgroup share the tiles of keys, which go from memory straight
// to LDS, two tiles in turn: the next one is on its way while one is computed
// with.  Pieces of 16 bytes are stored at places turned by the row, so that
// neither read meets its own banks.
//
// Rounded to fewer than 32 bits: p to V's type before it multiplies, and the
// result.  In bf16 that is off by up to 2^-8 of a weight; in fp16 by up to 2^-11 of
// it, and where p is below 2^-14, a subnormal number there, by up to 2^-25 of the
// weight at M (p below that is 0).  l is summed from the unrounded.
//
// A key that a row does not see has p = 0; so that an Inf or NaN in its V stays
// out of the sums, tiles that some row sees only part of are looked through for
// such values, and where there are any these enter by themselves, for the rows
// that see them.
//
// Rows and keys lie wherever the offsets on the device say, so every workgroup
// finds its tile of rows by itself.  Tiles that see the same keys run side by side.
//
// Bound by the softmax between the products: counters of one causal sequence of 8192
// tokens, 64/8 heads of 128, say 55% of the time in matrix instructions and 49% in vector
// ones (all keys seen: 59 and 49), at a clock that power has brought to 1.5 to 1.8 GHz by
// the card.  That is 1.02 ms (1080 TFLOP/s; a large plain product 1360 to 1560), all keys
// 1.97 ms (1117).  Heads of 64 have half the products beside the same softmax (42 and 66%,
// 0.62 ms), heads of 256 a single wave to a SIMD (29 and 30% at 4096 tokens, 0.76 ms).  16
// sequences of up to 2048, 32/32 heads of 128, 288 us; five of up to 100, 28/4 heads of
// 64, 7 us.  Reading LDS one product ahead, priorities for the waves in the products,
// and eight waves gained nothing.

#include <algorithm>
#include <type_traits>

#include "cq_elem.h"
#include "cq_step.h"

namespace cq {
namespace {

constexpr int kKeys = 64;                      // of a tile
constexpr int kRows = 32;                      // of a wave
// Two workgroups of four waves on a CU wait for their tiles and barriers apart.  (Eight
// waves read half as many tiles, and lose at the diagonal, where rows see half a tile;
// us, 4 and 8 waves: one sequence of 8192 tokens, 64/8 heads of 128, causal 1090 1113,
// all keys 1949 1925; 16 of up to 2048, 64/8: 518 598.)
constexpr int kWaves = 4;
constexpr float kNegInf = -__builtin_inff();
constexpr float kRaise = 8.f;

template <class T> struct Typed;
template <> struct Typed<_Float16> {
    using v8 = Vec<_Float16, 8>;
    static constexpr uint32_t kInf = 0x7C00;
    static __device__ __forceinline__ Vec<float, 16> mfma(v8 a, v8 b, Vec<float, 16> c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Typed<__bf16> {
    using v8 = Vec<__bf16, 8>;
    static constexpr uint32_t kInf = 0x7F80;
    static __device__ __forceinline__ Vec<float, 16> mfma(v8 a, v8 b, Vec<float, 16> c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

using u4 = Vec<uint32_t, 4>;
using f4 = Vec<float, 4>;
using f16v = Vec<float, 16>;
using s2 = Vec<short, 2>;
using s4 = Vec<short, 4>;

struct Args {
    cq_prompt_t a;
    int32_t group;        // query heads per key head
    int32_t heads;        // of a workgroup
    int32_t shift;        // log2 of a head's rows in a workgroup
    int32_t heads_apart;  // 1: neighbouring workgroups take heads of one run each
};

// f over a lane and its other half, in both.
template <class F>
__device__ __forceinline__ float half_fold(float v, F&& f) {
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return f(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// A workgroup's tile of rows, of 2^shift, and its sequence's keys.  Part p of the rows
// (those ahead of the first sequence, each sequence's, those behind the last) has the
// places from its first row / 2^shift + p on, which are as many as its tiles or one
// more.  Of few sequences each lane looks at one, of more a bisection finds a place's
// part.  The last places come first: of a sequence its last tile, which sees the most
// keys.  (Sorting the sequences by length, in a search over all of them, gained nothing
// and took 200 sequences of 40 tokens from 104 to 164 us, one head to a workgroup.)
// Offsets are cut to the tensors' rows.
struct Tile {
    int row0, rows, first;             // rows <= 0: none
    int tokens, key0, keys;            // of the sequence; none for rows of no sequence
    __device__ __forceinline__ Tile(const cq_prompt_t& a, int shift, int index, int lane) {
        const int most = (int)a.q_tokens, most_keys = (int)a.k_tokens;
        const int place = (most >> shift) + a.batch + 1 - index;
        const int32_t* k_offsets = a.k_offsets != nullptr ? a.k_offsets : a.q_offsets;
        auto begin = [&](int part) {
            return part <= 0 ? 0 : part > a.batch + 1 ? most : max(0, min(a.q_offsets[part - 1], most));
        };
        auto key = [&](int b) { return max(0, min(k_offsets[max(0, min(b, a.batch))], most_keys)); };
        int low = 0, end;
        if (a.batch + 2 < 64) {
            const int mine = begin(lane), mine_key = key(lane);
            const uint64_t here = __ballot(lane <= a.batch + 1 && (mine >> shift) + lane <= place);
            low = 63 - __builtin_clzll(here | 1);
            first = __builtin_amdgcn_readlane(mine, low);
            end = __builtin_amdgcn_readlane(mine, low + 1);
            key0 = __builtin_amdgcn_readlane(mine_key, max(low - 1, 0));
            keys = __builtin_amdgcn_readlane(mine_key, low);
        } else {
            int high = a.batch + 2;            // low: the last part that begins here or before
            while (high - low > 1) {
                const int mid = low + (high - low) / 2;
                if ((int64_t)(begin(mid) >> shift) + mid <= place) low = mid;
                else high = mid;
            }
            first = begin(low);
            end = begin(low + 1);
            key0 = key(low - 1);
            keys = key(low);
        }
        tokens = max(0, end - first);
        keys = low == 0 || low > a.batch ? 0 : max(0, keys - key0);
        row0 = (place - (first >> shift) - low) << shift;
        rows = min(1 << shift, tokens - row0);
    }
};

template <class T, int D, int W>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void prompt_kernel(Args s,
                                                                        uint32_t first_block) {
    using Ty = Typed<T>;
    using v8 = typename Ty::v8;
    constexpr int kSteps = D / 16;             // products over D
    constexpr int kDims = D / 32;              // dim tiles of O
    constexpr int kBytes = D * 2;              // of a row
    constexpr int kPieces = kBytes / 16;       // 16 bytes of a row
    constexpr int kLoadRows = 64 / kPieces;    // rows of a wave's load
    constexpr int kLoads = kKeys / kLoadRows / W;      // of a wave, for K (and for V)
    constexpr int kTileBytes = kKeys * kBytes;
    static_assert(kLoads * kLoadRows * W == kKeys, "whole loads");
    __shared__ __attribute__((aligned(1024))) uint8_t sm[4 * kTileBytes];     // K, V; twice
    const cq_prompt_t& a = s.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t block = first_block + blockIdx.x;
    // the workgroup's heads (of one key head) and each one's rows
    const uint32_t runs = (uint32_t)(a.q_heads / s.heads), place = block % runs;
    const int waves = W / s.heads;             // of a head
    const int h0 = (s.heads_apart ? (int)(place % 8 * (runs / 8) + place / 8) : (int)place) * s.heads;
    const int h = h0 + wave / waves;
    const Tile tile(a, s.shift, (int)(block / runs), lane);
    if (tile.rows <= 0) return;
    const int row0 = kRows * (wave % waves);   // of the tile
    T* out = static_cast<T*>(a.out) + ((int64_t)(tile.first + tile.row0) * a.q_heads + h) * D;
    const int64_t out_row = (int64_t)a.q_heads * D;
    // keys that row r of the tile sees
    auto limit_of = [&](int r) {
        if (!a.causal) return tile.keys;
        const int64_t n = (int64_t)tile.keys - tile.tokens + tile.row0 + r + 1;
        return (int)max((int64_t)0, min(n, (int64_t)tile.keys));
    };
    const int reach = limit_of(tile.rows - 1);         // of the workgroup
    if (reach == 0) {                          // no keys: zeros
        for (int i = threadIdx.x % (64 * waves); i < tile.rows * kPieces; i += 64 * waves)
            *reinterpret_cast<u4*>(out + i / kPieces * out_row + i % kPieces * 8) = u4{0, 0, 0, 0};
        return;
    }
    const bool live = row0 < tile.rows;
    const int r = min(row0 + col, tile.rows - 1);      // rows past the last repeat it
    const int limit = limit_of(r);
    const int full = limit_of(min(row0, tile.rows - 1));       // every row of the wave sees
    const int wave_reach = live ? limit_of(min(row0 + kRows, tile.rows) - 1) : 0;

    // the tiles of keys
    const int64_t k_row = a.k_token_stride * 2, v_row = a.v_token_stride * 2;      // bytes
    const uint8_t* kp = static_cast<const uint8_t*>(a.k) + tile.key0 * k_row +
                        (int64_t)(h / s.group) * a.k_head_stride * 2;
    const uint8_t* vp = static_cast<const uint8_t*>(a.v) + tile.key0 * v_row +
                        (int64_t)(h / s.group) * a.v_head_stride * 2;
    // where a row's pieces are turned to: K's reads take one piece of 16 rows, V's
    // four pieces of four rows
    auto k_turn = [](int row) { return D == 64 ? row >> 1 & 7 : row & 15; };
    auto v_turn = [](int row) { return D == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2; };
    int k_at[kLoads], v_at[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int row = (wave + W * i) * kLoadRows + lane / kPieces, piece = lane % kPieces;
        k_at[i] = row * (int)k_row + (piece ^ k_turn(row)) * 16;
        v_at[i] = row * (int)v_row + (piece ^ v_turn(row)) * 16;
    }
    auto fetch = [&](int t, int buf) {
        const int rows = min(kKeys, reach - t * kKeys);        // past them zeros come
        const uint8_t* kt = kp + t * (kKeys * k_row);
        const uint8_t* vt = vp + t * (kKeys * v_row);
        const int k_bytes = (int)((rows - 1) * k_row) + kBytes;
        const int v_bytes = (int)((rows - 1) * v_row) + kBytes;
        uint8_t* to = sm + buf * 2 * kTileBytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            load_to_lds(to + (wave + W * i) * 1024, kt, k_bytes, k_at[i]);
            load_to_lds(to + kTileBytes + (wave + W * i) * 1024, vt, v_bytes, v_at[i]);
        }
    };
    fetch(0, 0);

    // the queries; a negative scale goes into their signs, one of 0 into them whole
    v8 q[kSteps];
    {
        const T* p = static_cast<const T*>(a.q) +
                     (int64_t)(tile.first + tile.row0 + r) * a.q_token_stride +
                     (int64_t)h * a.q_head_stride + half * 8;
        const uint32_t turn = a.softmax_scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            u4 w = *reinterpret_cast<const u4*>(p + u * 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] ^= turn;
            q[u] = __builtin_bit_cast(v8, w);
            if (a.softmax_scale == 0.f) q[u] *= (T)0.f;
        }
    }
    const float by =
        a.softmax_scale == 0.f ? 1.f : fabsf(a.softmax_scale) * 1.4426950408889634f;
    f16v o[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i) o[i] = f16v{};
    float ref = 0.f, raise = kNegInf;                  // ref: M
    f4 sums = {0.f, 0.f, 0.f, 0.f};

    constexpr uint32_t kOver = (0x8000u - Ty::kInf) * 0x10001u;
    // A tile of keys.  MASKED: rows may see a part of it, or nothing.
    auto advance = [&](int t, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const int key0 = t * kKeys;
        const uint8_t* ks = sm + (t & 1) * 2 * kTileBytes;
        const uint8_t* vs = ks + kTileBytes;
        f16v x[2] = {f16v{}, f16v{}};
#pragma unroll
        for (int u = 0; u < kSteps; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = i * 32 + col;
                const v8 k = *reinterpret_cast<const v8*>(
                    ks + row * kBytes + ((u * 2 + half) ^ k_turn(row)) * 16);
                x[i] = Ty::mfma(k, q[u], x[i]);
            }
        // key of x[i][j]: key0 + 32 i + 8 (j / 4) + 4 half + j % 4
        const int mine = limit - key0 - 4 * half;
        auto sees = [&](int i, int j) { return 32 * i + 8 * (j / 4) + j % 4 < mine; };
        float top = kNegInf;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (MASKED && !sees(i, j)) x[i][j] = kNegInf;
                top = fmaxf(top, x[i][j]);
            }
        if (__any(__builtin_fmaf(top, by, -ref) > raise)) {
            top = half_fold(top, [](float m, float n) { return fmaxf(m, n); }) * by;
            const bool first = raise == kNegInf;
            if (top - ref > (first ? kNegInf : 0.f)) {
                const float keep = first ? 1.f : __builtin_amdgcn_exp2f(ref - top);
                ref = top;
                raise = kRaise;
                sums *= keep;
#pragma unroll
                for (int i = 0; i < kDims; ++i) o[i] *= keep;
            }
        }
        v8 p[4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][j], by, -ref));
                x[i][j] = e;
                sums[j % 4] += e;
                p[2 * i + j / 8][j % 8] = (T)e;
            }
        // V's part of step s and dim tile d: keys 16 s + 4 half + 0..3 and 8 more
        auto read_v = [&](int s, int d) {
            const int row = 16 * s + 4 * half + (lane >> 2 & 3);
            const int piece = 4 * d + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
            const uint8_t* at = vs + row * kBytes + (piece ^ v_turn(row)) * 16 + (lane & 1) * 8;
            auto read = [&](const uint8_t* from) {
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s4*)from);
            };
            const s4 lo = read(at), hi = read(at + 8 * kBytes);      // (the same turn)
            return __builtin_bit_cast(u4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // whether a masked key's V may spoil the sums
        bool spoilt = false;
        if constexpr (MASKED) {
            uint32_t over = 0;
            for (int i = lane; i < kTileBytes / 16; i += 64) {
                const u4 w = *reinterpret_cast<const u4*>(vs + i * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) over |= (w[j] & 0x7FFF7FFFu) + kOver;
            }
            spoilt = __any((over & 0x80008000u) != 0);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                u4 w = read_v(s, d);
                if constexpr (MASKED) {
                    if (spoilt) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const s2 bad =
                                __builtin_bit_cast(s2, (w[i] & 0x7FFF7FFFu) + kOver) >> 15;
                            w[i] &= ~__builtin_bit_cast(uint32_t, bad);
                        }
                    }
                }
                o[d] = Ty::mfma(__builtin_bit_cast(v8, w), p[s], o[d]);
            }
        if constexpr (MASKED) {
            // Inf and NaN, key by key
            for (int key = 0; spoilt && key < kKeys; ++key) {
                float e = 0.f;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        e = 32 * i + 8 * (j / 4) + 4 * half + j % 4 == key ? x[i][j] : e;
                e = half_fold(e, [](float m, float n) { return m + n; });
                const bool seen = key < limit - key0;
#pragma unroll
                for (int d = 0; d < kDims; ++d)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const int dim = 32 * d + 2 * j + 4 * half;
                        const Vec<uint32_t, 2> w = *reinterpret_cast<const Vec<uint32_t, 2>*>(
                            vs + key * kBytes + ((dim / 8) ^ v_turn(key)) * 16 + half * 8);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint16_t bits = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
                            const float v = (float)__builtin_bit_cast(T, bits);
                            if (seen && (bits & 0x7FFF) >= Ty::kInf) o[d][j + i] += e * v;
                        }
                    }
            }
        }
    };
    // tiles that every row of the workgroup sees all of, then the others
    const int tiles = (reach + kKeys - 1) / kKeys, whole = limit_of(0) / kKeys;
    auto next = [&](int t) {
        // this wave's loads of tile t have come and its reads of t - 1 are done, then
        // everybody's (a barrier alone waits for neither: a wave that has no keys in
        // t - 1 has not looked at any)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + 1 < tiles) fetch(t + 1, (t + 1) & 1);
    };
    int t = 0;
    for (; t < whole; ++t) {
        next(t);
        advance(t, std::false_type{});
    }
    for (; t < tiles; ++t) {
        next(t);
        // (heads of 256 have no registers for a third form)
        if (D < 256 && t * kKeys + kKeys <= full)
            advance(t, std::false_type{});
        else if (t * kKeys < wave_reach)
            advance(t, std::true_type{});
    }
    if (!live) return;
    const float sum = half_fold((sums[0] + sums[1]) + (sums[2] + sums[3]),
                                [](float m, float n) { return m + n; });
    const float share = sum == 0.f ? 0.f : 1.f / sum;
    // the halves of the wave change fours of dims, so that a lane has eight side by side
    T* to = out + (int64_t)(row0 + col) * out_row + 8 * half;
    const bool there = row0 + col < tile.rows;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
            using u2 = Vec<uint32_t, 2>;
            Vec<T, 4> v[2];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i / 4][i % 4] = (T)(sum == 0.f ? 0.f : o[d][j + i] * share);
            u2 x = __builtin_bit_cast(u2, v[0]), y = __builtin_bit_cast(u2, v[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t p = x[i], q = y[i];
                swap_halves(p, q);
                x[i] = p;
                y[i] = q;
            }
            if (there) *reinterpret_cast<u4*>(to + 32 * d + 2 * j) = u4{x[0], x[1], y[0], y[1]};
        }
}

// ------------------------------------------------------------------- host
template <class T, int D>
hipError_t launch_typed(const Args& s, hipStream_t stream) {
    const cq_prompt_t& a = s.a;
    // every sequence's last tile may be a part of one, and so those of the rows
    // that belong to none
    const int64_t tiles = a.q_tokens / (kRows * kWaves / s.heads) + a.batch + 2;
    const __int128 grid = (__int128)tiles * (a.q_heads / s.heads);
    if (grid > kMaxGrid) return hipErrorInvalidValue;
    return launch_parts((int64_t)grid, [&](dim3 blocks, uint32_t first) {
        prompt_kernel<T, D, kWaves><<<blocks, dim3(64 * kWaves), 0, stream>>>(s, first);
    });
}

template <class T>
hipError_t launch_head(const Args& s, hipStream_t stream) {
    if (s.a.head_dim == 64) return launch_typed<T, 64>(s, stream);
    if (s.a.head_dim == 128) return launch_typed<T, 128>(s, stream);
    return launch_typed<T, 256>(s, stream);
}

}  // namespace

hipError_t launch_prompt(const cq_prompt_t& a, hipStream_t stream) {
    Args s{};
    s.a = a;
    s.group = a.q_heads / a.k_heads;
    // where sequences are short of a workgroup's 128 rows, two or four heads of a key
    // head share it (200 sequences of 40 tokens, 32/8 heads of 128, us: one head 98, two
    // 66; of 20 tokens: one 92, four 37; heads without groups have no such form, and 32/32
    // heads take 103 and 95)
    const int64_t rows = a.q_tokens / a.batch;
    s.heads = rows <= 32 && s.group % 4 == 0 ? 4 : rows <= 64 && s.group % 2 == 0 ? 2 : 1;
    s.shift = __builtin_ctz((unsigned)(kRows * kWaves / s.heads));
    s.heads_apart = a.q_heads / s.heads % 8 == 0;
    return a.dtype == CQ_DTYPE_F16 ? launch_head<_Float16>(s, stream)
                                   : launch_head<__bf16>(s, stream);
}

}  // namespace cq
