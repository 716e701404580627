// Attention over the quantized paged key/value cache (gfx950).
//
//   s_j = scale * (q . kcode_j) * kscale_j, p = softmax(s) over what the row
//   sees, out_d = sum_j p_j * vscale_j * vcode_jd
//
// One pass over the keys with a running reference M and sum l: with
// vscale_j = f_j 2^e_j (f in [1/2, 1)) a wave keeps
//   l = sum_j 2^(s_j log2(e) - M),  o_d = sum_j w_j vcode_jd,
//   w_j = 2^(s_j log2(e) + e_j - M) f_j
// and raises M (scaling l and o down) when an exponent passes kRaise; triples
// (M, l, o) of disjoint keys join the same way.  Folding V's exponent into
// that of the softmax keeps w_j, which the matrix instructions take as fp16,
// in range: the largest w of a row lies in [2^-5, 2^kRaise), and what fp16 then
// rounds off is 2^-11 of each weight, or 2^-25 of 1.  Scores, statistics and
// sums are FP32; the weights' rounding is the one beside the result's (q's,
// below, is far under both).
//
// A key counts in l whatever its V scale, so l's term 2^(s_j log2(e) - M) is
// 2^-e_j times the exponential that w_j takes, and that must stay inside FP32's
// exponents.  So e_j is taken no lower than kSpan below the largest that the wave
// has met (a scale of zero has no exponent of its own, and smaller ones only a
// smaller f): keys down to 2^-56 of the row's largest probability are counted, and
// scales down to 2^-80 of the largest seen keep their digits.  l itself, a raise
// or a join may move by more than one exponential holds; it is scaled in two.
//
// A code of K goes into the matrix units as the fp16 subnormal
// (code + 2^(bits-1)) 2^-24, which is the code's bits with the sign bit turned
// and nothing else: one operation for two codes.  What the offset adds to a
// score is the same for every key of a row, so the score sums start at minus
// that.  V's codes go in as they are: there a common offset would cost digits
// where a key of large weight has small codes.  q is brought to fp16 times a
// power of two, the row's own, that puts its largest finite element into
// [2^13, 2^14): rows share waves with other heads, tokens and sequences, and
// with rows past the counts, whose numbers may be any.
//
// Matrix form, 64 keys at a time (v_mfma_f32_16x16x32_f16, FP32 sums):
//   S^T [keys x rows] = K [keys x D] Q^T [D x rows]
//   O^T [D x rows]   += V^T [D x keys] W^T [keys x rows]
// Rows are the query heads of a key head (times the new tokens), 16 to a
// matrix.  S comes out with a row's keys in the four lanes row + 16 g, four
// keys of each matrix in a lane, which is just how W goes in if lane group g
// owns keys 16 g .. 16 g + 15 of the 64: K's rows are loaded in that order, V
// is stored with 16 tokens of a dim together, and nothing crosses lanes but a
// raise of M and the last sums.  Both operands are loaded once from memory as
// codes, 16 bytes to a lane, and turned into fp16 in registers.
//
// Work is dealt out on the device, where the lengths are: the (sequence, row
// group, head) units are laid end to end as tiles of 64 keys, and each
// workgroup takes an equal run of tiles, wherever units begin and end.  A unit
// that lies in one run is finished there; a longer one leaves a triple per run
// in the workspace, which join_kernel joins.  Equal runs keep every workgroup
// busy to the end for any mix of lengths, and the grid never depends on them.
// Where whole units to a run are as even, they are dealt whole: 1024 new tokens
// of 64 heads over 8700 keys then leave nothing to join (399 us, whole 348).
//
// Three kernels:
//   tile_kernel   few rows (shape_of): a wave takes whole tiles, four waves
//                 every fourth, joined in LDS.  Bound by memory: 64 sequences
//                 of up to 16384 keys of 8 heads (int8, 1.14 GB) 196 us, 5.8
//                 TB/s.  A short call is bound by waits that follow one another
//                 (lengths, table, codes, the join).
//   block_kernel  more rows: four or eight waves of 32 rows share tiles that
//                 the workgroup unpacks into LDS once.  Bound by the matrix
//                 units and the softmax between their products: 1024 new tokens
//                 of 64 heads over 8700 keys (int4) 341 us, 805 TFLOP/s; a
//                 prefix of 16384 keys for 64 sequences of 64 heads 87 us, of
//                 which 40 are tiles (2.5 us each of 64 keys and 256 rows), 8
//                 the join of 16 triples to a row, the rest the sequences' own
//                 keys and starts and ends of units.
//   join_kernel   joins triples; one token over 4096 keys of 8 heads 3.9 us.

#include <algorithm>
#include <utility>

#include "cq_attn.h"
#include "cq_elem.h"

namespace cq {
namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kTile = 64;               // keys of a tile
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.f;
constexpr int kSpan = 70;               // of the exponents of V's scales
constexpr int kLeastExp = -96;          // 2^23 terms of l of 2^(96 + kRaise) fit FP32
constexpr int kMostExp = 122;           // of the largest numbers' scales; also Inf's, NaN's
constexpr int kEven = 4;

using h8 = Vec<_Float16, 8>;
using h2 = Vec<_Float16, 2>;
using f4 = Vec<float, 4>;
using u4 = Vec<uint32_t, 4>;

// One launch over one source of keys (the sequences' own, or the prefix).
struct Source {
    cq_kv_cache_t c;
    cq_attention_t a;
    int32_t group;         // query heads per key head
    int32_t rows;          // rows of a unit's sequence (or of the whole batch)
    int32_t row_groups;    // of rows_per_unit rows
    int32_t rows_per_unit;
    int32_t prefix;        // 1: the prefix's keys
    int32_t page_shift;    // log2 of the page size
    int32_t quantum;       // a run's length is a multiple of it
    int32_t cost;          // of a unit besides its tiles, in tiles
    uint32_t runs;         // workgroups
    int32_t fits;          // the deal's sums, keys and rows fit 31 bits
    int32_t finish;        // 1: units of one run write `out`; 0: their home
    // workspace: which runs have a unit's triples (first run and how many; none
    // for a unit without keys); triples of broken units, two per run, and of
    // whole units
    uint32_t* where;       // [entries * heads, 2]
    // runs * 2 * rows_per_unit of broken units from row `broken`, batch *
    // tokens * q_heads of whole ones from row `home` of both arrays
    float* o;              // [.., D]
    float* ml;             // [.., 2]
    int64_t broken, home;
};

// ------------------------------------------------- over a wave
// Maximum and sum over the four lanes l, l + 16, l + 32, l + 48, in each.
template <class F>
__device__ __forceinline__ float quad_fold(float v, F&& f) {
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t y = __float_as_uint(v);
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_max(float v) {
    return quad_fold(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float quad_sum(float v) {
    return quad_fold(v, [](float a, float b) { return a + b; });
}
// f over the 16 lanes of a row, in each.
template <class F>
__device__ __forceinline__ int row_fold(int v, F&& f) {
    v = f(v, (int)row_dpp<0x128>((uint32_t)v));
    v = f(v, (int)row_dpp<0x124>((uint32_t)v));
    v = f(v, (int)row_dpp<0x122>((uint32_t)v));
    return f(v, (int)row_dpp<0x121>((uint32_t)v));
}
__device__ __forceinline__ int row_min(int v) {
    return row_fold(v, [](int a, int b) { return min(a, b); });
}
__device__ __forceinline__ int row_max(int v) {
    return row_fold(v, [](int a, int b) { return max(a, b); });
}
// Maximum over the wave, for the scalar unit.
__device__ __forceinline__ int wave_most(int v) {
    v = row_max(v);
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, row_dpp<0x128>(v));
    v = fmaxf(v, row_dpp<0x124>(v));
    v = fmaxf(v, row_dpp<0x122>(v));
    v = fmaxf(v, row_dpp<0x121>(v));
    return quad_max(v);
}

// -------------------------------------------------------------- the units
__device__ __forceinline__ int new_tokens(const cq_attention_t& a, int b) {
    return a.counts != nullptr ? max(0, min(a.tokens, a.counts[b])) : a.tokens;
}

// Own positions that query t of sequence b sees (0 for t past the count).
__device__ __forceinline__ int own_limit(const Source& s, int length, int count, int t) {
    if (t >= count) return 0;
    const int64_t last = (int64_t)length - count + t + 1;
    return (int)max((int64_t)0, min(last, (int64_t)s.a.table_cols * s.c.page_size));
}

// Tiles of entry e: (sequence, row group), or the prefix's row group.
__device__ __forceinline__ int tiles_of(const Source& s, int e) {
    if (s.prefix) return (s.a.prefix_len + kTile - 1) / kTile;
    int b = e, last = s.a.tokens - 1, first = 0;
    if (s.row_groups > 1) {
        b = e / s.row_groups;
        const int row = (e - b * s.row_groups) * s.rows_per_unit;
        first = row / s.group;
        last = min(last, (row + s.rows_per_unit - 1) / s.group);
    }
    const int count = new_tokens(s.a, b);
    if (first >= count) return 0;
    return (own_limit(s, s.a.lengths[b], count, min(last, count - 1)) + kTile - 1) / kTile;
}

__device__ __forceinline__ int entries_of(const Source& s) {
    return s.prefix ? s.row_groups : s.a.batch * s.row_groups;
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {     // inclusive
    v += row_dpp<0x111>(v);                                     // row_shr 1, 2, 4, 8
    v += row_dpp<0x112>(v);
    v += row_dpp<0x114>(v);
    v += row_dpp<0x118>(v);
    // the last lane of a row to the rows behind it
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}

// A unit's place in the deal: as many steps as its tiles, rounded up to the
// quantum, and its cost.
__device__ __forceinline__ int steps_of(const Source& s, int tiles) {
    if (tiles == 0) return 0;
    return (tiles + s.quantum - 1) / s.quantum * s.quantum + s.cost;
}

// Entries base .. base + 63, one to a lane: tiles, steps, and the steps up to
// and with the lane's, of one head.
struct Entries {
    int base, tiles;
    uint32_t steps, upto;
    __device__ __forceinline__ Entries(const Source& s, int at, int lane) : base(at) {
        tiles = at + lane < entries_of(s) ? tiles_of(s, at + lane) : 0;
        steps = steps_of(s, tiles);
        upto = wave_scan(steps);
    }
    __device__ __forceinline__ void count_units() {
        steps = tiles > 0;
        upto = wave_scan(steps);
    }
    __device__ __forceinline__ uint32_t all() const { return __builtin_amdgcn_readlane(upto, 63); }
};

// How a source's units are dealt to the runs: in equal numbers of steps, or,
// where that leaves hardly more to the longest run, in whole units: those need
// no joining.  (The host sees to it that the steps of all heads stay below 2^31.)
struct Deal {
    bool whole;
    uint32_t all;      // steps or units of all heads
    uint32_t per;      // of a run
};

// `at`: entries 0 .. 63; afterwards counts units if those are dealt.
__device__ __forceinline__ Deal deal(const Source& s, Entries& at, int lane) {
    const uint32_t heads = s.c.heads;
    uint32_t steps = 0, units = 0, most = 0;
    for (int base = 0;;) {
        const Entries e = base == 0 ? at : Entries(s, base, lane);
        steps += e.all();
        units += __builtin_popcountll(__ballot(e.tiles > 0));
        most = max(most, (uint32_t)__builtin_amdgcn_readfirstlane((int)wave_max((float)e.steps)));
        // units without keys are no run's: any workgroup notes them
        if (threadIdx.x < 64 && base + lane < entries_of(s) && e.tiles == 0 &&
            (uint32_t)(base + lane) % s.runs == blockIdx.x)
            for (uint32_t h = 0; h < heads; ++h) s.where[((base + lane) * heads + h) * 2 + 1] = 0;
        base += 64;
        if (base >= entries_of(s)) break;
    }
    Deal d;
    const uint32_t q = s.quantum;
    d.all = steps * heads;
    d.per = (max(1u, (d.all + s.runs - 1) / s.runs) + q - 1) / q * q;
    const uint32_t each = (units * heads + s.runs - 1) / s.runs;
    d.whole = each * most <= d.per + d.per / 8;
    if (d.whole) {
        d.all = units * heads;
        d.per = max(1u, each);
        at.count_units();
    }
    return d;
}

// ----------------------------------------------------------- small pieces
// K's codes of a word as fp16 pairs, offset and in units of 2^-24: bytes (0, 2),
// (1, 3) of int8; of int4 the low and high nibbles of bytes (0, 2) and of
// (1, 3), the high ones 16 times what they stand for.
__device__ __forceinline__ void halves_of_bytes(uint32_t w, uint32_t& a, uint32_t& b) {
    a = (w & 0x00FF00FFu) ^ 0x00800080u;
    b = ((w >> 8) & 0x00FF00FFu) ^ 0x00800080u;
}
__device__ __forceinline__ void halves_of_nibbles(uint32_t w, uint32_t (&p)[4]) {
    const uint32_t x = w >> 8;
    p[0] = (w & 0x000F000Fu) ^ 0x00080008u;
    p[1] = (w & 0x00F000F0u) ^ 0x00800080u;
    p[2] = (x & 0x000F000Fu) ^ 0x00080008u;
    p[3] = (x & 0x00F000F0u) ^ 0x00800080u;
}

// V's codes as fp16 pairs in the same order: under the exponent of 1024 (of 64
// for a high nibble, whose last bits are then sixteenths), less the offset.
__device__ __forceinline__ uint32_t less(uint32_t a, float b) {
    const h2 v = __builtin_bit_cast(h2, a) - h2{(_Float16)b, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ void codes_of_bytes(uint32_t w, uint32_t& a, uint32_t& b) {
    a = less((w & 0x00FF00FFu) ^ 0x64806480u, 1152.f);
    b = less(((w >> 8) & 0x00FF00FFu) ^ 0x64806480u, 1152.f);
}
__device__ __forceinline__ void codes_of_nibbles(uint32_t w, uint32_t (&p)[4]) {
    const uint32_t x = w >> 8;
    p[0] = less((w & 0x000F000Fu) ^ 0x64086408u, 1032.f);
    p[1] = less((w & 0x00F000F0u) ^ 0x54805480u, 72.f);
    p[2] = less((x & 0x000F000Fu) ^ 0x64086408u, 1032.f);
    p[3] = less((x & 0x00F000F0u) ^ 0x54805480u, 72.f);
}

// The root of what a triple's sums are multiplied with to stand at reference
// `top`: l is large where V's scales are small, so it may be in range there
// though 2^(m - top) is not.  One that has seen no number has M = -Inf and sums
// of 0, or of NaN where it saw only NaN: l itself then.
__device__ __forceinline__ float root(float m, float l, float top) {
    return m == kNegInf ? l : __builtin_amdgcn_exp2f(0.5f * (m - top));
}

template <class T>
__device__ __forceinline__ void store4(T* p, f4 v) {
    Vec<T, 4> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
    *reinterpret_cast<Vec<T, 4>*>(p) = o;
}

// Lane J of each row of 16 lanes, to the whole row (an operand of the
// instruction that takes it, not one of its own).
template <int J>
__device__ __forceinline__ float of_lane(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0x150 + J,
                                                              0xF, 0xF, true));
}
template <class F, int... J>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, J...>) {
    (f(std::integral_constant<int, J>{}), ...);
}
// f(integral_constant 0), ..., f(integral_constant 15)
template <class F>
__device__ __forceinline__ void sixteen(F&& f) {
    each_of(f, std::make_integer_sequence<int, 16>{});
}

// --------------------------------------------------------------- the rows
// Row r of a unit's source: its sequence, new token and query head.
struct RowAt {
    int b, t, hq;
    __device__ __forceinline__ RowAt(const Source& s, int unit_b, int r, int h)
        : b(unit_b), t(0), hq(h * s.group + r) {
        if (s.prefix || s.a.tokens > 1) {
            const int all = r / s.group;
            hq = h * s.group + r - all * s.group;
            t = all;
            if (s.prefix) {
                b = all / s.a.tokens;
                t = all - b * s.a.tokens;
            }
        }
    }
    __device__ __forceinline__ int64_t flat(const Source& s) const {
        return ((int64_t)b * s.a.tokens + t) * s.a.q_heads + hq;
    }
};

// The unpacking of a word leaves pairs of bytes or nibbles apart: code order(i)
// of eight comes i-th.
template <int BITS>
constexpr int order(int i) {
    constexpr int o8[8] = {0, 2, 1, 3, 4, 6, 5, 7};
    constexpr int o4[8] = {0, 4, 1, 5, 2, 6, 3, 7};
    return BITS == 8 ? o8[i] : o4[i];
}

using ss2 = Vec<short, 2>;
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
    using us2 = Vec<unsigned short, 2>;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, a),
                                                                  __builtin_bit_cast(us2, b)));
}

// The state of a wave's 16 NB rows: queries, sums and references.  RAW: the
// score products take K's codes as they lie in memory, offset and in units
// (halves_of_*); else the codes themselves.
template <class T, int BITS, int D, int NB, bool RAW>
struct Rows {
    // (the short form for even scales is worth its code to many rows only)
    static constexpr bool kShort = !RAW;
    static constexpr int kSteps = D / 32;                  // products over D
    static constexpr int kOTiles = D / 16;
    static constexpr float kOffset = BITS == 8 ? 128.f : 8.f;
    static constexpr float kUnit = 0x1p-24f;
    // 1 / kUnit, half of it in K's scale and half in q's: neither leaves FP32's
    // range by it
    static constexpr float kHalfUnit = RAW ? 0x1p12f : 1.f;
    static constexpr uint32_t kInf = std::is_same_v<T, _Float16> ? 0x7C00u : 0x7F80u;

    h8 q[NB][kSteps];
    float start[NB];                     // what the score sums start at
    float qscale[NB];                    // of a score sum: scale log2(e), units, q's factor
    int limit[NB];                       // keys that the lane's row sees
    int full;                            // tiles of which every row sees all
    int reach;                           // keys that some row sees
    int largest;                         // exponent of V's scales met so far
    f4 o[NB][kOTiles];
    float l[NB], ref[NB], raise[NB];

    // dim(u): where the eight dims of step u that this lane multiplies start.
    template <class Dim>
    __device__ __forceinline__ void load(const Source& s, int b, int first_row, int h, int lane,
                                         Dim&& dim) {
        int least = 0x7FFFFFFF, most = 0;
        Vec<T, 8> raw[NB][kSteps];
        uint32_t top2[NB] = {};
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            // rows past the last repeat it (nobody stores them)
            const int r = min(first_row + 16 * rb + (lane & 15), s.rows - 1);
            const RowAt at(s, b, r, h);
            const int count = new_tokens(s.a, at.b);
            limit[rb] = s.prefix ? (at.t < count ? s.a.prefix_len : 0)
                                 : own_limit(s, s.a.lengths[at.b], count, at.t);
            least = min(least, limit[rb]);
            most = max(most, limit[rb]);
            const T* p = static_cast<const T*>(s.a.q) + at.b * s.a.q_batch_stride +
                         at.t * s.a.q_token_stride + at.hq * s.a.q_head_stride;
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
                raw[rb][u] = *reinterpret_cast<const Vec<T, 8>*>(p + dim(u));
                const u4 w = __builtin_bit_cast(u4, raw[rb][u]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // magnitudes, 0 for Inf and NaN: their sum with 2^15 - Inf
                    // is negative in 16 bits
                    const uint32_t m = w[i] & 0x7FFF7FFFu;
                    const ss2 bad = __builtin_bit_cast(ss2, m + (0x8000u - kInf) * 0x10001u) >> 15;
                    top2[rb] = pk_max(top2[rb], m & ~__builtin_bit_cast(uint32_t, bad));
                }
            }
        }
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            // exact down to 2^-23 of the row's largest element, to 2^-34 of it
            // below (2^4 more without the nibbles' 16): less than FP32 rounds off
            const uint32_t bits = max(top2[rb] & 0xFFFFu, top2[rb] >> 16);
            const float top =
                quad_max((float)__builtin_bit_cast(T, static_cast<unsigned short>(bits)));
            const int e = top > 0.f ? __builtin_amdgcn_frexp_expf(top) - 14 : 0;
            qscale[rb] = ldexpf(s.a.softmax_scale * kLog2e * kHalfUnit, e);
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < kSteps; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    // raw high nibbles come as 16 times their code
                    const int down = RAW && BITS == 4 && (order<BITS>(i) & 1) ? 4 : 0;
                    q[rb][u][i] = (_Float16)ldexpf((float)raw[rb][u][order<BITS>(i)], -e - down);
                    if (RAW) sum = __builtin_fmaf((float)q[rb][u][i], down ? 16.f : 1.f, sum);
                }
            start[rb] = RAW ? -kOffset * kUnit * quad_sum(sum) : 0.f;
        }
        full = __builtin_amdgcn_readfirstlane(row_min(least)) / kTile;
        reach = __builtin_amdgcn_readfirstlane(row_max(most));
        largest = kLeastExp;
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            l[rb] = ref[rb] = 0.f;
            raise[rb] = kNegInf;
#pragma unroll
            for (int i = 0; i < kOTiles; ++i) o[rb][i] = f4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // From a tile's score sums to its weights w, raising the references and
    // adding to l.  sc[.][t][i] is the lane's row against key 16 g + 4 t + i of
    // the tile (lane group g = lane / 16); ks, vs are the scales of key `lane`,
    // `there` whether the group's keys have a page.  Each lane prepares one key
    // for the 16 lanes of its row, whose keys these are: K's scale, V's as f 2^e.
    //
    // Where every row sees every key and V's scales lie within 2^kEven of the
    // largest, e is the tile's largest instead: the weight of the key with the
    // largest p is then 2^-kEven at least, well inside fp16, and e and 2^-e are
    // one addition for 16 keys instead of two operations for each.
    __device__ __forceinline__ void weights(const f4 (&sc)[NB][4], float ks, float vs, bool there,
                                            int tile, int lane, h8 (&w)[NB][2]) {
        // (a branch around the maximum costs the products their schedule: 1024
        // new tokens 351 us with it, 341 without)
        const int own = (int)((__float_as_uint(vs) >> 23) & 0xFF) - 126;
        const bool met = there && tile * kTile + lane < reach && own <= kMostExp;
        const int most = wave_most(met ? own : kLeastExp);
        largest = max(largest, most);
        const int least = max(largest - kSpan, kLeastExp);
        const bool even = kShort && tile < full && __all(met && own >= most - kEven);
        const int e = even ? max(most, least) : min(max(own, least), kMostExp);
        const float kf = ks * kHalfUnit, ef = (float)e, vf = __builtin_amdgcn_ldexpf(vs, -e);
        const float back = __builtin_amdgcn_ldexpf(1.f, -e);
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            float kfs[16];
            sixteen([&](auto j) { kfs[j] = of_lane<j>(kf) * qscale[rb]; });
            // keys of the lane's 16 that its row sees
            const int n = there ? limit[rb] - tile * kTile - (lane & 48) : 0;
            float x[16];
            if (even) {
                const float t = ef - ref[rb];
                sixteen([&](auto j) {
                    x[j] = __builtin_fmaf(kfs[j], sc[rb][j / 4][j % 4], t);
                });
            } else {
                sixteen([&](auto j) {
                    const float t = of_lane<j>(ef) - ref[rb];
                    x[j] = __builtin_fmaf(kfs[j], sc[rb][j / 4][j % 4], t);
                    x[j] = j < n ? x[j] : kNegInf;
                });
            }
            float top = kNegInf;
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, x[j]);
            if (__any(top > raise[rb])) {
                top = quad_max(top);
                const bool first = raise[rb] == kNegInf;
                if (top > (first ? kNegInf : 0.f)) {
                    const float half = first ? 1.f : __builtin_amdgcn_exp2f(-0.5f * top);
                    const float keep = half * half;
                    ref[rb] += top;
                    raise[rb] = kRaise;
                    l[rb] = l[rb] * half * half;
#pragma unroll
                    for (int i = 0; i < kOTiles; ++i) o[rb][i] *= keep;
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] -= top;
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = __builtin_amdgcn_exp2f(x[j]);
            if (even) {
                float sum = 0.f;
                sixteen([&](auto j) {
                    sum += x[j];
                    x[j] = of_lane<j>(vf) * x[j];
                });
                l[rb] = __builtin_fmaf(sum, back, l[rb]);
            } else {
                sixteen([&](auto j) {
                    l[rb] = __builtin_fmaf(of_lane<j>(back), x[j], l[rb]);
                    // what is not seen may have a scale of NaN or Inf
                    const float p = of_lane<j>(vf) * x[j];
                    x[j] = j < n ? p : 0.f;
                });
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) w[rb][u][i] = (_Float16)x[8 * u + order<8>(i)];
        }
    }

    __device__ __forceinline__ float reference(int rb) const {
        return raise[rb] == kNegInf ? kNegInf : ref[rb];
    }

    // f(dim, four values): the lane's part of the sums of row matrix rb, four
    // dims a call.  Dims of o[.][i] are four from 16 i + 4 g, or (4 bits) every
    // other of eight from 32 (i / 2) + 8 g.
    template <class F>
    __device__ __forceinline__ void each_four(int rb, int lane, F&& f) const {
        const int g = lane >> 4;
        if constexpr (BITS == 8) {
#pragma unroll
            for (int i = 0; i < kOTiles; ++i) f(16 * i + 4 * g, o[rb][i]);
        } else {
#pragma unroll
            for (int i = 0; i < kOTiles; i += 2) {
                const f4 a = o[rb][i], b = o[rb][i + 1];
                f(16 * i + 8 * g, f4{a[0], b[0], a[1], b[1]});
                f(16 * i + 8 * g + 4, f4{a[2], b[2], a[3], b[3]});
            }
        }
    }
};

// ------------------------------------------------------- a run of a kernel
// A run's way through its units: part(e, b, h, row0, tile, end, n) for each
// part of a unit, tiles [tile, end) of its n.
template <class Part>
__device__ __forceinline__ void walk_run(const Source& s, int lane, Part&& part) {
    Entries at(s, 0, lane);
    const Deal d = deal(s, at, lane);
    uint32_t pos = blockIdx.x * d.per;
    const uint32_t stop = min(pos + d.per, d.all), heads = s.c.heads;
    if (pos >= stop) return;
    auto next_entries = [&] {
        at = Entries(s, at.base + 64, lane);
        if (d.whole) at.count_units();
    };
    uint32_t before = 0;                // steps of one head ahead of entry at.base
    uint64_t past;
    while ((past = __ballot((before + at.upto) * heads > pos)) == 0) {
        before += at.all();
        if (at.base + 64 >= entries_of(s)) return;
        next_entries();
    }
    int slot_e = __builtin_ctzll(past);
    int n = __builtin_amdgcn_readlane(at.tiles, slot_e);
    int steps = __builtin_amdgcn_readlane(at.steps, slot_e);
    before += (uint32_t)__builtin_amdgcn_readlane(at.upto, slot_e) - (uint32_t)steps;
    const uint32_t in_entry = pos - before * heads;
    int h = __builtin_amdgcn_readfirstlane(in_entry / (uint32_t)steps);
    int tile = in_entry - h * steps;
    for (;;) {
        const int take = min(steps - tile, (int)(stop - pos));
        const int end = d.whole ? n : min(tile + take, n);
        const int e = at.base + slot_e;
        const int b = s.prefix ? 0 : s.row_groups == 1 ? e : e / s.row_groups;
        // (a unit's cost alone may be what is left of it)
        if (tile < end) {
            if (tile == 0 && threadIdx.x == 0) {
                uint32_t* w = s.where + (e * heads + h) * 2;
                w[0] = blockIdx.x;
                w[1] = d.whole ? 1 : (pos + n - 1) / d.per - blockIdx.x + 1;
            }
            part(b, h, (e - b * s.row_groups) * s.rows_per_unit, tile, end, n);
        }
        pos += take;
        if (pos >= stop) return;
        tile = 0;
        if (++h == s.c.heads) {
            h = 0;
            do {
                if (++slot_e == 64) {
                    if (at.base + 64 >= entries_of(s)) return;
                    next_entries();
                    slot_e = 0;
                }
                if (at.base + slot_e >= entries_of(s)) return;
                n = __builtin_amdgcn_readlane(at.tiles, slot_e);
            } while (n == 0);
            steps = __builtin_amdgcn_readlane(at.steps, slot_e);
        }
    }
}

// Where the rows of a part of a unit go: `out` or the rows' home if the part
// is the whole unit, else a slot of the run.
template <class T, int D>
struct Sink {
    T* out;            // null: a triple
    float* o;
    float* ml;
    __device__ __forceinline__ Sink(const Source& s, int b, int h, int row0, bool whole,
                                    bool behind, int r) {
        out = nullptr;
        int64_t to = s.broken + ((int64_t)blockIdx.x * 2 + (behind ? 0 : 1)) * s.rows_per_unit +
                     r - row0;
        if (whole) {
            const int64_t row = RowAt(s, b, r, h).flat(s);
            if (s.finish) out = static_cast<T*>(s.a.out) + row * D;
            to = s.home + row;
        }
        o = s.o + to * D;
        ml = s.ml + to * 2;
    }
    __device__ __forceinline__ void put(int dim, f4 v, float l) const {
        if (out != nullptr)
            store4(out + dim, l == 0.f ? f4{0.f, 0.f, 0.f, 0.f} : v * (1.f / l));
        else
            *reinterpret_cast<f4*>(o + dim) = v;
    }
    __device__ __forceinline__ void put(float m, float l) const {
        if (out == nullptr) *reinterpret_cast<Vec<float, 2>*>(ml) = Vec<float, 2>{m, l};
    }
};

// The block table of a unit's keys: the entry of 16 keys `sub` of a tile (past
// the table: its last).
struct Table {
    const int32_t* p;
    int cols;
    __device__ __forceinline__ Table(const Source& s, int b)
        : p(s.prefix ? s.a.prefix_table : s.a.table + b * s.a.table_stride),
          cols(s.prefix ? s.a.prefix_cols : s.a.table_cols) {}
    __device__ __forceinline__ uint32_t of(const Source& s, int tile, int sub) const {
        return (uint32_t)p[(uint32_t)min((tile * kTile + sub * 16) >> s.page_shift, cols - 1)];
    }
};

// Whether an entry names a page, and which (0 for none).
__device__ __forceinline__ bool is_page(const Source& s, uint32_t entry) {
    return entry < (uint32_t)s.c.pages;
}
__device__ __forceinline__ uint32_t page_or_0(const Source& s, uint32_t entry) {
    return is_page(s, entry) ? entry : 0;
}

// Bytes of K (or V) from the cache's start to a head of a page, and floats of
// the scales; `unit` bytes (floats) to a token.
__device__ __forceinline__ uint64_t head_of(const Source& s, uint32_t page, int h, int unit) {
    return ((uint64_t)page * (uint32_t)s.c.heads + (uint32_t)h) * (uint32_t)(s.c.page_size * unit);
}

// ------------------------------------------------------- few rows: a wave's
// The four waves of a workgroup take the same 16 NB rows and every fourth tile
// each, codes from memory to registers, and join their sums in LDS.
template <class T, int BITS, int D, int NB>
struct Tiles : Rows<T, BITS, D, NB, true> {
    using Base = Rows<T, BITS, D, NB, true>;
    using Base::kSteps;
    static constexpr int kRow = D * BITS / 8;              // bytes of a token's row
    static constexpr int kLane = kRow / 4;                 // K bytes of a lane and row
    static constexpr int kChunk = kLane < 16 ? kLane : 16;
    static constexpr int kChunks = kLane / kChunk;
    static constexpr int kWords = kChunk / 4;
    static constexpr int kVTiles = kRow / 16;              // 16 rows of V bytes

    Vec<uint32_t, kWords> kq[4][kChunks];
    u4 vq[kVTiles];
    float ks, vs;                        // scales of key `lane` of the tile
    bool there;                          // the lane group's 16 keys have a page

    // K's rows in the order that gives lane group g keys 16 g .. 16 g + 15.
    // Codes are read once, past the caches (64 sequences of up to 16384 keys:
    // 213 us with ordinary loads, 197 with non-temporal ones).
    __device__ __forceinline__ void load_k(const Source& s, uint32_t entry, int tile, int h,
                                           int lane) {
        const int g = lane >> 4, r = lane & 15;
        const int in = (tile * kTile + (r >> 2) * 16) & (s.c.page_size - 1);
        const uint8_t* p = static_cast<const uint8_t*>(s.c.k) +
                           head_of(s, page_or_0(s, entry), h, kRow) +
                           (in + (r & 3)) * kRow + g * kChunk;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
                kq[t][c] =
                    __builtin_nontemporal_load(reinterpret_cast<const Vec<uint32_t, kWords>*>(
                        p + t * 4 * kRow + c * 4 * kChunk));
    }

    __device__ __forceinline__ void load_v(const Source& s, uint32_t entry, int tile, int h,
                                           int lane) {
        const int g = lane >> 4, r = lane & 15;
        const uint32_t page = page_or_0(s, entry);
        there = is_page(s, entry);
        const int in = (tile * kTile + g * 16) & (s.c.page_size - 1);
        const float* sc = s.c.scales + head_of(s, page, h, 2) + in + r;
        ks = sc[0];
        vs = sc[s.c.page_size];
        const uint8_t* p = static_cast<const uint8_t*>(s.c.v) + head_of(s, page, h, kRow) +
                           in * kRow + r * 16;
#pragma unroll
        for (int i = 0; i < kVTiles; ++i)
            vq[i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p + i * 256));
    }

    static __device__ __forceinline__ h8 unpack_k(const Vec<uint32_t, kWords> (&row)[kChunks],
                                                  int u) {
        constexpr int per = kChunk / BITS;                 // steps of a chunk
        u4 w;
        if constexpr (BITS == 8) {
            uint32_t x, y, z, v;
            halves_of_bytes(row[u / per][2 * (u % per)], x, y);
            halves_of_bytes(row[u / per][2 * (u % per) + 1], z, v);
            w = u4{x, y, z, v};
        } else {
            uint32_t x[4];
            halves_of_nibbles(row[u / per][u % per], x);
            w = u4{x[0], x[1], x[2], x[3]};
        }
        return __builtin_bit_cast(h8, w);
    }

    // One tile of keys.  next_k and next_v issue the loads that the registers
    // freed by then can take.
    template <class NextK, class NextV>
    __device__ __forceinline__ void step(int tile, int lane, NextK&& next_k, NextV&& next_v) {
        f4 sc[NB][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int rb = 0; rb < NB; ++rb) {
                const float x = this->start[rb];
                sc[rb][t] = f4{x, x, x, x};
            }
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
                const h8 k = unpack_k(kq[t], u);
#pragma unroll
                for (int rb = 0; rb < NB; ++rb)
                    sc[rb][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, this->q[rb][u],
                                                                      sc[rb][t], 0, 0, 0);
            }
        }
        next_k();
        h8 w[NB][2];
        this->weights(sc, ks, vs, there, tile, lane, w);
        auto& o = this->o;
#pragma unroll
        for (int i = 0; i < kVTiles; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if constexpr (BITS == 8) {
                    uint32_t a, b, c, d;
                    codes_of_bytes(vq[i][2 * u], a, b);
                    codes_of_bytes(vq[i][2 * u + 1], c, d);
                    const h8 v = __builtin_bit_cast(h8, u4{a, b, c, d});
#pragma unroll
                    for (int rb = 0; rb < NB; ++rb)
                        o[rb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[rb][u], o[rb][i],
                                                                         0, 0, 0);
                } else {
                    // bytes are tokens here: low nibbles the even dim's, high
                    // ones the odd dim's
                    uint32_t p0[4], p1[4];
                    codes_of_nibbles(vq[i][2 * u], p0);
                    codes_of_nibbles(vq[i][2 * u + 1], p1);
                    const h8 even = __builtin_bit_cast(h8, u4{p0[0], p0[2], p1[0], p1[2]});
                    const h8 odd = __builtin_bit_cast(h8, u4{p0[1], p0[3], p1[1], p1[3]});
#pragma unroll
                    for (int rb = 0; rb < NB; ++rb) {
                        o[rb][2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            even, w[rb][u], o[rb][2 * i], 0, 0, 0);
                        o[rb][2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            odd, w[rb][u], o[rb][2 * i + 1], 0, 0, 0);
                    }
                }
            }
        next_v();
    }

    // Keys from tile `tile`, every `stride`th up to `end`.  The first loads go
    // out before the queries are fetched.
    __device__ __forceinline__ void run(const Source& s, int b, int first_row, int h, int tile,
                                        int end, int stride, int lane) {
        const int g = lane >> 4;
        const int ksub = (lane & 15) >> 2;
        const Table table(s, b);
        // Loads go out unconditionally, the last tile's again behind it: under a
        // condition they would be waited for with everything behind them.  (A
        // second copy of the step, or of the loads, costs more in instruction
        // fetches; scalar loads of the table doubled short calls.)
        const int last = end - 1 - (end - 1 - tile) % stride;
        auto next_of = [&](int t) { return t + stride < end ? t + stride : last; };
        uint32_t ke = 0, ve = 0;
        if (tile < end) {
            const uint32_t k0 = table.of(s, tile, ksub), v0 = table.of(s, tile, g);
            ke = table.of(s, next_of(tile), ksub);
            ve = table.of(s, next_of(tile), g);
            load_k(s, k0, tile, h, lane);
            load_v(s, v0, tile, h, lane);
        }
        this->load(s, b, first_row, h, lane, [&](int u) {
            constexpr int per = kChunk / BITS;
            return ((u / per) * 4 * kChunk + g * kChunk) * 8 / BITS + (u % per) * 8;
        });
        for (; tile < end; tile += stride) {
            const int next = next_of(tile), then = next_of(next);
            const uint32_t k2 = table.of(s, then, ksub), v2 = table.of(s, then, g);
            step(tile, lane, [&] { load_k(s, ke, next, h, lane); },
                 [&] { load_v(s, ve, next, h, lane); });
            ke = k2;
            ve = v2;
        }
    }
};

// Least waves per SIMD (registers) and workgroups that a CU is dealt.
constexpr int waves_of(int d, int nb) { return d * nb <= 128 ? 2 : 1; }

template <class T, int BITS, int D, int NB>
__global__ __launch_bounds__(kBlock, waves_of(D, NB)) void tile_kernel(Source s) {
    constexpr int kRows = 16 * NB;
    __shared__ __attribute__((aligned(16))) float sm_o[kWaves][kRows][D + 4];
    __shared__ float sm_m[kWaves][kRows], sm_l[kWaves][kRows];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tiles<T, BITS, D, NB> work;
    walk_run(s, lane, [&](int b, int h, int row0, int tile, int end, int n) {
        work.run(s, b, row0, h, tile + wave, end, kWaves, lane);
#pragma unroll
        for (int rb = 0; rb < NB; ++rb) {
            const int r = 16 * rb + (lane & 15);
            const float l = quad_sum(work.l[rb]);
            if (lane < 16) {
                sm_m[wave][r] = work.reference(rb);
                sm_l[wave][r] = l;
            }
            work.each_four(rb, lane,
                           [&](int dim, f4 x) { *reinterpret_cast<f4*>(&sm_o[wave][r][dim]) = x; });
        }
        __syncthreads();
        const int rows = min(kRows, s.rows - row0);
        for (int i = threadIdx.x; i < rows * (D / 4); i += kBlock) {
            const int r = i / (D / 4), dim = i % (D / 4) * 4;
            float top = sm_m[0][r], sum = 0.f;
#pragma unroll
            for (int v = 1; v < kWaves; ++v) top = fmaxf(top, sm_m[v][r]);
            f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                const float by = root(sm_m[v][r], sm_l[v][r], top);
                sum += sm_l[v][r] * by * by;
                x += *reinterpret_cast<const f4*>(&sm_o[v][r][dim]) * (by * by);
            }
            const Sink<T, D> sink(s, b, h, row0, tile == 0 && end == n, tile > 0, row0 + r);
            if (dim == 0) sink.put(top, sum);
            sink.put(dim, x, sum);
        }
        __syncthreads();
    });
}

// -------------------------------------------------- many rows: a workgroup's
// W waves take 32 rows each and the same keys: the codes of a tile become fp16
// once, in LDS, for all of them, two tiles in turn, while the next tile's codes
// are on their way to registers.
template <class T, int BITS, int D, int W>
__global__ __launch_bounds__(64 * W, W == 8 || D == 256 ? 1 : 2) void block_kernel(Source s) {
    constexpr int NB = 2, kThreads = 64 * W;
    constexpr int kRow = D * BITS / 8;
    constexpr int kParts = kRow / 16;                      // 16 bytes of a K row
    constexpr int kPieces = kTile * kParts;                // of a tile's K, and of its V
    constexpr int kEach = (kPieces + kThreads - 1) / kThreads;
    constexpr int kCodes = 128 / BITS;                     // codes of a piece
    // rows in LDS start 16 bytes apart from a multiple of the banks
    constexpr int kKRow = D + 8, kVRow = kTile + 8;
    __shared__ __attribute__((aligned(16))) _Float16 sm_k[2][kTile][kKRow];
    __shared__ __attribute__((aligned(16))) _Float16 sm_v[2][D][kVRow];
    const int lane = threadIdx.x & 63, g = lane >> 4, r16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Rows<T, BITS, D, NB, false> rows;
    u4 kq[kEach], vq[kEach];

    walk_run(s, lane, [&](int b, int h, int row0, int tile, int end, int n) {
        const Table table(s, b);
        const int mine = row0 + 32 * wave;
        const bool live = mine < s.rows;
        // pieces of a tile: K's by key and part, V's by 16 keys and row
        uint32_t ke[kEach], ve[kEach], se;
        auto look_up = [&](int t) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int c = threadIdx.x + i * kThreads;
                ke[i] = table.of(s, t, c / kParts >> 4 & 3);
                ve[i] = table.of(s, t, c / kRow & 3);
            }
        };
        auto fetch = [&](int t) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int c = threadIdx.x + i * kThreads;
                if (kPieces % kThreads != 0 && c >= kPieces) break;
                const int key = c / kParts, sub = c / kRow;
                const uint32_t kp = page_or_0(s, ke[i]), vp = page_or_0(s, ve[i]);
                const int kin = (t * kTile + key) & (s.c.page_size - 1);
                const int vin = (t * kTile + sub * 16) & (s.c.page_size - 1);
                kq[i] = *reinterpret_cast<const u4*>(static_cast<const uint8_t*>(s.c.k) +
                                                     head_of(s, kp, h, kRow) + kin * kRow +
                                                     (c % kParts) * 16);
                vq[i] = *reinterpret_cast<const u4*>(static_cast<const uint8_t*>(s.c.v) +
                                                     head_of(s, vp, h, kRow) + vin * kRow +
                                                     (c % kRow) * 16);
            }
        };
        auto spread = [&](int buf) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int c = threadIdx.x + i * kThreads;
                if (kPieces % kThreads != 0 && c >= kPieces) break;
                // key 16 s + 4 t + i lies in row 16 t + 4 s + i: the rows of
                // product t are then 16 side by side
                const int key = c / kParts, sub = c / kRow, vr = c % kRow;
                const int kr = (key >> 2 & 3) * 16 + (key >> 4) * 4 + (key & 3);
                u4* kd = reinterpret_cast<u4*>(&sm_k[buf][kr][(c % kParts) * kCodes]);
                if constexpr (BITS == 8) {
                    u4* vd = reinterpret_cast<u4*>(&sm_v[buf][vr][sub * 16]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t x[4], y[4];
                        codes_of_bytes(kq[i][2 * j], x[0], x[1]);
                        codes_of_bytes(kq[i][2 * j + 1], x[2], x[3]);
                        codes_of_bytes(vq[i][2 * j], y[0], y[1]);
                        codes_of_bytes(vq[i][2 * j + 1], y[2], y[3]);
                        kd[j] = u4{x[0], x[1], x[2], x[3]};
                        vd[j] = u4{y[0], y[1], y[2], y[3]};
                    }
                } else {
                    // V's row is two dims: the even ones' tokens, the odd ones'
                    u4* even = reinterpret_cast<u4*>(&sm_v[buf][vr / 16 * 32 + vr % 16][sub * 16]);
                    u4* odd = reinterpret_cast<u4*>(&sm_v[buf][vr / 16 * 32 + 16 + vr % 16][sub * 16]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t x[4];
                        codes_of_nibbles(kq[i][j], x);
                        kd[j] = u4{x[0], x[1], x[2], x[3]};
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t x[4], y[4];
                        codes_of_nibbles(vq[i][2 * j], x);
                        codes_of_nibbles(vq[i][2 * j + 1], y);
                        even[j] = u4{x[0], x[2], y[0], y[2]};
                        odd[j] = u4{x[1], x[3], y[1], y[3]};
                    }
                }
            }
        };
        float ks, vs;
        bool there;
        auto fetch_scales = [&](int t) {
            there = is_page(s, se);
            const int in = (t * kTile + g * 16) & (s.c.page_size - 1);
            const float* sc = s.c.scales + head_of(s, page_or_0(s, se), h, 2) + in + r16;
            ks = sc[0];
            vs = sc[s.c.page_size];
        };
        // (loads go out unconditionally, past the end for the last tile again:
        // under a condition they would be waited for with everything behind)
        se = table.of(s, tile, g);
        look_up(tile);
        fetch_scales(tile);
        fetch(tile);
        look_up(min(tile + 1, end - 1));
        if (live) rows.load(s, b, mine, h, lane, [&](int u) { return u * 32 + g * 8; });
        spread(0);
        fetch(min(tile + 1, end - 1));
        __syncthreads();
        for (int t = tile; t < end; ++t) {
            const int buf = (t - tile) & 1, t1 = min(t + 1, end - 1), t2 = min(t + 2, end - 1);
            se = table.of(s, t1, g);
            look_up(t2);
            h8 w[NB][2];
            if (live) {
                f4 sc[NB][4];
                h8 k[2][4];
                // reads four at a time, a group ahead of their products
                constexpr int kU = D / 32;
                auto read_k = [&](int group) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int i = (4 * group + j) / kU, u = (4 * group + j) % kU;
                        k[group & 1][j] = *reinterpret_cast<const h8*>(
                            &sm_k[buf][16 * i + r16][u * 32 + g * 8]);
                    }
                };
                read_k(0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int rb = 0; rb < NB; ++rb) sc[rb][i] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int group = 0; group < kU; ++group) {
                    if (group < kU - 1) read_k(group + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int i = (4 * group + j) / kU, u = (4 * group + j) % kU;
#pragma unroll
                        for (int rb = 0; rb < NB; ++rb)
                            sc[rb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                k[group & 1][j], rows.q[rb][u], sc[rb][i], 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                rows.weights(sc, ks, vs, there, t, lane, w);
            }
            fetch_scales(t1);
            if (live) {
                h8 v[2][4];
                auto read_v = [&](int i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[i & 1][j] = *reinterpret_cast<const h8*>(
                            &sm_v[buf][16 * (2 * i + j / 2) + r16][g * 16 + (j & 1) * 8]);
                };
                read_v(0);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    if (i < D / 32 - 1) read_v(i + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int rb = 0; rb < NB; ++rb)
                            rows.o[rb][2 * i + j / 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                v[i & 1][j], w[rb][j & 1], rows.o[rb][2 * i + j / 2], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            spread(buf ^ 1);
            fetch(t2);
            __syncthreads();
        }
        if (live) {
#pragma unroll
            for (int rb = 0; rb < NB; ++rb) {
                const int r = mine + 16 * rb + r16;
                const float l = quad_sum(rows.l[rb]);
                if (r < s.rows) {
                    const Sink<T, D> sink(s, b, h, row0, tile == 0 && end == n, tile > 0, r);
                    if (lane < 16) sink.put(rows.reference(rb), l);
                    rows.each_four(rb, lane, [&](int dim, f4 v) { sink.put(dim, v, l); });
                }
            }
        }
    });
}

// Joins the triples of rows: those of their own keys' runs and, with a prefix,
// those of the prefix's.  `W` waves per row, each its share of the triples, and
// `each` rows of a unit in turn, from the launch's first workgroup on.  Rows
// that a run has finished are left alone; rows without any keys become zeros.
template <int D>
constexpr int in_flight = D == 256 ? 8 : 16;       // triples
template <class T, int D, int W>
__global__ __launch_bounds__(kBlock) void join_kernel(Source own, Source ahead, int each,
                                                      uint32_t first_block) {
    constexpr int E = D / 64, J = in_flight<D>;
    using VE = Vec<float, E>;
    __shared__ float part[W > 1 ? W : 1][W > 1 ? D + 2 : 1];
    const int lane = threadIdx.x & 63;
    const cq_attention_t& a = own.a;
    const uint32_t blocks = (own.rows + each - 1) / each;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t block = first_block + blockIdx.x;
    const uint32_t place = W == 1 ? block * kWaves + w : block;
    const uint32_t unit = place / blocks;
    const int r0 = (place - unit * blocks) * each;
    const int h = unit % own.c.heads, b = unit / own.c.heads;
    if (b >= a.batch) return;          // uniform over the wave (W = 1) or workgroup

    // the runs that have a unit's triples
    struct Parts {
        uint32_t run = 0;
        int count = 0;
    };
    auto parts_of = [&](const Source& s, int entry) {
        const uint32_t* at = s.where + (entry * (uint32_t)s.c.heads + h) * 2;
        return Parts{at[0], (int)at[1]};
    };
    const Parts mine = parts_of(own, b * own.row_groups + r0 / own.rows_per_unit);
    if (own.finish && mine.count == 1) return;
    for (int r = r0; r < min(r0 + each, own.rows); ++r) {
        const int t = r / own.group;
        const int64_t row = ((int64_t)b * a.tokens + t) * a.q_heads + h * own.group +
                            (r - t * own.group);
        Parts pre;
        // where a source's triples start: one at home, or the first run's last
        // row block and every next one's first
        auto start_of = [&](const Source& s, const Parts& p, int local) {
            return p.count == 1 ? s.home + row
                                : s.broken + (int64_t)p.run * 2 * s.rows_per_unit + local;
        };
        const int64_t at_mine = start_of(own, mine, r % own.rows_per_unit);
        int64_t at_pre = 0;
        int pre_rows = 0;
        if (!own.finish) {
            const int pr = b * own.rows + r;
            pre = parts_of(ahead, pr / ahead.rows_per_unit);
            pre_rows = ahead.rows_per_unit;
            at_pre = start_of(ahead, pre, pr % pre_rows);
        }
        const int count = mine.count + pre.count;
        auto triple = [&](int i) {
            const bool first = i < mine.count;
            const int j = first ? i : i - mine.count;
            const int n = first ? mine.count : pre.count;
            const int step = first ? own.rows_per_unit : pre_rows;
            const int64_t from = first ? at_mine : at_pre;
            return from + (n == 1 ? 0 : (j == 0 ? 1 : 2 * j) * step);
        };
        float ref = kNegInf, sum = 0.f;
        VE acc = {};
        for (int base = W == 1 ? 0 : w * J; base < count; base += W * J) {
            // a triple's reference and sum to a lane, its row over the wave
            const Vec<float, 2> ml = *reinterpret_cast<const Vec<float, 2>*>(
                own.ml + triple(min(base + min(lane, J - 1), count - 1)) * 2);
            VE v[J];
#pragma unroll
            for (int i = 0; i < J; ++i)
                v[i] = *reinterpret_cast<const VE*>(
                    own.o + triple(min(base + i, count - 1)) * D + lane * E);
            const float top = fmaxf(ref, wave_max(ml[0]));
            const float keep = root(ref, sum, top);
            const float half = root(ml[0], ml[1], top);
            const float by = half * half, share = ml[1] * half * half;
            sum = sum * keep * keep;
#pragma unroll
            for (int j = 0; j < E; ++j) acc[j] *= keep * keep;
            ref = top;
#pragma unroll
            for (int i = 0; i < J; ++i) {
                const bool more = base + i < count;
                const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(by), i));
                const float g = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(share), i));
                sum += more ? g : 0.f;
#pragma unroll
                for (int j = 0; j < E; ++j) acc[j] += more ? v[i][j] * f : 0.f;
            }
        }
        if constexpr (W > 1) {
            if (r > r0) __syncthreads();
#pragma unroll
            for (int j = 0; j < E; ++j) part[w][lane * E + j] = acc[j];
            if (lane == 0) {
                part[w][D] = ref;
                part[w][D + 1] = sum;
            }
            __syncthreads();
            if (w > 0) continue;
            float top = ref;
#pragma unroll
            for (int i = 1; i < W; ++i) top = fmaxf(top, part[i][D]);
            sum = 0.f;
            acc = VE{};
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float by = root(part[i][D], part[i][D + 1], top);
                sum += part[i][D + 1] * by * by;
#pragma unroll
                for (int j = 0; j < E; ++j) acc[j] += by * by * part[i][lane * E + j];
            }
        }
        T* out = static_cast<T*>(a.out) + row * D + lane * E;
#pragma unroll
        for (int j = 0; j < E; ++j) out[j] = (T)(sum == 0.f ? 0.f : acc[j] / sum);
    }
}

// ------------------------------------------------------------------- host
constexpr int kCus = 256;

// Which kernel takes a source: the tile kernel with nb row matrices to a wave,
// or the block kernel with `waves` waves.
struct Shape {
    int nb;          // 0: the block kernel
    int waves;
    int rows;        // of a unit
    int resident;    // workgroups that a CU holds
};

// The tile kernel unpacks every code once per row group; the block kernel once
// for up to 256 rows, but has a unit's start and end to pay for.  So with few
// units of many keys (as the table has room for) the tile kernel is ahead for
// longer.
// Measured on 8 heads over 4096 keys, us, tile and block kernel:
//   heads of 128, 16 sequences: 32 rows 48, 61; 64 rows 61, 77; 80 rows 105, 79
//                 64 sequences of 1000 keys: 40 rows 101, 63
//                 2 sequences of 700 keys: 64 rows 18.1, 17.7
//   heads of 64, 16 sequences: 64 rows 51, 59; 96 rows 71, 64
//                 7 sequences of up to 1501 keys, 4 heads: 35 rows 16.7, 15.0
//   heads of 256 (groups of 16), 16 sequences: 32 rows 82, 142; 48 rows 154, 151
//                 64 sequences of 600 keys: 32 rows 106, 97
// and of the block kernel four waves or eight: 128 rows 94, 100; 160 rows 135, 124.
Shape shape_of(int64_t rows, int64_t units, int64_t keys, int d) {
    const bool few = units <= kCus;
    if (rows <= (d == 256 && few ? 32 : 16)) return {1, kWaves, 16, waves_of(d, 1)};
    if (d <= 128 && rows <= (few && keys >= 2048 ? 64 : 32)) return {2, kWaves, 32, waves_of(d, 2)};
    if (d == 256) return {0, 4, 128, 1};
    if (rows <= 128) return {0, 4, 128, 2};
    return {0, 8, 256, 1};
}

Source source_of(const cq_kv_cache_t& c, const cq_attention_t& a, bool prefix, Shape* shape) {
    Source s{};
    s.c = c;
    s.a = a;
    s.prefix = prefix;
    s.group = a.q_heads / c.heads;
    s.page_shift = __builtin_ctz((unsigned)c.page_size);
    const int64_t rows = (int64_t)a.tokens * s.group * (prefix ? a.batch : 1);
    s.rows = (int32_t)rows;
    const int64_t keys = prefix ? a.prefix_len : (int64_t)a.table_cols * c.page_size;
    *shape = shape_of(rows, (int64_t)c.heads * (prefix ? 1 : a.batch), keys, c.head_dim);
    s.rows_per_unit = shape->rows;
    s.row_groups = (int32_t)((rows + s.rows_per_unit - 1) / s.rows_per_unit);
    // a workgroup of the tile kernel takes four tiles at a time; a unit's start
    // and end take as long as two rounds of them, or two tiles of the block
    // kernel
    s.quantum = shape->nb > 0 ? kWaves : 2;
    s.cost = shape->nb > 0 ? 2 * kWaves : 2;
    s.finish = a.prefix_len == 0;
    // no more runs than quanta, as far as the tables' sizes tell
    const int64_t entries = (int64_t)s.row_groups * (prefix ? 1 : a.batch);
    const __int128 steps = (__int128)((keys + kTile - 1) / kTile + s.quantum + s.cost) * entries *
                           c.heads;
    s.fits = steps + (__int128)kCus * 8 * s.quantum < ((__int128)1 << 31) &&
             keys <= 0x7FFFFFFF - kTile && rows <= 0x7FFFFFFF;
    const int64_t room = (int64_t)kCus * shape->resident;
    const __int128 most = steps / s.quantum;
    s.runs = (uint32_t)(most < room ? (int64_t)most : room);
    return s;
}

// Lays out the workspace from `base` (null: only sizes); returns its bytes.
int64_t lay_out(const cq_kv_cache_t& c, const cq_attention_t& a, Source* own, Source* ahead,
                char* base) {
    const int64_t all = (int64_t)a.batch * a.tokens * a.q_heads;
    int64_t triples = 0;
    for (Source* s : {own, ahead}) {
        if (s->rows == 0) continue;
        s->broken = triples;
        triples += (int64_t)s->runs * 2 * s->rows_per_unit;
        s->home = triples;
        if (!s->finish) triples += all;
    }
    int64_t used = triples * (c.head_dim + 2) * 4;
    used = (used + 15) / 16 * 16;
    for (Source* s : {own, ahead}) {
        if (s->rows == 0) continue;
        if (base != nullptr) {
            s->o = reinterpret_cast<float*>(base);
            s->ml = reinterpret_cast<float*>(base + triples * c.head_dim * 4);
            s->where = reinterpret_cast<uint32_t*>(base + used);
        }
        used += ((int64_t)s->row_groups * (s->prefix ? 1 : a.batch) * c.heads * 8 + 15) / 16 * 16;
    }
    return used;
}

template <class T, int BITS, int D>
hipError_t launch_tiles(const Source& s, Shape shape, hipStream_t stream) {
    auto go = [&](auto* kernel) {
        kernel<<<dim3(s.runs), dim3(64 * shape.waves), 0, stream>>>(s);
        return hipGetLastError();
    };
    if (shape.nb == 1) return go(&tile_kernel<T, BITS, D, 1>);
    if constexpr (D <= 128) {
        if (shape.nb == 2) return go(&tile_kernel<T, BITS, D, 2>);
        if (shape.waves == 8) return go(&block_kernel<T, BITS, D, 8>);
    }
    return go(&block_kernel<T, BITS, D, 4>);
}

template <class T, int D>
hipError_t launch_typed(const Source& own, Shape os, const Source& ahead, Shape as,
                        hipStream_t stream) {
    hipError_t e = hipSuccess;
    const bool wide = own.c.bits == 8;
    if (ahead.rows > 0)
        e = wide ? launch_tiles<T, 8, D>(ahead, as, stream) : launch_tiles<T, 4, D>(ahead, as, stream);
    if (e != hipSuccess) return e;
    e = wide ? launch_tiles<T, 8, D>(own, os, stream) : launch_tiles<T, 4, D>(own, os, stream);
    if (e != hipSuccess) return e;
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

}  // namespace

int64_t attention_workspace(const cq_kv_cache_t& c, const cq_attention_t& a) {
    Shape os{}, as{};
    Source own = source_of(c, a, false, &os), ahead{};
    if (a.prefix_len > 0) ahead = source_of(c, a, true, &as);
    if (!own.fits || (ahead.rows > 0 && !ahead.fits)) return -1;
    return lay_out(c, a, &own, &ahead, nullptr);
}

hipError_t launch_attention(const cq_kv_cache_t& c, const cq_attention_t& a,
                            hipStream_t stream) {
    Shape os{}, as{};
    Source own = source_of(c, a, false, &os), ahead{};
    if (a.prefix_len > 0) ahead = source_of(c, a, true, &as);
    lay_out(c, a, &own, &ahead, static_cast<char*>(a.workspace));
    auto typed = [&](auto elem) {
        using T = decltype(elem);
        if (c.head_dim == 64) return launch_typed<T, 64>(own, os, ahead, as, stream);
        if (c.head_dim == 128) return launch_typed<T, 128>(own, os, ahead, as, stream);
        return launch_typed<T, 256>(own, os, ahead, as, stream);
    };
    return a.dtype == CQ_DTYPE_F16 ? typed(_Float16{}) : typed(__bf16{});
}

}  // namespace cq
