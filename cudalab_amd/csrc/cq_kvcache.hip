// A paged key/value cache quantized as it is written, and read back (gfx950).
//
// Per token and head, for K and for V, with qmax 127 (8 bits) or 7 (4 bits):
//   scale = amax * fl(1 / qmax), code = clamp(rint(x * fl(1 / scale)), +-qmax)
// with every product, the quotient and the scale rounded to FP32, so the codes
// are the same on any device.  A vector whose amax is below 2^-100 (its scale
// or reciprocal would leave FP32's normal range) is stored as zeros; one with
// NaN or Inf gets scale NaN and codes 0, so that whatever sees it becomes NaN.
//
// K keeps a token's row together; V keeps 16 tokens of a dim together
// ([page_size / 16, row, 16] bytes, row = head_dim bytes, or head_dim / 2 of
// two dims each), so that the attention kernels read both as matrix operands.
// Both kernels work on tiles of 16 tokens of one head, aligned in the page:
// 16 lanes hold a token's vector, and V turns through LDS.
//
// Bound by memory at long inputs, by the launch at one token per sequence.  What
// is read or written once goes past the caches (non-temporal): reading 54009
// tokens of 8 heads of 128 back took 59 us with ordinary stores, 40 with these.

#include "cq_elem.h"
#include "cq_step.h"

namespace cq {
namespace {

constexpr int kBlock = 256;

// Largest |x| of the 16 lanes that share a token, as FP32 bits (NaN above
// Inf above every number).  Magnitudes of 16 bits are compared as they are, two
// at a time.
template <class T, int E>
__device__ __forceinline__ uint32_t amax16(const T (&x)[E]) {
    auto over16 = [](uint32_t m, auto&& larger) {
        m = larger(m, row_dpp<0x128>(m));
        m = larger(m, row_dpp<0x124>(m));
        m = larger(m, row_dpp<0x122>(m));
        return larger(m, row_dpp<0x121>(m));
    };
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
        auto larger = [](uint32_t a, uint32_t b) { return max(a, b); };
#pragma unroll
        for (int i = 0; i < E; ++i) m = larger(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
        return over16(m, larger);
    } else {
        using u2 = Vec<unsigned short, 2>;
        auto larger = [](uint32_t a, uint32_t b) {
            return __builtin_bit_cast(uint32_t,
                                      __builtin_elementwise_max(__builtin_bit_cast(u2, a),
                                                                __builtin_bit_cast(u2, b)));
        };
#pragma unroll
        for (int i = 0; i < E; i += 2)
            m = larger(m, __builtin_bit_cast(uint32_t, Vec<T, 2>{x[i], x[i + 1]}) & 0x7FFF7FFFu);
        m = over16(m, larger);
        const unsigned short top = (unsigned short)max(m & 0xFFFFu, m >> 16);
        return __float_as_uint((float)__builtin_bit_cast(T, top));
    }
}

// Bytes are transposed among lanes l, l + 16, l + 32, l + 48: byte j of lane
// l + 16 i becomes byte i of lane l + 16 j.
__device__ __forceinline__ uint32_t turn_bytes(uint32_t x) {
    const int q = (threadIdx.x >> 4) & 3;
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t y = __builtin_amdgcn_perm(a[1], a[0], q & 1 ? 0x07030501u : 0x06020400u);
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return __builtin_amdgcn_perm(b[1], b[0], q & 2 ? 0x07060302u : 0x05040100u);
}

// E elements at p; `wide` when 16 bytes (or all E) may be loaded at once.
template <class T, int E>
__device__ __forceinline__ void load_row(T (&x)[E], const T* p, bool wide) {
    if (wide) {
        constexpr int N = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
#pragma unroll
        for (int i = 0; i < E; i += N) {
            const Vec<T, N> v =
                __builtin_nontemporal_load(reinterpret_cast<const Vec<T, N>*>(p + i));
#pragma unroll
            for (int j = 0; j < N; ++j) x[i + j] = v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = p[i];
    }
}

// Bytes of a lane's E codes: E (8 bits) or E / 2.
template <int BITS, int E>
struct Codes {
    static constexpr int kBytes = BITS == 8 ? E : E / 2;
    static constexpr int kWords = (kBytes + 3) / 4;
    uint32_t w[kWords] = {};
    // x * inv lies within qmax (1 + 2^-21), so rounding it needs no clamp.  Four
    // codes make one number: bytes are the low bits of 1.5 * 2^23 and the code;
    // nibbles are digits 8 above their code, all four below 2^16.
    template <class T>
    __device__ __forceinline__ void pack(const T (&x)[E], float inv) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            uint32_t four;
            if constexpr (BITS == 8) {
                uint32_t c[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    c[j] = __float_as_uint((float)x[i + j] * inv + 0x1.8p23f);
                four = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0C0C0400u),
                                             __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u),
                                             0x05040100u);
            } else {
                float sum = rintf((float)x[i + 3] * inv);
#pragma unroll
                for (int j = 2; j >= 0; --j)
                    sum = __builtin_fmaf(sum, 16.f, rintf((float)x[i + j] * inv));
                four = (__float_as_uint(sum + (0x1p23f + 0x8888)) & 0xFFFFu) ^ 0x8888u;
            }
            // inv 0 stands for a vector of zeros, whose x may be NaN or Inf
            if (inv == 0.f) four = 0;
            if constexpr (BITS == 8) w[i / 4] = four;
            else w[i / 8] |= four << (4 * (i % 8));
        }
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
        if constexpr (kBytes == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
        else *reinterpret_cast<Vec<uint32_t, kWords>*>(p) = vec();
    }
    __device__ __forceinline__ void load(const uint8_t* p) {
        if constexpr (kBytes == 2) {
            w[0] = *reinterpret_cast<const uint16_t*>(p);
        } else {
            const Vec<uint32_t, kWords> v = *reinterpret_cast<const Vec<uint32_t, kWords>*>(p);
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = v[i];
        }
    }
    __device__ __forceinline__ int code(int i) const {
        if constexpr (BITS == 8) return (int)(int8_t)(w[i / 4] >> (8 * (i % 4)));
        else return (int)(w[i / 8] << (28 - 4 * (i % 8))) >> 28;
    }

   private:
    __device__ __forceinline__ Vec<uint32_t, kWords> vec() const {
        Vec<uint32_t, kWords> v;
#pragma unroll
        for (int i = 0; i < kWords; ++i) v[i] = w[i];
        return v;
    }
};

// Tokens of a call that lie in tile `tile` of sequence b: position
// base + i, i < 16, is token base + i - start.
struct Tile {
    int64_t page;      // -1: none
    int64_t first;     // call's token of the tile's first position (may be < 0)
    int in_page;       // offset of the tile's first position in its page
    int count;         // tokens of the sequence
    __device__ __forceinline__ Tile(const cq_kv_cache_t& c, const cq_kv_slots_t& s, int b,
                                    int tile) {
        const int32_t start = s.starts[b];
        count = s.tokens;
        if (s.counts != nullptr) count = min(count, s.counts[b]);
        const int64_t base = ((int64_t)start & ~(int64_t)15) + 16 * (int64_t)tile;
        first = base - start;
        page = -1;
        in_page = 0;
        if (base >= 0) {
            const int64_t col = base / c.page_size;
            in_page = (int)(base % c.page_size);
            if (col < s.table_cols) page = page_in(s.table[b * s.table_stride + col], c.pages);
        }
    }
};

// One workgroup per (sequence, tile, head), heads side by side: neighbouring
// workgroups read neighbouring rows.  `first` is the launch's first workgroup.
template <class T, int BITS, int D>
__global__ __launch_bounds__(kBlock) void append_kernel(cq_kv_cache_t c, cq_kv_slots_t s,
                                                        uint32_t tiles, const T* k, KvStrides ks,
                                                        const T* v, KvStrides vs, bool wide,
                                                        uint32_t first) {
    constexpr int E = D / 16;
    constexpr int R = BITS == 8 ? D : D / 2;       // bytes of a row
    using C = Codes<BITS, E>;
    // a lane's rows, and 16 bytes of padding
    __shared__ __attribute__((aligned(16))) uint8_t turned[16][C::kBytes * 16 + 16];
    const uint32_t block = first + blockIdx.x;
    const int h = block % c.heads;
    const uint32_t bt = block / c.heads;
    const int b = bt / tiles;
    const Tile tile(c, s, b, bt % tiles);
    const int i = threadIdx.x >> 4, lane = threadIdx.x & 15;
    const int64_t t = tile.first + i;
    const int64_t lo = tile.first < 0 ? 0 : tile.first;
    if (lo >= tile.count) return;                      // uniform over the workgroup
    const bool live = t >= 0 && t < tile.count;
    T x[E] = {}, y[E] = {};
    if (live) {
        load_row(x, k + b * ks.batch + t * ks.token + h * ks.head + lane * E, wide);
        load_row(y, v + b * vs.batch + t * vs.token + h * vs.head + lane * E, wide);
    }
    if (tile.page < 0) return;
    const int64_t ph = tile.page * c.heads + h;
    C kc, vc;
    float kscale, vscale, kinv, vinv;
    scale_of<BITS>(amax16(x), kscale, kinv);
    scale_of<BITS>(amax16(y), vscale, vinv);
    kc.pack(x, kinv);
    vc.pack(y, vinv);
    if (live) {
        const int64_t at = ph * c.page_size + tile.in_page + i;
        kc.store(static_cast<uint8_t*>(c.k) + at * R + lane * C::kBytes);
        if (lane == 0) {
            float* sc = c.scales + ph * 2 * c.page_size + tile.in_page + i;
            sc[0] = kscale;
            sc[c.page_size] = vscale;
        }
    }
    // four tokens of a row to a word
#pragma unroll
    for (int m = 0; m < C::kWords; ++m) {
        const uint32_t word = turn_bytes(vc.w[m]);
        const int r = 4 * m + (i & 3);
        if (r < C::kBytes) *reinterpret_cast<uint32_t*>(turned[lane] + r * 16 + (i & ~3)) = word;
    }
    __syncthreads();
    uint8_t* vd = static_cast<uint8_t*>(c.v) +
                  (ph * (c.page_size / 16) + tile.in_page / 16) * R * 16;
    if ((int)threadIdx.x < R) {
        const int r = threadIdx.x;
        const uint8_t* row = turned[r / C::kBytes] + r % C::kBytes * 16;
        const int from = (int)(lo - tile.first);
        const int to = (int)min((int64_t)16, tile.count - tile.first);
        if (from == 0 && to == 16)
            *reinterpret_cast<uint4*>(vd + r * 16) = *reinterpret_cast<const uint4*>(row);
        else
            for (int j = from; j < to; ++j) vd[r * 16 + j] = row[j];
    }
}

// Packed rows to their slots (page * page_size + offset): row t of k and v goes
// to slots[t].  Rows whose slots follow one another inside 16 aligned places
// form a group, which is what a tile of the cache is; a workgroup takes the
// groups that begin in its 16 rows (and so up to 31 rows, 16 at a time), one
// head.  A whole group leaves as whole words of V, anything else byte by byte.
// 64 sequences of 5 tokens, three of them kept (every group broken), 8 heads of 128:
// 5.2 us, of which the launch and three loads in a row are most.  16 prompts of up to
// 2048 in 4 bits: 20 us, as fast as a copy of the bytes.
template <class T, int BITS, int D>
__global__ __launch_bounds__(kBlock) void append_rows_kernel(cq_kv_cache_t c, uint32_t tokens,
                                                             const int64_t* slots, const T* k,
                                                             KvStrides ks, const T* v,
                                                             KvStrides vs, bool wide,
                                                             uint32_t first) {
    constexpr int E = D / 16;
    constexpr int R = BITS == 8 ? D : D / 2;       // bytes of a row
    using C = Codes<BITS, E>;
    __shared__ __attribute__((aligned(16))) uint8_t turned[16][C::kBytes * 16 + 16];
    const uint32_t block = first + blockIdx.x;
    const int h = block % c.heads;
    const uint32_t t0 = block / c.heads * 16;
    const int i = threadIdx.x >> 4, lane = threadIdx.x & 15;
    // lane j of a wave: the slot of row t0 - 1 + j, -1 for none
    const int j = threadIdx.x & 63;
    const int64_t at = (int64_t)t0 - 1 + j;
    const int64_t mine = at >= 0 && at < tokens ? slots[at] : -1;
    const int64_t ahead = __shfl_up(mine, 1);
    const bool starts = at >= tokens || (uint64_t)mine != (uint64_t)ahead + 1 || mine % 16 == 0 ||
                        at == 0;
    const uint64_t begins = __ballot(j > 0 && starts) >> 1;     // of rows t0 .. t0 + 62
    if ((begins & 0xFFFF) == 0) return;            // uniform over the workgroup
    const int from = __builtin_ctzll(begins);
    const int to = 16 + __builtin_ctzll(begins >> 16);          // row t0 + 31 is in reach
    const int64_t places = c.pages * c.page_size;
    const int shift = __builtin_ctz(c.page_size);
    for (int base = from; base < to; base += 16) {
        const int r = base + i;
        const uint32_t t = t0 + r;
        const int64_t its = __shfl(mine, r + 1);   // (r is below 47)
        const int64_t slot = r < to ? its : -1;
        const bool live = slot >= 0 && slot < places;
        T x[E] = {}, y[E] = {};
        if (live) {
            load_row(x, k + t * ks.token + h * ks.head + lane * E, wide);
            load_row(y, v + t * vs.token + h * vs.head + lane * E, wide);
        }
        C kc, vc;
        float kscale, vscale, kinv, vinv;
        scale_of<BITS>(amax16(x), kscale, kinv);
        scale_of<BITS>(amax16(y), vscale, vinv);
        kc.pack(x, kinv);
        vc.pack(y, vinv);
        if (live) {
            const int64_t ph = (slot >> shift) * c.heads + h;
            const int64_t in = slot & (c.page_size - 1);
            kc.store(static_cast<uint8_t*>(c.k) + (ph * c.page_size + in) * R + lane * C::kBytes);
            if (lane == 0) {
                float* sc = c.scales + ph * 2 * c.page_size + in;
                sc[0] = kscale;
                sc[c.page_size] = vscale;
            }
        }
#pragma unroll
        for (int m = 0; m < C::kWords; ++m) {
            const uint32_t word = turn_bytes(vc.w[m]);
            const int row = 4 * m + (i & 3);
            if (row < C::kBytes)
                *reinterpret_cast<uint32_t*>(turned[lane] + row * 16 + (i & ~3)) = word;
        }
        __syncthreads();
        auto v_at = [&](int64_t s) {               // dim 0 of a slot
            const int64_t in = s & (c.page_size - 1);
            return static_cast<uint8_t*>(c.v) +
                   (((s >> shift) * c.heads + h) * (c.page_size / 16) + in / 16) * R * 16 + in % 16;
        };
        // the slots of the 16 rows, the same in every wave
        const int64_t slot0 = __shfl(mine, base + 1);
        const bool whole = base + 16 <= to && slot0 >= 0 && slot0 < places && slot0 % 16 == 0 &&
                           ((begins >> base) & 0xFFFF) == 1;
        if (whole) {
            if ((int)threadIdx.x < R) {
                const int row = threadIdx.x;
                *reinterpret_cast<uint4*>(v_at(slot0) + row * 16) =
                    *reinterpret_cast<const uint4*>(turned[row / C::kBytes] + row % C::kBytes * 16);
            }
        } else {
            // a dim (or two) of as many rows to a thread as fill the workgroup
            constexpr int kEach = 16 * R / kBlock > 0 ? 16 * R / kBlock : 1;
            const int dim = threadIdx.x % R, n0 = threadIdx.x / R * kEach;
            int64_t s[kEach];
            uint8_t code[kEach];
#pragma unroll
            for (int n = 0; n < kEach; ++n) {
                s[n] = __shfl(mine, min(base + n0 + n + 1, 63));
                if (base + n0 + n >= to) s[n] = -1;
                code[n] = turned[dim / C::kBytes][dim % C::kBytes * 16 + n0 + n];
            }
#pragma unroll
            for (int n = 0; n < kEach; ++n)
                if (s[n] >= 0 && s[n] < places) v_at(s[n])[dim * 16] = code[n];
        }
        __syncthreads();
    }
}

template <class T, int BITS, int D>
__global__ __launch_bounds__(kBlock) void read_kernel(cq_kv_cache_t c, cq_kv_slots_t s,
                                                      uint32_t tiles, T* k, T* v,
                                                      uint32_t first) {
    constexpr int E = D / 16;
    constexpr int R = BITS == 8 ? D : D / 2;
    using C = Codes<BITS, E>;
    // 16 bytes of padding a token: four tokens' words lie in different banks
    __shared__ __attribute__((aligned(16))) uint8_t turned[16][R + 16];
    const uint32_t block = first + blockIdx.x;
    const int h = block % c.heads;
    const uint32_t bt = block / c.heads;
    const int b = bt / tiles;
    const Tile tile(c, s, b, bt % tiles);
    const int i = threadIdx.x >> 4, lane = threadIdx.x & 15;
    const int64_t t = tile.first + i;
    const bool there = tile.page >= 0;                 // uniform over the workgroup
    if (tile.first + 15 < 0 || tile.first >= s.tokens) return;
    const int64_t ph = there ? tile.page * c.heads + h : 0;
    const int wave = threadIdx.x >> 6;
    if (there && wave * 64 < R) {                      // uniform over the wave
        const int r = wave * 64 + 4 * lane + (i & 3);
        uint4 q = {};
        if (r < R)
            q = *reinterpret_cast<const uint4*>(
                static_cast<const uint8_t*>(c.v) +
                ((ph * (c.page_size / 16) + tile.in_page / 16) * R + r) * 16);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {                  // four rows of a token to a word
            const uint32_t word = turn_bytes(w[j]);
            if (r < R)
                *reinterpret_cast<uint32_t*>(turned[4 * j + (i & 3)] + wave * 64 + 4 * lane) = word;
        }
    }
    __syncthreads();
    if (t < 0 || t >= s.tokens) return;
    float kscale = 0.f, vscale = 0.f;
    C kc, vc;
    if (there && t < tile.count) {
        const int64_t at = ph * c.page_size + tile.in_page + i;
        kc.load(static_cast<const uint8_t*>(c.k) + at * R + lane * C::kBytes);
        vc.load(turned[i] + lane * C::kBytes);
        const float* sc = c.scales + ph * 2 * c.page_size + tile.in_page + i;
        kscale = sc[0];
        vscale = sc[c.page_size];
    }
    const int64_t to = (((int64_t)b * s.tokens + t) * c.heads + h) * D + lane * E;
    constexpr int N = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
#pragma unroll
    for (int e = 0; e < E; e += N) {
        Vec<T, N> x, y;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            x[j] = (T)((float)kc.code(e + j) * kscale);
            y[j] = (T)((float)vc.code(e + j) * vscale);
        }
        __builtin_nontemporal_store(x, reinterpret_cast<Vec<T, N>*>(k + to + e));
        __builtin_nontemporal_store(y, reinterpret_cast<Vec<T, N>*>(v + to + e));
    }
}

// Tiles that the tokens of a sequence may touch, wherever they start.
int64_t tiles_of(const cq_kv_slots_t& s) { return ((int64_t)s.tokens + 15 + 15) / 16; }

// Workgroups of a call; kMaxGrid + 1 for more (the product may pass 64 bits).
int64_t workgroups(const cq_kv_cache_t& c, const cq_kv_slots_t& s) {
    const __int128 n = (__int128)s.batch * tiles_of(s) * c.heads;
    return n <= kMaxGrid ? (int64_t)n : kMaxGrid + 1;
}

template <class F>
hipError_t by_form(const cq_kv_cache_t& c, F&& go) {
    if (c.bits == 8)
        return c.head_dim == 64 ? go(std::integral_constant<int, 8>{}, std::integral_constant<int, 64>{})
               : c.head_dim == 128 ? go(std::integral_constant<int, 8>{}, std::integral_constant<int, 128>{})
                                   : go(std::integral_constant<int, 8>{}, std::integral_constant<int, 256>{});
    return c.head_dim == 64 ? go(std::integral_constant<int, 4>{}, std::integral_constant<int, 64>{})
           : c.head_dim == 128 ? go(std::integral_constant<int, 4>{}, std::integral_constant<int, 128>{})
                               : go(std::integral_constant<int, 4>{}, std::integral_constant<int, 256>{});
}

template <class T>
hipError_t append_typed(const cq_kv_cache_t& c, const cq_kv_slots_t& s, const void* k,
                        KvStrides ks, const void* v, KvStrides vs, hipStream_t stream) {
    const int64_t tiles = tiles_of(s), grid = workgroups(c, s);
    if (grid > kMaxGrid) return hipErrorInvalidValue;
    return by_form(c, [&](auto bits, auto dim) {
        constexpr int E = decltype(dim)::value / 16;
        constexpr int N = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
        bool wide = true;
        for (const KvStrides& st : {ks, vs})
            wide = wide && st.batch % N == 0 && st.token % N == 0 && st.head % N == 0;
        wide = wide && (uintptr_t)k % (N * sizeof(T)) == 0 && (uintptr_t)v % (N * sizeof(T)) == 0;
        return launch_parts(grid, [&](dim3 blocks, uint32_t first) {
            append_kernel<T, decltype(bits)::value, decltype(dim)::value>
                <<<blocks, dim3(kBlock), 0, stream>>>(c, s, (uint32_t)tiles,
                                                      static_cast<const T*>(k), ks,
                                                      static_cast<const T*>(v), vs, wide, first);
        });
    });
}

template <class T>
hipError_t append_rows_typed(const cq_kv_cache_t& c, int64_t tokens, const int64_t* slots,
                             const void* k, KvStrides ks, const void* v, KvStrides vs,
                             hipStream_t stream) {
    const __int128 grid = (__int128)((tokens + 15) / 16) * c.heads;
    if (grid > kMaxGrid) return hipErrorInvalidValue;
    return by_form(c, [&](auto bits, auto dim) {
        constexpr int E = decltype(dim)::value / 16;
        constexpr int N = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
        bool wide = (uintptr_t)k % (N * sizeof(T)) == 0 && (uintptr_t)v % (N * sizeof(T)) == 0;
        for (const KvStrides& st : {ks, vs})
            wide = wide && st.token % N == 0 && st.head % N == 0;
        return launch_parts((int64_t)grid, [&](dim3 blocks, uint32_t first) {
            append_rows_kernel<T, decltype(bits)::value, decltype(dim)::value>
                <<<blocks, dim3(kBlock), 0, stream>>>(c, (uint32_t)tokens, slots,
                                                      static_cast<const T*>(k), ks,
                                                      static_cast<const T*>(v), vs, wide, first);
        });
    });
}

template <class T>
hipError_t read_typed(const cq_kv_cache_t& c, const cq_kv_slots_t& s, void* k, void* v,
                      hipStream_t stream) {
    const int64_t tiles = tiles_of(s), grid = workgroups(c, s);
    if (grid > kMaxGrid) return hipErrorInvalidValue;
    return by_form(c, [&](auto bits, auto dim) {
        return launch_parts(grid, [&](dim3 blocks, uint32_t first) {
            read_kernel<T, decltype(bits)::value, decltype(dim)::value>
                <<<blocks, dim3(kBlock), 0, stream>>>(c, s, (uint32_t)tiles, static_cast<T*>(k),
                                                      static_cast<T*>(v), first);
        });
    });
}

}  // namespace

hipError_t launch_kv_append(const cq_kv_cache_t& c, const cq_kv_slots_t& s, int dtype,
                            const void* k, KvStrides ks, const void* v, KvStrides vs,
                            hipStream_t stream) {
    if (dtype == CQ_DTYPE_F16) return append_typed<_Float16>(c, s, k, ks, v, vs, stream);
    if (dtype == CQ_DTYPE_BF16) return append_typed<__bf16>(c, s, k, ks, v, vs, stream);
    return append_typed<float>(c, s, k, ks, v, vs, stream);
}

hipError_t launch_kv_append_rows(const cq_kv_cache_t& c, int dtype, int64_t tokens,
                                 const int64_t* slots, const void* k, KvStrides ks, const void* v,
                                 KvStrides vs, hipStream_t stream) {
    if (dtype == CQ_DTYPE_F16)
        return append_rows_typed<_Float16>(c, tokens, slots, k, ks, v, vs, stream);
    if (dtype == CQ_DTYPE_BF16)
        return append_rows_typed<__bf16>(c, tokens, slots, k, ks, v, vs, stream);
    return append_rows_typed<float>(c, tokens, slots, k, ks, v, vs, stream);
}

hipError_t launch_kv_read(const cq_kv_cache_t& c, const cq_kv_slots_t& s, int dtype,
                          void* k_out, void* v_out, hipStream_t stream) {
    if (dtype == CQ_DTYPE_F16) return read_typed<_Float16>(c, s, k_out, v_out, stream);
    if (dtype == CQ_DTYPE_BF16) return read_typed<__bf16>(c, s, k_out, v_out, stream);
    return read_typed<float>(c, s, k_out, v_out, stream);
}

}  // namespace cq
