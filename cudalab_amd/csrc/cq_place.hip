// Pages, slots and positions of a packed batch, from the requests' lengths
// (gfx950).
//
//   n_b      tokens that sequence b adds, offsets_b = n_0 + .. + n_{b-1}
//   have_b   ceil(start_b / page) pages that it holds, or as many as the caller
//            says, where those are more: pages taken for tokens that were given up
//   need_b   max(0, ceil((start_b + n_b) / page) - have_b) pages that it gets,
//   first_b  need_0 + .. + need_{b-1}, its place in the free list
// and token t of the packed batch, in sequence b with offsets_b <= t, has the
// position p = start_b + t - offsets_b, the page of column c = p / page (the
// table's entry for c < have_b, else free[first_b + c - have_b]) and the slot
// page * size + p % size.
//
// Bound by its launch and by loads that follow one another: counts, the table's
// or the list's entry, the store.  So it is one launch, in which every workgroup
// scans the lengths by itself, 256 at a time, and then finds its own tokens'
// sequences by bisection in LDS.  A new page begins at a token of the call,
// which also writes the table's entry; entries that are read are those that the
// sequences held before, so no workgroup waits for another.  256 sequences of one
// token 3.0 us, 64 prompts of up to 4096 (131 workgroups) 4.8, where a launch that
// does nothing takes 1.8 (1.6 in a graph, of which the first case takes 3.5 there).

#include "cq_elem.h"
#include "cq_step.h"

namespace cq {
namespace {

constexpr int kBlock = 256;
constexpr int kEach = 2;                       // tokens of a thread
constexpr uint32_t kTokens = kBlock * kEach;   // of a workgroup
constexpr uint32_t kMost = 0x7FFFFFFF;

// Inclusive sums over the workgroup, capped at `cap`: adding with a cap is
// associative over numbers that are not negative, and cap + cap < 2^32.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t cap, uint32_t* waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t up = (uint32_t)__shfl_up((int)v, off);
        if (lane >= off) v = min(v + up, cap);
    }
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v = min(v + waves[w], cap);
    __syncthreads();
    return v;
}

// HELD: with counts of held pages (either may be null).
template <bool HELD>
__global__ __launch_bounds__(kBlock) void place_kernel(cq_place_t a, uint32_t first_block,
                                                       const int32_t* held_in, int32_t* held_out) {
    __shared__ uint32_t sums[kBlock / 64];
    // of 256 sequences: where their tokens end, begin and start, and their pages
    __shared__ uint32_t end[kBlock], begin[kBlock], start[kBlock], have[kBlock], page0[kBlock];
    const uint32_t tid = threadIdx.x, block = first_block + blockIdx.x;
    const uint32_t tokens = (uint32_t)a.tokens, page = (uint32_t)a.page_size;
    const uint32_t t0 = block * kTokens;
    const int shift = __builtin_ctz(page);
    const uint32_t room = (uint32_t)a.table_cols << shift;     // below 2^31
    const uint32_t taken = a.taken_in != nullptr ? (uint32_t)max(0, *a.taken_in) : 0;
    uint32_t placed = 0, pages = 0;            // of the sequences before these 256
    for (uint32_t base = 0; base < (uint32_t)a.batch; base += kBlock) {
        const uint32_t b = base + tid;
        uint32_t n = 0, s = 0, own = 0;
        if (b < (uint32_t)a.batch) {
            n = (uint32_t)max(0, a.counts[b]);
            s = (uint32_t)max(0, a.starts[b]);
            if (HELD && held_in != nullptr) own = (uint32_t)max(0, held_in[b]);
        }
        // what does not fit the call's tokens is not placed
        const uint32_t upto = min(placed + block_scan(min(n, tokens), tokens, sums), tokens);
        end[tid] = upto;
        if (tid == 0) begin[0] = placed;
        if (tid + 1 < kBlock) begin[tid + 1] = upto;
        __syncthreads();
        n = upto - begin[tid];
        const uint32_t held = max(s / page + (s % page != 0), own);
        const uint32_t last = min(s + n, room);
        const uint32_t want = last / page + (last % page != 0);
        const uint32_t need = n > 0 && want > held ? want - held : 0;
        const uint32_t sum = block_scan(need, kMost, sums);
        start[tid] = s;
        have[tid] = held;
        page0[tid] = min(pages + sum - need, kMost);
        if (block == 0 && b < (uint32_t)a.batch) {
            if (b == 0) a.offsets[0] = 0;
            a.offsets[b + 1] = (int32_t)upto;
            a.lengths[b] = (int32_t)min(s + n, kMost);
            if (HELD && held_out != nullptr) {         // of the pages it needs those that the list has
                const uint64_t at = (uint64_t)taken + page0[tid];
                const uint64_t left =
                    (uint64_t)a.free_count > at ? (uint64_t)a.free_count - at : 0;
                held_out[b] = (int32_t)min((uint64_t)held + min((uint64_t)need, left),
                                           (uint64_t)kMost);
            }
        }
        __syncthreads();
        const uint32_t lo = begin[0], hi = end[kBlock - 1];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t t = t0 + i * kBlock + tid;
            if (t < lo || t >= hi) continue;
            uint32_t e = 0;                    // the first with end > t
#pragma unroll
            for (int step = kBlock / 2; step > 0; step >>= 1)
                if (end[e + step - 1] <= t) e += step;
            const uint32_t pos = start[e] + (t - begin[e]);
            const uint32_t col = pos >> shift, off = pos & (page - 1);
            int32_t entry = -1;
            if (col < (uint32_t)a.table_cols) {
                int32_t* at = a.table + (int64_t)(base + e) * a.table_stride + col;
                if (col < have[e]) {
                    entry = *at;
                } else {
                    const uint64_t index = (uint64_t)taken + page0[e] + (col - have[e]);
                    if (index < (uint64_t)a.free_count) entry = a.free_pages[index];
                    if (off == 0) *at = entry;
                }
            }
            a.slots[t] = entry >= 0 ? ((int64_t)entry << shift) + off : -1;
            a.positions[t] = (int32_t)min(pos, kMost);
        }
        if (tid == kBlock - 1) sums[0] = sum;
        __syncthreads();
        placed = hi;
        pages = min(pages + sums[0], kMost);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {          // rows behind the last sequence
        const uint32_t t = t0 + i * kBlock + tid;
        if (t >= placed && t < tokens) {
            a.slots[t] = -1;
            a.positions[t] = 0;
        }
    }
    if (block == 0 && tid == 0) a.taken_out[0] = (int32_t)min(taken + pages, kMost);
}

}  // namespace

hipError_t launch_place_held(const cq_place_t& a, const int32_t* held_in, int32_t* held_out,
                             hipStream_t stream) {
    const int64_t grid = std::max<int64_t>(1, (a.tokens + kTokens - 1) / kTokens);
    return launch_parts(grid, [&](dim3 blocks, uint32_t first) {
        if (held_in != nullptr || held_out != nullptr)
            place_kernel<true><<<blocks, dim3(kBlock), 0, stream>>>(a, first, held_in, held_out);
        else
            place_kernel<false><<<blocks, dim3(kBlock), 0, stream>>>(a, first, nullptr, nullptr);
    });
}

hipError_t launch_place(const cq_place_t& a, hipStream_t stream) {
    return launch_place_held(a, nullptr, nullptr, stream);
}

}  // namespace cq
