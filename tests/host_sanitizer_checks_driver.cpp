// The argument checks of the calls around attention (cq_attn_capi.cpp) to
// their ends, under AddressSanitizer and UndefinedBehaviorSanitizer: mixtures
// of sizes, strides and pointers at the ends of their types, of which some are
// accepted.  The launchers behind the checks are stubs here that only count, so
// nothing is launched and no pointer followed.  Built and run by
// tests/test_host_sanitizers_checks_cpu.py.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>

#include "cq_attn.h"

static long reached[4];
static std::string text;

namespace cq {
int set_error(int code, const std::string& msg) {
    text = msg;
    return code;
}
hipError_t launch_norm_rope(const cq_norm_rope_t&, hipStream_t) { return ++reached[0], hipSuccess; }
hipError_t launch_kv_append(const cq_kv_cache_t&, const cq_kv_slots_t&, int, const void*, KvStrides,
                            const void*, KvStrides, hipStream_t) {
    return ++reached[1], hipSuccess;
}
hipError_t launch_kv_read(const cq_kv_cache_t&, const cq_kv_slots_t&, int, void*, void*,
                          hipStream_t) {
    return ++reached[2], hipSuccess;
}
int64_t attention_workspace(const cq_kv_cache_t&, const cq_attention_t&) { return 1 << 20; }
hipError_t launch_attention(const cq_kv_cache_t&, const cq_attention_t&, hipStream_t) {
    return ++reached[3], hipSuccess;
}
}  // namespace cq

static uint64_t state = 88172645463325252ull;
static uint64_t next() {
    state ^= state << 13;
    state ^= state >> 7;
    state ^= state << 17;
    return state;
}
template <class T, int N>
static T pick(const T (&x)[N]) { return x[next() % N]; }
template <class T, int N>
static T mostly(T usual, const T (&x)[N]) { return next() % 16 ? usual : pick(x); }

int main() {
    const int32_t ints[] = {INT_MIN, -1, 0, 1, 2, 16, 65535, 65536, 1 << 20, INT_MAX - 63, INT_MAX};
    const int64_t longs[] = {INT64_MIN, -8, 0, 8, 128, 1024, (int64_t)1 << 33, (int64_t)1 << 40,
                             ((int64_t)1 << 40) + 8, INT64_MAX};
    const int64_t near[] = {0, 64, 128, 256, 512, 1024, 4096, 65536};
    char* const P = (char*)0x100000000000ull;
    auto at = [&](int i) { return P + ((int64_t)i << 44); };     // far from one another
    long overlaps = 0, interleaved = 0, last = 0, wrong = 0;
    auto count = [&](int st, bool plain) {
        if (st == CQ_OK) return;
        if (plain) ++wrong;
        if (text.find("overlap") != std::string::npos) ++overlaps;
        if (text.find("a weight, a table or the positions") != std::string::npos) ++last;
    };
    for (int i = 0; i < 400000; ++i) {
        cq_norm_rope_t n;
        std::memset(&n, 0, sizeof n);
        n.q_heads = mostly(8, ints);
        n.k_heads = mostly(2, ints);
        n.head_dim = mostly(128, ints);
        n.tokens = mostly((int64_t)9, longs);
        const bool fused = next() % 2;           // q and k side by side, in place
        n.q = at(1);
        n.k = fused ? at(1) + 2 * 128 * 8 : at(2);
        n.q_token_stride = mostly(fused ? (int64_t)1280 : (int64_t)1024, longs);
        n.k_token_stride = mostly(fused ? n.q_token_stride : (int64_t)256, longs);
        n.q_head_stride = mostly((int64_t)128, longs);
        n.k_head_stride = mostly((int64_t)128, longs);
        n.q_out = fused ? const_cast<void*>(n.q) : next() % 8 ? at(3) : at(1) + pick(near);
        n.k_out = fused ? const_cast<void*>(n.k) : next() % 8 ? at(4) : at(3) + pick(near);
        n.q_out_token_stride = mostly(n.q_token_stride, longs);
        n.q_out_head_stride = mostly(n.q_head_stride, longs);
        n.k_out_token_stride = mostly(n.k_token_stride, longs);
        n.k_out_head_stride = mostly(n.k_head_stride, longs);
        n.q_weight = next() % 8 ? at(5) : (char*)n.q_out + pick(near);
        n.k_weight = at(6);
        n.cos_table = next() % 4 ? (const float*)at(7) : nullptr;
        n.sin_table = n.cos_table == nullptr ? nullptr : (const float*)at(8);
        n.positions = next() % 8 ? at(9) : (char*)n.k_out + pick(near);
        n.table_rows = mostly((int64_t)4096, longs);
        n.rot_dim = mostly(64, ints);
        n.eps = 1e-6f;
        const long before = reached[0];
        count(cq_qk_norm_rope(&n, nullptr), false);
        if (fused && reached[0] > before) ++interleaved;

        cq_kv_cache_t c{at(1), at(2), (float*)at(3), mostly((int64_t)1000, longs),
                        mostly(8, ints), 128, 64, 8};
        cq_kv_slots_t s{(const int32_t*)at(4), (const int32_t*)at(5),
                        next() % 2 ? (const int32_t*)at(6) : nullptr, mostly((int64_t)5, longs),
                        mostly(5, ints), mostly(3, ints), mostly(7, ints)};
        auto where = [&](int k) { return next() % 8 ? at(k) : at(1) + (int64_t)pick(near); };
        count(cq_kv_append(&c, &s, (int)(next() % 4), where(7), mostly((int64_t)7168, longs),
                           mostly((int64_t)1024, longs), mostly((int64_t)128, longs), where(8),
                           mostly((int64_t)7168, longs), mostly((int64_t)1024, longs),
                           mostly((int64_t)128, longs), nullptr), false);
        count(cq_kv_read(&c, &s, (int)(next() % 4), where(7), where(8), nullptr), false);

        cq_attention_t a;
        std::memset(&a, 0, sizeof a);
        a.q = where(7);
        a.out = next() % 8 ? at(8) : at(7) + pick(near);
        a.q_batch_stride = mostly((int64_t)65536, longs);
        a.q_token_stride = mostly((int64_t)8192, longs);
        a.q_head_stride = mostly((int64_t)128, longs);
        a.table = s.table;
        a.lengths = s.starts;
        a.counts = s.counts;
        a.prefix_table = (const int32_t*)at(9);
        a.table_stride = mostly((int64_t)5, longs);
        a.workspace = next() % 8 ? at(10) : at(8) + pick(near);
        a.workspace_bytes = mostly((int64_t)1 << 20, longs);
        a.table_cols = mostly(5, ints);
        a.prefix_cols = mostly(3, ints);
        a.prefix_len = mostly(150, ints);
        a.batch = mostly(3, ints);
        a.tokens = mostly(2, ints);
        a.q_heads = mostly(64, ints);
        a.dtype = next() % 2 ? CQ_DTYPE_F16 : CQ_DTYPE_BF16;
        a.softmax_scale = 0.1f;
        count(cq_attention(&c, &a, nullptr), false);
    }
    // the plain calls themselves are accepted
    cq_kv_cache_t c{at(1), at(2), (float*)at(3), 1000, 8, 128, 64, 8};
    cq_kv_slots_t s{(const int32_t*)at(4), (const int32_t*)at(5), nullptr, 5, 5, 3, 7};
    count(cq_kv_append(&c, &s, CQ_DTYPE_F16, at(7), 7168, 1024, 128, at(8), 7168, 1024, 128,
                       nullptr), true);
    count(cq_kv_read(&c, &s, CQ_DTYPE_BF16, at(7), at(8), nullptr), true);
    std::printf("norms %ld, interleaved %ld, appends %ld, reads %ld, attention %ld\n", reached[0],
                interleaved, reached[1], reached[2], reached[3]);
    std::printf("overlaps %ld, at the last check %ld, wrong %ld\n", overlaps, last, wrong);
    const bool all = reached[0] > 1000 && interleaved > 1000 && reached[1] > 1000 &&
                     reached[2] > 1000 && reached[3] > 1000 && overlaps > 1000 && last > 1000;
    std::printf("%s\n", all && wrong == 0 ? "done" : "not all checks reached");
    return all && wrong == 0 ? 0 : 1;
}
