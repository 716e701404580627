// Host-only exercise of the calls around attention (include/cdnaqgemv.h) under
// AddressSanitizer and UndefinedBehaviorSanitizer: sizes, strides and pointers
// at the ends of their types, in many mixtures.  Nothing here launches a
// kernel: cq_attention_workspace only plans, and every other call names an
// output that is one of its inputs, or a null pointer, and is refused.  Built
// and run by tests/test_host_sanitizers_attention_cpu.py.
#include "cdnaqgemv.h"
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstring>

static uint64_t state = 88172645463325252ull;
static uint64_t next() {
    state ^= state << 13;
    state ^= state >> 7;
    state ^= state << 17;
    return state;
}
template <class T, int N>
static T pick(const T (&x)[N]) { return x[next() % N]; }

int main() {
    const int32_t ints[] = {INT_MIN, -1, 0, 1, 2, 5, 8, 16, 63, 64, 128, 1000, 65535, 65536,
                            1 << 20, (1 << 25) + 1, INT_MAX - 63, INT_MAX};
    const int64_t longs[] = {INT64_MIN, -8, 0, 8, 128, 1024, 1 << 20, (int64_t)1 << 33,
                             (int64_t)1 << 40, ((int64_t)1 << 40) + 8, INT64_MAX};
    const int32_t dims[] = {64, 128, 256, 100}, pages[] = {16, 64, 256, 24}, bits[] = {4, 8, 5};
    char* P = (char*)0x100000000000ull;
    long refused = 0, planned = 0, wrong = 0;
    for (int i = 0; i < 200000; ++i) {
        cq_kv_cache_t c{P, P + ((int64_t)1 << 44), (float*)(P + ((int64_t)1 << 45)),
                        next() % 2 ? (int64_t)1000 : pick(longs), next() % 2 ? 8 : pick(ints),
                        pick(dims), pick(pages), pick(bits)};
        cq_attention_t a;
        std::memset(&a, 0, sizeof a);
        a.q = P;
        a.out = next() % 4 ? (void*)P : nullptr;         // q itself, or none: refused
        a.q_batch_stride = pick(longs);
        a.q_token_stride = pick(longs);
        a.q_head_stride = pick(longs);
        a.table = (const int32_t*)(P + 64);
        a.lengths = (const int32_t*)(P + 128);
        a.table_stride = pick(longs);
        a.table_cols = pick(ints);
        a.prefix_cols = pick(ints);
        a.prefix_len = next() % 2 ? 0 : pick(ints);
        a.prefix_table = next() % 2 ? nullptr : (const int32_t*)(P + 4);
        a.batch = pick(ints);
        a.tokens = pick(ints);
        a.q_heads = next() % 2 ? 64 : pick(ints);
        a.dtype = (int32_t)(next() % 4);
        a.softmax_scale = next() % 8 ? 0.1f : __builtin_inff();
        a.workspace = P + ((int64_t)1 << 46);
        a.workspace_bytes = INT64_MAX;
        const int64_t need = cq_attention_workspace(&c, &a);
        need < 0 ? ++refused : ++planned;
        if (cq_attention(&c, &a, nullptr) == CQ_OK) ++wrong;
        cq_kv_slots_t s{(const int32_t*)(P + 64), (const int32_t*)(P + 128), nullptr, pick(longs),
                        pick(ints), pick(ints), pick(ints)};
        const int dt = (int)(next() % 4);
        // k is the cache's own memory; the two outputs are one
        if (cq_kv_append(&c, &s, dt, P, pick(longs), pick(longs), pick(longs), P, pick(longs),
                         pick(longs), pick(longs), nullptr) == CQ_OK)
            ++wrong;
        if (cq_kv_read(&c, &s, dt, P + 256, P + 256, nullptr) == CQ_OK) ++wrong;
        cq_norm_rope_t n;
        std::memset(&n, 0, sizeof n);
        n.q = P;
        n.k = P;
        n.q_out = n.k_out = nullptr;                     // refused, also without heads
        n.q_token_stride = pick(longs);
        n.q_head_stride = pick(longs);
        n.k_token_stride = pick(longs);
        n.k_head_stride = pick(longs);
        n.q_weight = P;
        n.cos_table = next() % 2 ? nullptr : (const float*)P;
        n.sin_table = n.cos_table;
        n.positions = P;
        n.tokens = pick(longs);
        n.table_rows = pick(longs);
        n.q_heads = 1 + (int32_t)(next() % 70000);
        n.k_heads = pick(ints);
        n.head_dim = pick(dims);
        n.rot_dim = pick(ints);
        n.dtype = dt;
        n.weight_dtype = (int32_t)(next() % 4);
        n.eps = 1e-6f;
        if (cq_qk_norm_rope(&n, nullptr) == CQ_OK) ++wrong;
    }
    std::printf("refused %s, planned %s, wrong %ld\ndone\n", refused > 0 ? "some" : "none",
                planned > 0 ? "some" : "none", wrong);
    return wrong == 0 ? 0 : 1;
}
