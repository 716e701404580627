// The argument checks of the calls of a step of many tokens (cq_step_capi.cpp) to
// their ends, under AddressSanitizer and UndefinedBehaviorSanitizer: mixtures of
// sizes, strides and pointers at the ends of their types, of which some are
// accepted.  The launchers behind the checks are stubs here that only count, so
// nothing is launched and no pointer followed.  Built and run by
// tests/test_host_sanitizers_step_cpu.py.
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <string>

#include "cq_step.h"

static long reached[6];
static std::string text;

namespace cq {
int set_error(int code, const std::string& msg) {
    text = msg;
    return code;
}
hipError_t launch_norm_rope(const cq_norm_rope_t&, hipStream_t) { return hipSuccess; }
hipError_t launch_kv_append(const cq_kv_cache_t&, const cq_kv_slots_t&, int, const void*, KvStrides,
                            const void*, KvStrides, hipStream_t) {
    return hipSuccess;
}
hipError_t launch_kv_read(const cq_kv_cache_t&, const cq_kv_slots_t&, int, void*, void*,
                          hipStream_t) {
    return hipSuccess;
}
int64_t attention_workspace(const cq_kv_cache_t&, const cq_attention_t&) { return 1 << 20; }
hipError_t launch_attention(const cq_kv_cache_t&, const cq_attention_t&, hipStream_t) {
    return hipSuccess;
}
hipError_t launch_place(const cq_place_t&, hipStream_t) { return ++reached[0], hipSuccess; }
hipError_t launch_kv_append_rows(const cq_kv_cache_t&, int, int64_t, const int64_t*, const void*,
                                 KvStrides, const void*, KvStrides, hipStream_t) {
    return ++reached[1], hipSuccess;
}
hipError_t launch_prompt(const cq_prompt_t&, hipStream_t) { return ++reached[2], hipSuccess; }
int64_t attention_tree_workspace(const cq_kv_cache_t&, const cq_attention_t&) { return 1 << 19; }
hipError_t launch_attention_tree(const cq_kv_cache_t&, const cq_attention_t&, const int64_t*,
                                 hipStream_t) {
    return ++reached[3], hipSuccess;
}
hipError_t launch_quantize_tokens(int, const void*, int64_t, int64_t, int64_t, int8_t*, float*,
                                  hipStream_t) {
    return ++reached[4], hipSuccess;
}
int64_t qgemm_workspace(const cq_qgemm_t& a) { return a.k % 4 ? 1 << 18 : 0; }
hipError_t launch_qgemm(const cq_qgemm_t&, hipStream_t) { return ++reached[5], hipSuccess; }
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
// `usual` as a rule, now and then one of x.
template <class T, class X, int N>
static T mostly(T usual, const X (&x)[N]) { return next() % 24 ? usual : static_cast<T>(pick(x)); }

int main() {
    const int32_t ints[] = {INT_MIN, -1, 0, 1, 2, 16, 65535, 65536, 1 << 20, INT_MAX - 63, INT_MAX};
    const int64_t longs[] = {INT64_MIN, -8, 0, 1, 8, 128, 1024, (int64_t)1 << 24,
                             (int64_t)1 << 33, (int64_t)1 << 40, ((int64_t)1 << 40) + 8, INT64_MAX};
    char* const P = (char*)0x100000000000ull;
    auto at = [&](int i) { return P + ((int64_t)i << 44); };     // far from one another
    long refused = 0, wrong = 0;
    auto ptr = [&](int i) -> char* {
        switch (next() % 32) {
            case 0: return nullptr;
            case 1: return at(i) + next() % 17;
            case 2: return at(next() % 10) + 16 * (next() % 64);
            default: return at(i);
        }
    };
    auto count = [&](int st) {
        if (st != CQ_OK) ++refused;
        if (st != CQ_OK && st != CQ_ERR_INVALID_ARG && st != CQ_ERR_BUFFER_TOO_SMALL) ++wrong;
    };
    for (long i = 0; i < 400000; ++i) {
        cq_kv_cache_t c{ptr(0), ptr(1), (float*)ptr(2), mostly<int64_t>(64, longs),
                        mostly<int32_t>(8, ints), mostly<int32_t>(128, ints),
                        mostly<int32_t>(64, ints), mostly<int32_t>(8, ints)};
        switch (i % 6) {
            case 0: {
                cq_place_t a{(int32_t*)ptr(0), (int32_t*)ptr(1), (int32_t*)ptr(2), (int32_t*)ptr(3),
                             (int32_t*)ptr(4), (int64_t*)ptr(5), (int32_t*)ptr(6), (int32_t*)ptr(7),
                             (int32_t*)ptr(8), (int32_t*)ptr(9), mostly<int64_t>(40, longs),
                             mostly<int64_t>(1000, longs), mostly<int64_t>(500, longs),
                             mostly<int32_t>(32, ints), mostly<int32_t>(16, ints),
                             mostly<int32_t>(64, ints)};
                count(cq_place(&a, nullptr));
                break;
            }
            case 1:
                count(cq_kv_append_rows(&c, (int)(next() % 4), mostly<int64_t>(77, longs),
                                        (int64_t*)ptr(3), ptr(4), mostly<int64_t>(1024, longs),
                                        mostly<int64_t>(128, longs), ptr(5),
                                        mostly<int64_t>(1024, longs), mostly<int64_t>(128, longs),
                                        nullptr));
                break;
            case 2: {
                cq_prompt_t a{ptr(0), ptr(1), ptr(2), ptr(3), mostly<int64_t>(8192, longs),
                              mostly<int64_t>(128, longs), mostly<int64_t>(1024, longs),
                              mostly<int64_t>(128, longs), mostly<int64_t>(1024, longs),
                              mostly<int64_t>(128, longs), (int32_t*)ptr(4), (int32_t*)ptr(5),
                              mostly<int64_t>(300, longs), mostly<int64_t>(400, longs),
                              mostly<int32_t>(3, ints), mostly<int32_t>(64, ints),
                              mostly<int32_t>(8, ints), mostly<int32_t>(128, ints),
                              (int32_t)(next() % 2 * 2), (int32_t)(next() % 2),
                              next() % 16 ? 0.1f : INFINITY};
                count(cq_prompt_attention(&a, nullptr));
                break;
            }
            case 3: {
                cq_attention_t a{};
                a.q = ptr(3), a.out = ptr(4);
                a.q_batch_stride = mostly<int64_t>(8192, longs);
                a.q_token_stride = mostly<int64_t>(1024, longs);
                a.q_head_stride = mostly<int64_t>(128, longs);
                a.table = (int32_t*)ptr(5), a.lengths = (int32_t*)ptr(6);
                a.table_stride = 9, a.workspace = ptr(7), a.workspace_bytes = 1 << 20;
                a.table_cols = mostly<int32_t>(9, ints);
                a.batch = mostly<int32_t>(3, ints), a.tokens = mostly<int32_t>(8, ints);
                a.q_heads = mostly<int32_t>(8, ints), a.softmax_scale = 0.1f;
                count(cq_attention_tree(&c, &a, (int64_t*)ptr(8), nullptr));
                if (cq_attention_tree_workspace(&c, &a) == 0) ++wrong;
                break;
            }
            case 4:
                count(cq_quantize_tokens((int)(next() % 4), ptr(0), mostly<int64_t>(512, longs),
                                         mostly<int64_t>(99, longs), mostly<int64_t>(512, longs),
                                         (int8_t*)ptr(1), (float*)ptr(2), nullptr));
                break;
            default: {
                cq_qgemm_t a{(int8_t*)ptr(0), (float*)ptr(1), (int8_t*)ptr(2), (float*)ptr(3), ptr(4),
                             mostly<int64_t>(512, longs), mostly<int64_t>(99, longs),
                             mostly<int64_t>(300, longs), mostly<int64_t>(510 + i / 6 % 2 * 2, longs),
                             ptr(5), 1 << 20, (int32_t)(next() % 4)};
                count(cq_qgemm(&a, nullptr));
                const int64_t need = cq_qgemm_workspace(&a);
                if (need < 0 && need != -CQ_ERR_INVALID_ARG) ++wrong;
            }
        }
    }
    for (long n : reached)
        if (n == 0) ++wrong;
    std::printf("refused %s, reached %ld %ld %ld %ld %ld %ld, wrong %ld\ndone\n",
                refused > 0 ? "some" : "none", reached[0], reached[1], reached[2], reached[3],
                reached[4], reached[5], wrong);
    return wrong != 0 || refused == 0;
}
