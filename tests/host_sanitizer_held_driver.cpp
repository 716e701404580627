// The checks of place with counts of held pages (cq_place_capi.cpp) to their ends,
// under AddressSanitizer and UndefinedBehaviorSanitizer, as
// host_sanitizer_step_driver.cpp has the other calls'.  The launcher is a stub that
// counts.  Built and run by tests/test_host_sanitizers_held_cpu.py.
#include <climits>
#include <cstdint>
#include <cstdio>
#include <string>

#include "cq_step.h"

static long reached;

namespace cq {
int set_error(int code, const std::string&) { return code; }
hipError_t launch_place_held(const cq_place_t&, const int32_t*, int32_t*, hipStream_t) {
    return ++reached, hipSuccess;
}
}  // namespace cq

static uint64_t state = 88172645463325252ull;
static uint64_t next() {
    state ^= state << 13;
    state ^= state >> 7;
    state ^= state << 17;
    return state;
}
template <class T, class X, int N>
static T mostly(T usual, const X (&x)[N]) {
    return next() % 24 ? usual : static_cast<T>(x[next() % N]);
}

int main() {
    const int32_t ints[] = {INT_MIN, -1, 0, 1, 16, 65536, INT_MAX - 1, INT_MAX};
    const int64_t longs[] = {INT64_MIN, -8, 0, 1, 128, (int64_t)1 << 31, (int64_t)1 << 40,
                             INT64_MAX};
    char* const P = (char*)0x100000000000ull;
    auto ptr = [&](int i) -> char* {
        char* const at = P + ((int64_t)i << 42);
        switch (next() % 40) {
            case 0: return nullptr;
            case 1: return at + next() % 9;
            case 2: return P + ((int64_t)(next() % 12) << 42) + 4 * (next() % 64);
            default: return at;
        }
    };
    long refused = 0, wrong = 0;
    for (long i = 0; i < 200000; ++i) {
        cq_place_t a{(int32_t*)ptr(0), (int32_t*)ptr(1), (int32_t*)ptr(2), (int32_t*)ptr(3),
                     (int32_t*)ptr(4), (int64_t*)ptr(5), (int32_t*)ptr(6), (int32_t*)ptr(7),
                     (int32_t*)ptr(8), (int32_t*)ptr(9), mostly<int64_t>(40, longs),
                     mostly<int64_t>(1000, longs), mostly<int64_t>(500, longs),
                     mostly<int32_t>(32, ints), mostly<int32_t>(16, ints), mostly<int32_t>(64, ints)};
        const int st = cq_place_held(&a, (int32_t*)ptr(10), (int32_t*)ptr(11), nullptr);
        if (st != CQ_OK) ++refused;
        if (st != CQ_OK && st != CQ_ERR_INVALID_ARG) ++wrong;
    }
    std::printf("refused %ld, reached %ld, wrong %ld\ndone\n", refused, reached, wrong);
    return wrong != 0 || refused == 0 || reached == 0;
}
