// C entry point of place with counts of held pages (declared in
// include/cdnaqgemv.h), apart from cq_step_capi.cpp's, which need no launcher of
// it.

#include "cq_checks.h"
#include "cq_step.h"

using namespace cq::checks;

extern "C" int cq_place_held(const cq_place_t* args, const int32_t* held_in, int32_t* held_out,
                             void* stream) {
    return guarded([&]() -> int {
        if (args == nullptr) return invalid("null pointer: args");
        const int st = check_place(*args, held_in, held_out);
        if (st != CQ_OK) return st;
        return hip_status(cq::launch_place_held(*args, held_in, held_out,
                                                static_cast<hipStream_t>(stream)),
                          "cq_place_held");
    });
}
