// gn_linear_act_f32.hip — the forward products of gn_linear_act.hip with Y in f32.
#include "gn_linear_act_core.h"

namespace gn {

int linear_act_f32(const GemmDesc& d, int act, const void* b, const void* R, void* Y, void* P, bool vec, hipStream_t s) {
    return vec ? forward<float, true>(d, act, b, R, Y, P, s) : forward<float, false>(d, act, b, R, Y, P, s);
}

}  // namespace gn
