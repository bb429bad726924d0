// gn_linear_act_bf16.hip — the forward products of gn_linear_act.hip with Y in bf16.
#include "gn_linear_act_core.h"

namespace gn {

int linear_act_bf16(const GemmDesc& d, int act, const void* b, const void* R, void* Y, void* P, bool vec, hipStream_t s) {
    return vec ? forward<bf16_t, true>(d, act, b, R, Y, P, s) : forward<bf16_t, false>(d, act, b, R, Y, P, s);
}

}  // namespace gn
