// gn_linear_act_bwd.hip — the backward's product of gn_linear_act.hip, dP = (dY W) act'(P).
#include "gn_linear_act_core.h"

namespace gn {
namespace {

template <bool VEC>
int backward(const GemmDesc& d, int act, const void* P, void* dP, int N, hipStream_t s) {
    auto make = [&](auto A) { return Backward<VEC, decltype(A)::value>{(const bf16_t*)P, (bf16_t*)dP, N, act}; };
    using std::integral_constant;
    return launch<false>(d, make(integral_constant<int, kAny>{}), [&](auto&& go) {
        switch (act) {
            case GN_ACT_RELU: return go(make(integral_constant<int, GN_ACT_RELU>{}));
            case GN_ACT_GELU_TANH: return go(make(integral_constant<int, GN_ACT_GELU_TANH>{}));
            case GN_ACT_GELU_ERF: return go(make(integral_constant<int, GN_ACT_GELU_ERF>{}));
            case GN_ACT_SILU: return go(make(integral_constant<int, GN_ACT_SILU>{}));
            case GN_ACT_TANH: return go(make(integral_constant<int, GN_ACT_TANH>{}));
            default: return go(make(integral_constant<int, GN_ACT_SIGMOID>{}));
        }
    }, s);
}

}  // namespace

int act_linear_dp(const GemmDesc& d, int act, const void* P, void* dP, int N, bool vec, hipStream_t s) {
    return vec ? backward<true>(d, act, P, dP, N, s) : backward<false>(d, act, P, dP, N, s);
}

}  // namespace gn
