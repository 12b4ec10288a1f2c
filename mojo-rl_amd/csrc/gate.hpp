// The logistic function of the gated layers.
#pragma once
#include "mrl_device.hpp"

namespace mrl {

// sigmoid(g) and 1 - sigmoid(g), each relative to its own value: e = exp(-g) is 2^y with what rounding y left taken back, the reciprocal
// takes a Newton step.  The argument is held where e stays finite.  (minimum and maximum keep NaN.)
MRL_DEV void sigmoid_pair(float g, float &a, float &rest) {
    g = __builtin_elementwise_minimum(__builtin_elementwise_maximum(g, -87.0f), 200.0f);
    const float y = g * -1.44269502f;
    float e = __builtin_amdgcn_exp2f(y);
    e = fmaf(e, fmaf(y, -0.693147182f, -g), e);
    const float u = 1.0f + e;
    a = __builtin_amdgcn_rcpf(u);
    a = fmaf(a, fmaf(-u, a, 1.0f), a);
    rest = e * a;
}

}  // namespace mrl
