// ssm_ops.h — the scalar functions that the state space mixers' kernels share.
#pragma once

#include "hip_common.h"

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// 2^x by the hardware's instruction, off by at most one unit
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// log(1 + e^x) = max(x, 0) + log1p(u), u = e^-|x|, with log1p(u) = 2 atanh(s), s = u / (2 + u) <= 1/3, as
// its series: nine terms leave 3^-19 / 19 < 2^-34 of s. u keeps the rounding of |x| log2(e) as a factor.
// Within four units over all x, and below -88, where u underflows, 0.
__device__ __forceinline__ float softplus(float x) {
    const float z = -fabsf(x), t = z * LOG2E;
    const float r = fmaf(z, LOG2E, -t) + z * 1.92596299e-8f;      // log2(e) - float(log2(e))
    const float u = z < -88.0f ? 0.0f : exp2_hw(t) * fmaf(r, LN2, 1.0f);
    const float s = u * __builtin_amdgcn_rcpf(2.0f + u), q = s * s;
    float p = 1.0f / 17.0f;
    p = fmaf(p, q, 1.0f / 15.0f);
    p = fmaf(p, q, 1.0f / 13.0f);
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    p = p * q;
    // a NaN stays one
    return x != x ? x : fmaxf(x, 0.0f) + 2.0f * fmaf(s, p, s);
}
