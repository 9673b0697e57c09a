// exp, silu and softplus of the state space and group norm kernels: fp32, off by a few roundings of the result or, where that is more, by 2^-119: below the normal numbers the
// instructions give 0, and with them what stands on 1 / (1 + e^-x) from x = -87 down.  Infinities and NaN as the formulas bring them.
#pragma once

namespace eddlhip {

constexpr float LOG2_E = 1.44269504088896340736f, LOG2_E_LOW = 1.92596299112661746887e-8f, LN_2 = 0.693147180559945309417f;

// e^x; past 150, infinity or 0; of NaN, any number.  The product with log2 e is formed with its rounding error, which comes back as a factor: an
// argument of 80 rounded alone would move the result by 60 EPS.
__device__ __forceinline__ float exp_rounded(float x) {
    const float t = __builtin_amdgcn_fmed3f(x, -150.0f, 150.0f);
    const float hi = t * LOG2_E, lo = __builtin_fmaf(t, LOG2_E_LOW, __builtin_fmaf(t, LOG2_E, -hi));
    return __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, LN_2, 1.0f);
}

// x / (1 + e^-x); the reciprocal instruction is off by one unit at most.  (-infinity gives NaN, as the formula does.)
__device__ __forceinline__ float silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + exp_rounded(-x)); }

// log(1 + e^x) = max(x, 0) + log(1 + e), e = e^-|x|.  u = 1 + e rounds: what it loses, over u, is added to the logarithm (1 / u as 1.5 - u / 2: a twelfth
// off at most, of half a step of u).
__device__ __forceinline__ float softplus(float x) {
    const float e = exp_rounded(-__builtin_fabsf(x)), u = 1.0f + e, lost = e - (u - 1.0f);
    return (x < 0.0f ? 0.0f : x) + __builtin_fmaf(__builtin_amdgcn_logf(u), LN_2, lost * __builtin_fmaf(u, -0.5f, 1.5f));
}

// The activations of EDDLHIP_ACT_*.
__device__ __forceinline__ float activated(float x, int kind) {
    return kind == EDDLHIP_ACT_SILU ? silu(x) : kind == EDDLHIP_ACT_RELU ? (x > 0.0f || x != x ? x : 0.0f) : x;
}

}  // namespace eddlhip
