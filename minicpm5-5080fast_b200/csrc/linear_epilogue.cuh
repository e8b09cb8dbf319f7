// linear_epilogue.cuh -- what the linears with a fused epilogue share: the epilogue's operands and its arithmetic.
#pragma once

#include "common.cuh"

namespace mcl {

// z = scale * acc + bias ; v = act(z) [gated: act(z_gate) * z_up] ; y = bf16(v + residual), fp32 throughout.
struct EpiArgs {
    const float* scale;        // [N] fp32 row scales (e4m3 weights) or null
    const uint16_t* bias;      // [N] bf16 or null
    const uint16_t* res;       // [M, res_stride] bf16 or null; may be y
    uint16_t* y;               // [M, y_stride] bf16
    uint32_t y_stride, res_stride;
    uint32_t act, gated;
    uint32_t wait_first;       // 1: nothing is read before the previous kernel in the stream has ended, the weights neither
};

#if defined(__CUDACC__)

// __expf and __fdividef are off by a few units of 2^-23 (e^-a by a * 2^-24 more); the result is rounded to bf16 (2^-9) right after.
// __fdividef gives 0 for divisors above 2^126: from a = -87.4 on, where the value is below 1e-36.
__device__ __forceinline__ float epi_sigmoid_mul(float z, float a) { return __fdividef(z, 1.0f + __expf(-a)); }   // z / (1 + e^-a)

// z Phi(z), Phi(-a) = erfc(a / sqrt 2) / 2 = t Q(t) e^(-a^2 / 2) with t = 1 / (1 + 0.36 a), the form of Hastings' approximations; Q is
// our own fit (weighted least squares against erfcx over 0 <= a <= 14: 9e-7 of the value), so that the negative tail keeps its
// digits: the exponent, up to 120, is rounded twice, which adds up to 2 * 120 * 2^-24 * ln 2 = 1e-5 of the value at z = -13 and
// 2e-6 at z = -6 (where z has the few digits of a bf16, z * z is exact and half of that goes).  erfcf, exact to a few units, is most of an epilogue: M 3563, 22400 x 368, 242 us; this 151.
__device__ __forceinline__ float epi_gelu(float z) {
    const float t = __fdividef(1.0f, fmaf(0.36f, fabsf(z), 1.0f));
    float q = fmaf(0.04705774784f, t, -0.17976957560f);
    q = fmaf(q, t, 0.18096032739f);
    q = fmaf(q, t, 0.02654529363f);
    q = fmaf(q, t, 0.13972060382f);
    q = fmaf(q, t, 0.14177224040f);
    q = fmaf(q, t, 0.14371305704f);
    const float h = q * t * exp2f(-0.72134752044f * (z * z));
    return z * (z < 0.f ? h : 1.0f - h);
}

__device__ __forceinline__ float epi_act(float z, uint32_t act) {
    switch (act) {
        case MC_SM100_ACT_RELU: return z < 0.f ? 0.f : z;                       // a NaN stays a NaN
        case MC_SM100_ACT_GELU: return epi_gelu(z);
        case MC_SM100_ACT_GELU_TANH:                                            // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
            return epi_sigmoid_mul(z, 1.5957691216057308f * (z + 0.044715f * z * z * z));
        case MC_SM100_ACT_SILU: return epi_sigmoid_mul(z, z);
        default: return z;
    }
}

#endif

}  // namespace mcl
