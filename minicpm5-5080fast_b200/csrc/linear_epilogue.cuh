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

// __expf and __fdividef are off by a few units of 2^-23; the result is rounded to bf16 (2^-9) right after.
__device__ __forceinline__ float epi_sigmoid_mul(float z, float a) { return __fdividef(z, 1.0f + __expf(-a)); }   // z / (1 + e^-a)

__device__ __forceinline__ float epi_act(float z, uint32_t act) {
    switch (act) {
        case MC_SM100_ACT_RELU: return z < 0.f ? 0.f : z;                       // a NaN stays a NaN
        case MC_SM100_ACT_GELU: return 0.5f * z * erfcf(z * -0.70710678118654752f);   // 1 + erf(u) = erfc(-u), without its cancellation
        case MC_SM100_ACT_GELU_TANH:                                            // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
            return epi_sigmoid_mul(z, 1.5957691216057308f * (z + 0.044715f * z * z * z));
        case MC_SM100_ACT_SILU: return epi_sigmoid_mul(z, z);
        default: return z;
    }
}

#endif

}  // namespace mcl
