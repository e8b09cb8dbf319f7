// linear_rows.cuh -- interface of the register-streaming e4m3 linear with the fused epilogue for a few rows.
#pragma once

#include "linear_epilogue.cuh"

namespace mcl {

// Whether the kernel takes this call: e4m3 weights, 2 <= M <= 16, K a multiple of 16, 16-byte aligned operands, an activation
// row pitch that is a multiple of 8, and an activation that fits shared memory.
bool linear_rows_ok(uint32_t M, uint32_t K, uint32_t x_pitch);

mc_status_t linear_rows(const uint8_t* w, const uint16_t* x, uint32_t x_pitch, uint32_t M, uint32_t N, uint32_t K, const EpiArgs& ep,
                        cudaStream_t stream, bool pdl);

}  // namespace mcl
