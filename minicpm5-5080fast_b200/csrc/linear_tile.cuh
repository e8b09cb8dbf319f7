// linear_tile.cuh -- interface of the tiled tcgen05 GEMM with the fused epilogue (prompt chunks, M > 64; from 17 rows on where K is
// short, from 33 where the weights have many rows).
#pragma once

#include "linear_epilogue.cuh"

namespace mcl {

// w [N, K] bf16 (wb = 2) or e4m3 codes (wb = 1), x [M, x_pitch] bf16; w and x 16-byte aligned, K * wb and x_pitch * 2
// multiples of 16.  Everything else as in EpiArgs.
mc_status_t linear_tile(int wb, const void* w, const uint16_t* x, uint32_t x_pitch, uint32_t M, uint32_t N, uint32_t K,
                        const EpiArgs& ep, cudaStream_t stream, bool pdl);

// How a call is cut: CTAs per tile pair (1 or 2), features per tile, K slices.  Host logic alone.
struct TilePlan { uint32_t cg, bn, splits; };
TilePlan tile_plan(int wb, uint32_t M, uint32_t N, uint32_t K, uint32_t sms);

bool tile_forced();                                           // such a plan is set
// Every call takes this plan; cg = 0: tile_plan's.  A plan that tile_plan does not choose from is refused and changes nothing.
mc_status_t tile_force(uint32_t cg, uint32_t bn, uint32_t splits);

// 1 when a bounded wait inside the kernel ran out since the last query (clears it), -1 on a CUDA error.
int linear_tile_take_error();

}  // namespace mcl
