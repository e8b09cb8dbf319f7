// tcgen05.cuh -- what the tensor-core kernels share: mbarriers, TMA loads, operand descriptors, tensor maps.
#pragma once

#include "common.cuh"

#include <cuda.h>

namespace mcl {

constexpr int kRowBytes = 128;     // bytes per operand-tile row in shared memory (one swizzle row)

#if defined(__CUDACC__)

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// 2-D tiled TMA load global -> this CTA's shared memory; x is the innermost
// (K) coordinate in elements, y the row.  x * element size is a multiple of 16 bytes
// at every call site (K steps of 64 bf16 / 64 or 128 e4m3).
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

// K-major, 128-byte swizzle: 8-row groups are 1024 bytes apart; the leading
// offset is unused for swizzled K-major layouts (encoded as 1); version 1.
__device__ __forceinline__ uint64_t make_desc(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// swizzled byte offset of 16-byte chunk `cc` (0..7) of tile row `row`
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t cc) { return row * kRowBytes + ((cc ^ (row & 7u)) << 4); }

// One lane of a converged warp.  A loop that the whole warp runs, with the issue elected, keeps addresses in uniform registers;
// run by lane 0 alone it took 0.28 us a K block where this takes 0.22.
__device__ __forceinline__ bool elect_lane() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0u;
}

// Four e4m3 codes -> four bf16 of value * 2^-120 (the 7 magnitude bits dropped at bit 4), byte-wise: 7 integer operations
// where placing pair by pair takes 8; then * 2^120, exact.
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& p01, uint32_t& p23) {
    const uint32_t hi = ((w >> 4) & 0x07070707u) | (w & 0x80808080u), lo = (w << 4) & 0xF0F0F0F0u;
    p01 = __byte_perm(lo, hi, 0x5140u);
    p23 = __byte_perm(lo, hi, 0x7362u);
    asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(p01) : "r"(0x7B807B80u));
    asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(p23) : "r"(0x7B807B80u));
}

#endif  // __CUDACC__

// Row-major [rows, K] matrix of 1- or 2-byte elements (pitch in elements), box = [box_rows x box_k], out-of-range reads are
// zero.  The second form keeps encoded maps, which depend on these arguments alone, in a small process-wide cache.
mc_status_t tma_encode_2d(CUtensorMap* map, const void* ptr, uint32_t rows, uint32_t K, uint32_t pitch, uint32_t elem_bytes,
                          uint32_t box_k, uint32_t box_rows, bool swizzle128);
mc_status_t tma_map_2d(CUtensorMap* map, const void* ptr, uint32_t rows, uint32_t K, uint32_t pitch, uint32_t elem_bytes,
                       uint32_t box_k, uint32_t box_rows, bool swizzle128);

}  // namespace mcl
