// linear_tile.cu -- y = epilogue(x W^T) for M > 64 (from 17 rows on in places) on the 5th-generation tensor cores.
//
// The MMA's A operand is a tile of 128 activation rows per CTA, B a tile of BN weight rows, D [128 x BN] fp32 in TMEM (lane =
// activation row, column = feature).  With CG = 2 two CTAs of a cluster work on one 256 x BN tile (cta_group::2): each loads
// its own 128 activation rows and HALF of the weight rows, so a weight row enters shared memory once per 256 activation rows.
//   first EPI warps: epilogue (warp w reads TMEM lanes 32 (w % 4) .. + 31; groups of four take alternate column chunks)
//   next            : TMA producer of the ring of (A, B) stages, one or two K blocks each (64 K elements = a 128-byte swizzled row)
//   next            : MMA issuer (of the pair's first CTA)
//   e4m3 only, next : TMA producer of raw weight tiles; one warp idle; then eight warps that widen raw tiles to bf16 (exact)
//                     into the B stages, two groups of four on alternate K blocks
// Whole K per tile (splits = 1): the kernel is persistent, one CTA per SM, and D is double-buffered, so that the epilogue of a
// tile runs under the products of the next.  K split over the CTAs of a larger cluster (few tiles): every CTA pushes the
// column slices that others finish into their shared memory, one cluster barrier, each sums its slice in split order.
// No atomics; every sum has a fixed order.  Every wait is bounded; one that runs out raises a flag and all roles fall through.
#include "linear_tile.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace mcl {

namespace {

constexpr uint32_t kBK = 64;                                   // K elements of a block: rows of 128 bytes
constexpr uint32_t kRing = 196608;                             // bytes of the rings
constexpr uint32_t kResBuf = 2048;                             // an epilogue warp's residual chunk stands behind its output chunk
constexpr uint32_t kWarpBuf = 4096;
constexpr uint32_t kTileNapNs = 1000000u;                      // a poll may sleep this long; spinning warps take issue slots from working ones
constexpr unsigned long long kTileWaitNs = 200ull * 1000ull * 1000ull;
constexpr uint32_t kProgress = 16;                             // stages between two marks of the producer

__device__ int g_tile_error;

// K blocks of a stage.  A turn of the producer or of the MMA warp (wait, four copies or eight MMAs, arrival) takes 350 - 390
// cycles whatever the tile's width: at one block a stage that is 0.20 us a block, where the MMAs of 128 features take 0.13.
// 256 features keep the tensor pipe busy for longer than a turn, and e4m3's widening does.
constexpr uint32_t stage_blocks(int wb, int bn) { return wb == 2 && bn < 256 ? 2u : 1u; }

template <int WB, int CG, int BN> struct TileGeom {
    static constexpr uint32_t KPS = stage_blocks(WB, BN), BROWS = BN / CG;
    static constexpr uint32_t A1 = 128u * kRowBytes, B1 = BROWS * kRowBytes, A = KPS * A1, B = KPS * B1, RAW = WB == 1 ? BROWS * kBK : 0u;
    static constexpr uint32_t RAWS = WB == 1 ? (kRing / 4u / RAW < 8u ? kRing / 4u / RAW : 8u) : 0u;
    // Even: a raw stage is then always the same group's.  With an odd count the groups take turns on a stage, and the one that
    // is ahead can find the parity of the use before the last where it waits for the last: it would pass too early.
    static_assert(RAWS % 2u == 0u, "two groups of widening warps take alternate raw stages");
    static constexpr uint32_t FIT = (kRing - RAWS * RAW) / (A + B), STAGES = FIT < 8u ? FIT : 8u;
    static constexpr uint32_t EPI = 8u;                        // epilogue warps
    // e4m3: 640 threads launched with 96 registers each; the roles trade them (setmaxnreg, warpgroups of 128 threads):
    // 2 x 128 x 136 (epilogue) + 128 x 48 (producers, MMA) + 2 x 128 x 80 (widening) = 640 x 96, what the CTA was launched with.
    static constexpr uint32_t THREADS = 32u * (EPI + (WB == 1 ? 12u : 2u));
    static constexpr uint32_t COLS = BN;                       // TMEM columns of one accumulator
    // rings, output and residual chunks of the epilogue warps, scale (fp32) and bias (bf16) of a tile, alignment
    static constexpr uint32_t SMEM = kRing + EPI * kWarpBuf + BN * 6u + 1024u;
};

struct TileArgs {
    EpiArgs ep;
    uint32_t M, N, nkb, n_out;
    uint32_t m_tiles, n_tiles, tiles, splits;
    uint32_t y_vec, res_vec;                                   // rows of y / of the residual start on 16-byte boundaries
    int32_t* status;
};

constexpr uint32_t kRowGroup = 16;                             // row tiles walked before the next feature tile

__device__ __forceinline__ void tile_of(const TileArgs& a, uint32_t t, uint32_t& mt, uint32_t& nt) {
    const uint32_t per = kRowGroup * a.n_tiles, g = t / per, rem = t - g * per;
    const uint32_t rows = min(kRowGroup, a.m_tiles - g * kRowGroup);
    nt = rem / rows;
    mt = g * kRowGroup + (rem - nt * rows);
}

// acquire at cluster scope: arrivals come from both CTAs of a pair.  Every lane polls for itself: where a wait runs out while
// the phase turns, some lanes of a warp may see the phase and others the flag.  What stands behind (elect.sync, tcgen05.ld,
// __syncwarp) wants all 32, so no lane leaves a warp's loop alone.
// The limit is a stage's; who waits for a whole slice of K hands over the count that this CTA's producer keeps (kProgress), and the
// clock starts anew whenever it has moved: a slice of 2^22 K blocks takes a second and more.
__device__ __forceinline__ bool tile_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status, const volatile uint32_t* progress = nullptr) {
    unsigned long long t0 = 0;
    uint32_t seen = 0;
    for (uint32_t spin = 0;; ++spin) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done) : "r"(bar), "r"(parity), "r"(kTileNapNs) : "memory");
        if (done) return true;
        if (*abort_flag) return false;
        if ((spin & 15u) == 15u) {
            const unsigned long long now = global_timer_ns();
            if (t0 == 0) {
                t0 = now;
                if (progress != nullptr) seen = *progress;
            } else if (now - t0 > kTileWaitNs) {
                if (progress == nullptr || *progress == seen) break;
                t0 = now; seen = *progress;
            }
        }
    }
    *abort_flag = 1;
    g_tile_error = 1;
    if (status != nullptr) *reinterpret_cast<volatile int32_t*>(status) = 1;
    return false;
}

__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// Nothing that the other CTA's threads read stands behind these arrivals: a widened tile is read by the tensor core out of
// the arriving CTA's own shared memory (fence.proxy.async has run), a drained accumulator is written by it (tcgen05 fences).
// So the release stays at CTA scope; at cluster scope it made the arrival cost more than the widening (M = 8192, 2304 x 5760:
// 291 against 177 us).
__device__ __forceinline__ void arrive_remote(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// The load lands in this CTA; with CG = 2 the bytes are counted on the barrier of the pair's first CTA (a cluster address).
template <int CG>
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
    if constexpr (CG == 1) {
        tma_load_2d(dst, map, bar, x, y);
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    }
}

template <int CG>
__device__ __forceinline__ void tile_mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}

// Arrives on the same barrier of every CTA of the pair once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void tile_commit(uint32_t bar, uint16_t pair_mask) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"(pair_mask) : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts16(uint32_t a, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// One warp's 32 rows x 32 accumulator columns -> 32 (behind the gate 16) outputs a row.  A lane holds one row while values
// are computed, and 16-byte pieces of consecutive columns, several rows apart, while they cross global memory; a 2 KB buffer
// turns one into the other (pieces swizzled by row: neither side meets a bank twice).  The residual comes the other way.
template <bool GATED>
struct ChunkIO {
    static constexpr uint32_t LG = GATED ? 1u : 2u, PIECES = 1u << LG, OUTS = 8u * PIECES, ROWS = 32u >> LG, ROW_BYTES = 2u * OUTS;
    const TileArgs& a;
    uint32_t buf, lane, own, own_swz, across, col;      // shared addresses of this lane's row / first piece; its first column
    uint32_t m_base;
    int32_t rows_left;                                  // rows from this lane's first piece's to the end of y
    uint32_t res_first = 0;                             // first residual of this lane's row, where it crosses alone
    uint16_t* y;
    const uint16_t* res;

    static __device__ __forceinline__ uint32_t swizzle(uint32_t row) { return GATED ? (row >> 2) & 1u : (row >> 1) & 3u; }
    __device__ __forceinline__ ChunkIO(const TileArgs& args, uint32_t buffer, uint32_t l, uint32_t row0) : a(args), buf(buffer), lane(l), m_base(row0) {
        own = buf + lane * ROW_BYTES; own_swz = swizzle(lane);
        const uint32_t row = lane >> LG, piece = lane & (PIECES - 1u);
        across = buf + row * ROW_BYTES + ((piece ^ swizzle(row)) << 4);     // + 512 bytes per ROWS rows: the swizzle repeats
        col = piece * 8u;
        rows_left = (int32_t)a.M - (int32_t)(m_base + row);
        y = a.ep.y + (size_t)(m_base + row) * a.ep.y_stride + col;
        res = a.ep.res != nullptr ? a.ep.res + (size_t)(m_base + row) * a.ep.res_stride + col : nullptr;
    }
    __device__ __forceinline__ uint32_t own_piece(uint32_t k) const { return own + ((k ^ own_swz) << 4); }

    __device__ __forceinline__ uint32_t odd_res(uint32_t row) const {   // a row of the residual starts in the upper half of a word
        return ((uint32_t)(reinterpret_cast<uintptr_t>(a.ep.res) >> 1) + row * a.ep.res_stride) & 1u;
    }
    // Ahead of use and without registers; beyond the edges zeros, which are not stored.
    __device__ __forceinline__ void fetch_res(uint32_t j0) {
        if (!a.res_vec) { fetch_words(j0); return; }
        const uint32_t bytes = j0 + col + 8u <= a.n_out ? 16u : (j0 + col < a.n_out ? 2u * (a.n_out - j0 - col) : 0u);
#pragma unroll
        for (uint32_t i = 0; i < PIECES; ++i) {
            const bool in = (int32_t)(i * ROWS) < rows_left && bytes != 0u;
            const uint16_t* src = in ? res + (size_t)(i * ROWS) * a.ep.res_stride + j0 : a.ep.res;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(across + kResBuf + i * 512u), "l"(src), "r"(in ? bytes : 0u) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // Rows of the residual anywhere: the halves [odd, odd + OUTS) of each, two a word, and the first one of an odd row alone; a
    // half-warp (gated: a quarter) takes a row.  odd is the same for all rows of a lane: their distance is even.  M 2595, N 19101,
    // K 696: 104 us; with element loads through registers, eight in flight, 117.
    __device__ __forceinline__ void fetch_words(uint32_t j0) {
        constexpr uint32_t LW = LG + 2u, WORDS = 1u << LW, WROWS = 32u >> LW;
        const uint32_t r0 = lane >> LW, w = lane & (WORDS - 1u), e = j0 + 2u * w + odd_res(r0);
        const uint32_t bytes = e + 2u <= a.n_out ? 4u : (e < a.n_out ? 2u : 0u);
        const int32_t left = (int32_t)a.M - (int32_t)(m_base + r0);
        const uint16_t* from = a.ep.res + (size_t)(m_base + r0) * a.ep.res_stride + e;
        const uint16_t* none = reinterpret_cast<const uint16_t*>(reinterpret_cast<uintptr_t>(a.ep.res + 1) & ~(uintptr_t)3);     // aligned, not read
        const uint32_t to = buf + kResBuf + r0 * ROW_BYTES + (w & 3u) * 4u;
#pragma unroll
        for (uint32_t i = 0; i < WORDS; ++i) {
            const bool in = (int32_t)(i * WROWS) < left && bytes != 0u;
            const uint16_t* src = in ? from + (size_t)(i * WROWS) * a.ep.res_stride : none;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + i * 128u + (((w >> 2) ^ (i & (PIECES - 1u))) << 4)), "l"(src), "r"(in ? bytes : 0u) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        res_first = 0u;
        if (m_base + lane < a.M && odd_res(lane)) res_first = a.ep.res[(size_t)(m_base + lane) * a.ep.res_stride + j0];
    }
    // Rows of y anywhere: a lane holds one column of every row (gated: of every second row), so that one instruction writes all
    // of a row's chunk.  Two rows an instruction in 4-byte words are slower, though they are half as many (M 2595, K 64: 66 us at
    // N 19102, with the ends of odd rows apart 75 at N 19101; so 56 at either).
    __device__ __forceinline__ void store_elements(uint32_t j0) const {
        const uint32_t c = lane & (OUTS - 1u), r0 = lane / OUTS;
        const int32_t left = (int32_t)a.M - (int32_t)(m_base + r0);
        const bool in = j0 + c < a.n_out;
        uint16_t* dst = a.ep.y + (size_t)(m_base + r0) * a.ep.y_stride + j0 + c;
        const size_t step = (size_t)(32u / OUTS) * a.ep.y_stride;
#pragma unroll
        for (uint32_t r = 0; r < OUTS; r += 8u) {
            uint16_t v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                const uint32_t row = r0 + (r + e) * (32u / OUTS);
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v[e]) : "r"(buf + row * ROW_BYTES + (((c >> 3) ^ swizzle(row)) << 4) + (c & 7u) * 2u) : "memory");
            }
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) {
                if (in && (int32_t)((r + e) * (32u / OUTS)) < left) *dst = v[e];
                dst += step;
            }
        }
    }
    __device__ __forceinline__ void store(uint32_t j0) const {
        if (a.y_vec) {
            uint4 v[PIECES];
#pragma unroll
            for (uint32_t i = 0; i < PIECES; ++i) v[i] = lds16(across + i * 512u);
#pragma unroll
            for (uint32_t i = 0; i < PIECES; ++i) {
                uint16_t* dst = y + (size_t)(i * ROWS) * a.ep.y_stride + j0;
                if ((int32_t)(i * ROWS) < rows_left) {
                    if (j0 + col + 8u <= a.n_out) *reinterpret_cast<uint4*>(dst) = v[i];
                    else if (j0 + col < a.n_out) {
                        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                        for (uint32_t e = 0; e < 7; ++e)
                            if (j0 + col + e < a.n_out) dst[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                    }
                }
            }
        } else {
            store_elements(j0);
        }
    }
    // v: the 32 finished accumulators of this lane's row, columns n .. n + 31 (tile column c); col_s: staged scales, biases
    template <uint32_t BN>
    __device__ __forceinline__ void finish(float (&v)[32], uint32_t n, uint32_t c, uint32_t col_s, bool has_scale, bool has_bias, uint32_t next_n) {
        const uint32_t j0 = GATED ? n >> 1 : n;
        const bool has_res = a.ep.res != nullptr;
        if (has_scale) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float4 f = lds_f4(col_s + (c + 4u * k) * 4u);
                v[4 * k] *= f.x; v[4 * k + 1] *= f.y; v[4 * k + 2] *= f.z; v[4 * k + 3] *= f.w;
            }
        }
        if (has_bias) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 f = lds16(col_s + BN * 4u + (c + 8u * k) * 2u);
                const uint32_t p[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[8 * k + 2 * e] += bf16lo(p[e]); v[8 * k + 2 * e + 1] += bf16hi(p[e]); }
            }
        }
        const uint32_t act = a.ep.act;
        auto apply = [&](auto f) {
            if constexpr (GATED) {
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = f(v[2 * k]) * v[2 * k + 1];
            } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) v[k] = f(v[k]);
            }
        };
        // one loop per activation: no choice inside
        if (act == MC_SM100_ACT_SILU) apply([](float z) { return epi_act(z, MC_SM100_ACT_SILU); });
        else if (act == MC_SM100_ACT_GELU) apply([](float z) { return epi_act(z, MC_SM100_ACT_GELU); });
        else if (act == MC_SM100_ACT_GELU_TANH) apply([](float z) { return epi_act(z, MC_SM100_ACT_GELU_TANH); });
        else if (act == MC_SM100_ACT_RELU) apply([](float z) { return epi_act(z, MC_SM100_ACT_RELU); });
        else if (GATED) apply([](float z) { return z; });
        if (has_res) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncwarp();
            uint32_t before = res_first << 16;
            const uint32_t shift = a.res_vec ? 0u : 16u * odd_res(lane);
#pragma unroll
            for (uint32_t k = 0; k < PIECES; ++k) {
                const uint4 m = lds16(own_piece(k) + kResBuf);
                const uint32_t r[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint32_t h = __funnelshift_l(before, r[e], shift);
                    v[8 * k + 2 * e] += bf16lo(h); v[8 * k + 2 * e + 1] += bf16hi(h);
                    before = r[e];
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < PIECES; ++k)
            sts16(own_piece(k), make_uint4(pack_bf16(v[8 * k], v[8 * k + 1]), pack_bf16(v[8 * k + 2], v[8 * k + 3]),
                                           pack_bf16(v[8 * k + 4], v[8 * k + 5]), pack_bf16(v[8 * k + 6], v[8 * k + 7])));
        __syncwarp();                                                  // pieces written, residual read
        if (has_res && next_n != 0xFFFFFFFFu) fetch_res(GATED ? next_n >> 1 : next_n);
        store(j0);
        __syncwarp();
    }
};

}  // namespace

// WB: bytes per weight element.  CG: CTAs per tile.  BN: features per tile.
template <int WB, int CG, int BN>
__global__ void __launch_bounds__(TileGeom<WB, CG, BN>::THREADS, 1)
linear_tile_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const TileArgs a) {
    using G = TileGeom<WB, CG, BN>;
    constexpr uint32_t STAGES = G::STAGES, RAWS = G::RAWS, EPI = G::EPI, KPS = G::KPS;
    constexpr uint32_t IDESC = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((128 * CG) >> 4) << 24);
    constexpr uint32_t CONV_WARPS = 4;                           // warps that widen one K block

    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[36];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ uint32_t progress;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sA = base, sB = base + STAGES * G::A, sRaw = sB + STAGES * G::B;
    const uint32_t sBuf = base + kRing, sCol = sBuf + EPI * kWarpBuf;
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty = [&](uint32_t s) { return bar0 + 8u * (8u + s); };
    auto raw_full = [&](uint32_t s) { return bar0 + 8u * (16u + s); };
    auto raw_empty = [&](uint32_t s) { return bar0 + 8u * (24u + s); };
    auto acc_full = [&](uint32_t b) { return bar0 + 8u * (32u + b); };
    auto acc_empty = [&](uint32_t b) { return bar0 + 8u * (34u + b); };

    const uint32_t S = a.splits, csize = CG * S, crank = blockIdx.x % csize, cid = blockIdx.x / csize, clusters = gridDim.x / csize;
    const uint32_t split = crank / CG, sub = crank % CG, lead = crank - sub;
    const bool leader = sub == 0u;
    const uint32_t kb0 = split * a.nkb / S, kb1 = (split + 1u) * a.nkb / S;
    const uint32_t bufs = S == 1u ? 2u : 1u;
    const uint32_t tmem_cols = bufs * BN < 32u ? 32u : bufs * BN;

    pdl_trigger();
    // One CTA per tile: its first stages are asked for before the tensor memory and the other roles are ready (weights before
    // the previous kernel's end is waited for): -0.5 us a call.  A pair has to know its partner's barriers first.
    const uint32_t nloc = cid < a.tiles ? kb1 - kb0 : 0u;
    constexpr uint32_t EARLY = 4u / KPS;
    const uint32_t early = CG == 1 ? min(nloc, EARLY) : 0u;
    static_assert(STAGES >= EARLY && (WB == 2 || RAWS >= EARLY), "the early stages are all the ring's");
    if (tid == EPI * 32u) {
        abort_flag = 0; progress = 0u;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        for (uint32_t s = 0; s < STAGES; ++s) { mbar_init(full(s), 1u + (WB == 1 ? CONV_WARPS * CG : 0u)); mbar_init(empty(s), 1); }
        if constexpr (WB == 1)
            for (uint32_t s = 0; s < RAWS; ++s) { mbar_init(raw_full(s), 1); mbar_init(raw_empty(s), CONV_WARPS); }
        for (uint32_t b = 0; b < 2; ++b) { mbar_init(acc_full(b), 1); mbar_init(acc_empty(b), EPI * CG); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if constexpr (CG == 1) {
            uint32_t mt = 0, nt = 0;
            if (nloc != 0u) tile_of(a, cid, mt, nt);
            const int32_t m0 = (int32_t)(mt * 128u), n0 = (int32_t)(nt * BN);
            if (a.ep.wait_first) pdl_wait();
            for (uint32_t it = 0; it < early; ++it) {
                const uint32_t bar = WB == 1 ? raw_full(it) : full(it);
                mbar_expect_tx(bar, WB == 1 ? G::RAW : G::A + G::B);
#pragma unroll
                for (uint32_t h = 0; h < KPS; ++h)
                    tma_load_2d(WB == 1 ? sRaw + it * G::RAW : sB + it * G::B + h * G::B1, &map_w, bar, (int32_t)(((kb0 + it) * KPS + h) * kBK), n0);
            }
            pdl_wait();
            for (uint32_t it = 0; it < early; ++it) {
                if constexpr (WB == 1) mbar_expect_tx(full(it), G::A);
#pragma unroll
                for (uint32_t h = 0; h < KPS; ++h) tma_load_2d(sA + it * G::A + h * G::A1, &map_x, full(it), (int32_t)(((kb0 + it) * KPS + h) * kBK), m0);
            }
        }
    }
    if (warp == EPI + 1u) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();                       // barriers and TMEM of every CTA are there
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;
    volatile int* abortp = &abort_flag;
    volatile uint32_t* progressp = &progress;
    pdl_wait();

    if (warp < EPI) {
        if constexpr (WB == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        // ------------------------------------------------------ epilogue
        constexpr uint32_t GROUPS = EPI / 4u;
        const uint32_t q = warp & 3u, group = warp >> 2;
        const bool has_scale = a.ep.scale != nullptr, has_bias = a.ep.bias != nullptr;
        auto run = [&](auto gated) {
            using IO = ChunkIO<decltype(gated)::value>;
            bool ok = true;
            uint32_t i = 0;
            // scale and bias of this thread's column of a tile
            static_assert(BN <= (int)(EPI * 32u), "one column per epilogue thread");
            float my_scale = 1.f;
            uint16_t my_bias = 0;
            auto load_column = [&](uint32_t t) {
                if (t >= a.tiles || tid >= BN) return;
                uint32_t mt, nt;
                tile_of(a, t, mt, nt);
                const uint32_t n = nt * BN + tid;
                if (n >= a.N) return;
                if (has_scale) my_scale = a.ep.scale[n];
                if (has_bias) my_bias = a.ep.bias[n];
            };
            if (has_scale || has_bias) load_column(cid);
            for (uint32_t t = cid; t < a.tiles; t += clusters, ++i) {
                uint32_t mt, nt;
                tile_of(a, t, mt, nt);
                const uint32_t b = i % bufs, n0 = nt * BN;
                IO io(a, sBuf + warp * kWarpBuf, lane, (mt * CG + sub) * 128u + q * 32u);
                if (has_scale || has_bias) {
                    asm volatile("bar.sync 1, %0;" ::"n"(EPI * 32u) : "memory");     // the previous tile's have been read
                    if (tid < BN) {
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(sCol + tid * 4u), "f"(my_scale) : "memory");
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(sCol + BN * 4u + tid * 2u), "h"(my_bias) : "memory");
                    }
                    load_column(t + clusters);                                       // of the next tile, under this one's work
                    asm volatile("bar.sync 1, %0;" ::"n"(EPI * 32u) : "memory");
                }
                // This CTA finishes columns [c_lo, c_hi), this warp every GROUPS-th chunk of them.  More slices than chunks: a
                // chunk's rows are dealt out too, in `parts` of rows (pairs: never).
                const uint32_t per = CG == 2 ? BN / S : max(BN / S, 32u), parts = CG == 2 ? 1u : per * S / BN, rows = 128u / parts, part_of_warp = q * parts / 4u;
                const uint32_t c_lo = split / parts * per;
                uint32_t c_hi = n0 + c_lo + per <= a.N ? c_lo + per : (a.N - n0 > c_lo ? a.N - n0 : c_lo);
                if (part_of_warp != split % parts) c_hi = c_lo;
                const uint32_t c_first = c_lo + group * 32u;
                if (a.ep.res != nullptr && c_first < c_hi) io.fetch_res((n0 + c_first) >> a.ep.gated);
                if (ok) ok = tile_wait(acc_full(b), (i / bufs) & 1u, abortp, a.status, progressp);
                __syncwarp();
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t taddr = tmem + b * G::COLS + ((q * 32u) << 16);
                const uint32_t row = q * 32u + lane - part_of_warp * rows;          // in its part
                auto release = [&]() {       // this warp has read its part of the accumulator; one that did not come is not given back
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0 && ok) { if (CG == 2) arrive_remote(map_to_rank(acc_empty(b), lead)); else mbar_arrive(acc_empty(b)); }
                };
                if (S > 1u) {
                    // the cluster's rings are idle: they become the exchange [source split][row of the part][per] of fp32
                    cluster_sync();
                    // Sums that did not come are pushed all the same: whoever adds them up stores nothing either.  (Where they came
                    // they are whole: the lane that commits them has seen every stage.)
                    if (!ok)
                        for (uint32_t p = 0; p < csize; ++p)
                            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_rank(smem_u32(&abort_flag), p)), "r"(1u) : "memory");
                    uint32_t turn = 0;
                    for (uint32_t o = 0; o < S; ++o) {
                        if (o == split) continue;
                        const uint32_t src = split < o ? split : split - 1u;
                        if (part_of_warp != o % parts) continue;
                        const uint32_t dst = map_to_rank(base + (src * rows + row) * per * 4u, o * CG + sub);
                        for (uint32_t c = 0; c < per; c += 32u, ++turn) {
                            if (turn % GROUPS != group) continue;
                            float v[32];
                            tmem_ld32(taddr + o / parts * per + c, v);
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};"
                                             ::"r"(dst + ((((c >> 2) + k) ^ (row & 7u)) << 4)), "f"(v[4 * k]), "f"(v[4 * k + 1]), "f"(v[4 * k + 2]), "f"(v[4 * k + 3]) : "memory");
                        }
                    }
                    cluster_sync();
                } else if (c_first >= c_hi) release();
                const bool failed = __any_sync(0xFFFFFFFFu, !ok || *abortp != 0) != 0;      // finish() has warp barriers
                for (uint32_t c = c_first; c < c_hi; c += 32u * GROUPS) {
                    const bool last = c + 32u * GROUPS >= c_hi;
                    float v[32];
                    tmem_ld32(taddr + c, v);
                    if (S == 1u && last) release();
                    if (S > 1u) {
                        // this CTA's own part first, then the others in split order
                        for (uint32_t src = 0; src + 1u < S; ++src) {
                            const uint32_t at = base + (src * rows + row) * per * 4u;
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float4 f = lds_f4(at + (((((c - c_lo) >> 2) + k) ^ (row & 7u)) << 4));
                                v[4 * k] += f.x; v[4 * k + 1] += f.y; v[4 * k + 2] += f.z; v[4 * k + 3] += f.w;
                            }
                        }
                    }
                    if (!failed) io.template finish<BN>(v, n0 + c, c, sCol, has_scale, has_bias, last ? 0xFFFFFFFFu : n0 + c + 32u * GROUPS);
                }
            }
        };
        if (a.ep.gated) run(std::true_type{});
        else run(std::false_type{});
    } else {
        if (warp < EPI + 4u) {
            if constexpr (WB == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
            if (warp == EPI) {
                if (lane == 0) {
                    // -------------------------------------------------- producer of A (bf16: A and B)
                    bool ok = true;
                    uint32_t it = 0;
                    for (uint32_t t = cid; t < a.tiles && ok; t += clusters) {
                        uint32_t mt, nt;
                        tile_of(a, t, mt, nt);
                        const int32_t m0 = (int32_t)((mt * CG + sub) * 128u), n0 = (int32_t)(nt * BN + sub * G::BROWS);
                        for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                            const uint32_t s = it % STAGES;
                            if (it < early) continue;
                            if (it >= STAGES) ok = tile_wait(empty(s), ((it / STAGES) - 1u) & 1u, abortp, a.status);
                            if (!ok) break;
                            if (it % kProgress == 0u) *progressp = it;
                            if (leader) mbar_expect_tx(full(s), CG * (G::A + (WB == 2 ? G::B : 0u)));
                            const uint32_t bar = CG == 2 ? map_to_rank(full(s), lead) : full(s);
#pragma unroll
                            for (uint32_t h = 0; h < KPS; ++h) {                     // a block beyond K comes as zeros
                                const int32_t k = (int32_t)((kb * KPS + h) * kBK);
                                tile_load<CG>(sA + s * G::A + h * G::A1, &map_x, bar, k, m0);
                                if constexpr (WB == 2) tile_load<CG>(sB + s * G::B + h * G::B1, &map_w, bar, k, n0);
                            }
                        }
                    }
                    // the last arrivals of the MMAs on this CTA's stages: none is under way when the CTA leaves
                    for (uint32_t u = it < STAGES ? 0u : it - STAGES; u < it && ok; ++u) ok = tile_wait(empty(u % STAGES), (u / STAGES) & 1u, abortp, a.status);
                }
            } else if (warp == EPI + 1u) {
                if (leader) {
                    // -------------------------------------------------- MMA issuer: the warp together, one lane elected to issue
                    const uint16_t pair = (uint16_t)(CG == 2 ? 3u << lead : 1u);
                    bool ok = true;
                    uint32_t it = 0, i = 0, s = 0, par = 0;
                    // A lane whose wait ran out stays in the loop and issues nothing; the elected lane is the same every time.  (A vote
                    // behind each wait instead: M = 301, 2304 x 2304 11.5 -> 12.0 us.)
                    for (uint32_t t = cid; t < a.tiles; t += clusters, ++i) {
                        const uint32_t b = i % bufs;
                        if (ok && i >= bufs) ok = tile_wait(acc_empty(b), ((i / bufs) - 1u) & 1u, abortp, a.status);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t acc = tmem + b * G::COLS;
                        for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                            if (ok) ok = tile_wait(full(s), par, abortp, a.status);
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            const uint64_t da = make_desc(sA + s * G::A), db = make_desc(sB + s * G::B);
                            if (elect_lane() && ok) {
#pragma unroll
                                for (uint32_t k = 0; k < 4u * KPS; ++k) {           // 32 bytes of K each; addresses in units of 16 bytes
                                    const uint64_t ka = (k >> 2) * (G::A1 >> 4) + (k & 3u) * 2u, kw = (k >> 2) * (G::B1 >> 4) + (k & 3u) * 2u;
                                    tile_mma<CG>(acc, da + ka, db + kw, IDESC, (kb > kb0 || k > 0) ? 1u : 0u);
                                }
                                tile_commit<CG>(empty(s), pair);
                            }
                            __syncwarp();
                            if (++s == STAGES) { s = 0; par ^= 1u; }
                        }
                        if (elect_lane() && ok) tile_commit<CG>(acc_full(b), pair);
                        __syncwarp();
                    }
                }
            } else if (warp == EPI + 2u) {
                if constexpr (WB == 1) if (lane == 0) {
                    // -------------------------------------------------- producer of raw weight tiles
                    bool ok = true;
                    uint32_t it = 0;
                    for (uint32_t t = cid; t < a.tiles && ok; t += clusters) {
                        uint32_t mt, nt;
                        tile_of(a, t, mt, nt);
                        const int32_t n0 = (int32_t)(nt * BN + sub * G::BROWS);
                        for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                            const uint32_t r = it % RAWS;
                            if (it < early) continue;
                            if (it >= RAWS) ok = tile_wait(raw_empty(r), ((it / RAWS) - 1u) & 1u, abortp, a.status);
                            if (!ok) break;
                            mbar_expect_tx(raw_full(r), G::RAW);
                            tma_load_2d(sRaw + r * G::RAW, &map_w, raw_full(r), (int32_t)(kb * kBK), n0);
                        }
                    }
                }
            }
        } else {
            // -------------------------------------------------- e4m3 -> bf16
            if constexpr (WB == 1) {
                asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
                constexpr uint32_t R = RAWS;
                const uint32_t group = (warp - (EPI + 4u)) / CONV_WARPS, ct = tid & (CONV_WARPS * 32u - 1u);
                const uint32_t my_tiles = cid < a.tiles ? (a.tiles - cid + clusters - 1u) / clusters : 0u, total = my_tiles * (kb1 - kb0);
                // A lane whose wait ran out stays with its warp, whose barriers want all 32, up to the vote behind the second wait:
                // the whole warp leaves there, without the arrival on a stage that would miss a part.  A raw stage goes back only where
                // the lane that returns it has seen it land: nobody arms a barrier whose copy is still pending.
                for (uint32_t it = group; it < total; it += 2u) {
                    const uint32_t r = it % R, s = it % STAGES;
                    bool ok = tile_wait(raw_full(r), (it / R) & 1u, abortp, a.status);
                    // 16-byte raw chunks, eight lanes on 128 consecutive bytes; widened in registers before the stage is free
                    constexpr uint32_t PER = G::BROWS / 32u;
                    const uint32_t row0 = ct >> 2, cc = ct & 3u;
                    uint4 wide[PER][2];
#pragma unroll
                    for (uint32_t i = 0; i < PER; ++i) wide[i][0] = lds16(sRaw + r * G::RAW + (row0 + 32u * i) * kBK + cc * 16u);
#pragma unroll
                    for (uint32_t i = 0; i < PER; ++i) {
                        const uint4 v = wide[i][0];
                        widen4(v.x, wide[i][0].x, wide[i][0].y); widen4(v.y, wide[i][0].z, wide[i][0].w);
                        widen4(v.z, wide[i][1].x, wide[i][1].y); widen4(v.w, wide[i][1].z, wide[i][1].w);
                    }
                    __syncwarp();
                    if (lane == 0 && ok) mbar_arrive(raw_empty(r));
                    if (it >= STAGES) ok = tile_wait(empty(s), ((it / STAGES) - 1u) & 1u, abortp, a.status) && ok;
                    if (!__all_sync(0xFFFFFFFFu, ok)) break;
#pragma unroll
                    for (uint32_t i = 0; i < PER; ++i) {
                        sts16(sB + s * G::B + swz(row0 + 32u * i, 2u * cc), wide[i][0]);
                        sts16(sB + s * G::B + swz(row0 + 32u * i, 2u * cc + 1u), wide[i][1]);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 2) arrive_remote(map_to_rank(full(s), lead));
                        else mbar_arrive(full(s));
                    }
                }
            }
        }
        if (S > 1u) {
            // these warps pass the two barriers of the exchange
            __syncwarp();
            cluster_sync();
            cluster_sync();
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*abortp) {                                               // a wait ran out: let this CTA's copies in flight land before it leaves
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
    // Nobody addresses a CTA that has left.  Without pairs the last that arrives from outside is in front of the exchange's second
    // barrier, and nothing comes from outside before its first: two barriers of a split call instead of four.
    if constexpr (CG == 2) cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == EPI + 1u) {
        if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
    }
}

namespace {

template <int WB, int CG, int BN>
mc_status_t launch_tile(const void* w, const uint16_t* x, uint32_t x_pitch, uint32_t K, TileArgs a, cudaStream_t stream, bool pdl) {
    using G = TileGeom<WB, CG, BN>;
    auto kern = linear_tile_kernel<WB, CG, BN>;
    static SmemOptIn optin;
    const cudaError_t e = optin.ensure(kern, G::SMEM);
    if (e != cudaSuccess) {
        set_error("linear_tile: cannot raise shared memory to %u: %s", G::SMEM, cudaGetErrorString(e));
        return MC_E_CUDA;
    }
    CUtensorMap map_w, map_x;
    mc_status_t s = tma_encode_2d(&map_w, w, a.N, K, K, WB, kBK, G::BROWS, WB == 2);
    if (s == MC_OK) s = tma_encode_2d(&map_x, x, a.M, K, x_pitch, 2, kBK, 128, true);
    if (s != MC_OK) return s;
    const uint64_t mt = (a.M + 128ull * CG - 1) / (128ull * CG), nt = (a.N + BN - 1ull) / BN;
    if (mt * nt * CG * a.splits > 0x7FFFFFFFull) {
        set_error("mc_sm100_linear_epilogue: M=%u N=%u make too many tiles", a.M, a.N);
        return MC_E_UNSUPPORTED;
    }
    a.nkb = (K + G::KPS * kBK - 1u) / (G::KPS * kBK);
    a.m_tiles = (uint32_t)mt; a.n_tiles = (uint32_t)nt; a.tiles = (uint32_t)(mt * nt);
    uint32_t clusters = a.tiles;
    if (a.splits == 1u) {
        const uint32_t room = (uint32_t)sm_count() / CG;
        if (clusters > room) clusters = room;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(clusters * CG * a.splits);
    cfg.blockDim = dim3(G::THREADS);
    cfg.dynamicSmemBytes = G::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG * a.splits;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, kern, map_w, map_x, a);
    MCL_CHECK_LAUNCH("linear_tile");
    return MC_OK;
}

}  // namespace

// The plan with the least estimated time.  The terms were fitted to 2400 timings on B200 (100 shapes, M 66 .. 8192, N 65 ..
// 23000, K 256 .. 8100, both weight types, every plan); over them the choice is on average 0.5 % and at most 19 % slower than
// the best plan, where 2 CTAs x 256 features for every call would be 30 % slower on average.  In us:
//   a K block     0.19 - 0.30, not in proportion to the tile's width (what one SM draws from L2 bounds the narrow ones, the
//                 MMA the widest); e4m3 0.29 - 0.41 (widening)
//   an epilogue   1.0 for 64 columns, e4m3 1.2 times that (fewer registers)
//   a K slice     2.4 for barriers and a cluster's start, 3.4 with pairs, 1.2 per 32 columns sent away
struct TileForm { uint32_t cg, bn, splits; double block[2]; };
static constexpr TileForm kForms[] = {{1, 64, 1, {0.19, 0.29}}, {1, 64, 2, {0.19, 0.29}}, {1, 64, 4, {0.19, 0.29}}, {1, 128, 1, {0.24, 0.41}},
                                      {1, 128, 2, {0.24, 0.41}}, {1, 128, 4, {0.24, 0.41}}, {2, 128, 1, {0.245, 0.30}}, {2, 128, 2, {0.245, 0.30}},
                                      {2, 128, 4, {0.245, 0.30}}, {2, 256, 1, {0.295, 0.36}}, {2, 256, 2, {0.295, 0.36}}, {2, 256, 4, {0.295, 0.36}}};
TilePlan tile_plan(int wb, uint32_t M, uint32_t N, uint32_t K, uint32_t sms) {
    TilePlan best{2, 256, 1};
    double least = 1e30;
    for (const TileForm& f : kForms) {
        const uint32_t per = stage_blocks(wb, (int)f.bn), stages = (K + per * kBK - 1u) / (per * kBK);
        if (f.splits > stages) continue;
        const double tiles = (double)((M + 128ull * f.cg - 1) / (128ull * f.cg)) * (double)((N + f.bn - 1ull) / f.bn);
        // clusters that run at once: all SMs as pairs, fewer of the larger ones (whole GPCs do not divide evenly)
        const uint32_t size = f.cg * f.splits;
        double room = size == 1u ? sms : size == 2u ? sms / 2u : size == 4u ? sms * 32u / 148u : sms * 14u / 148u;
        if (room < 1.0) room = 1.0;
        const double rounds = (double)(uint64_t)((tiles + room - 1.0) / room);
        const double block = f.block[wb == 1 ? 1 : 0], epi = 1.0 * f.bn / 64.0 * (wb == 1 ? 1.2 : 1.0);
        const double slice = (double)((stages + f.splits - 1u) / f.splits * per);
        const double t = f.splits == 1u ? rounds * (slice * block + epi)
                                        : rounds * ((f.cg == 1u ? 2.4 : 3.4) + slice * block + 1.2 * (f.splits - 1.0) / f.splits * f.bn / 32.0) + epi / f.splits;
        if (t < least) { least = t; best = {f.cg, f.bn, f.splits}; }
    }
    return best;
}

// benchmark and test hook: every call takes this plan (cg = 0: the rule above).  Only the plans that the rule chooses from: a slice
// of the exchange is a whole number of 32 columns, or of rows.
static std::atomic<uint32_t> g_forced{0};
bool tile_forced() { return g_forced.load() != 0u; }
mc_status_t tile_force(uint32_t cg, uint32_t bn, uint32_t splits) {
    bool known = cg == 0u;
    for (const TileForm& f : kForms) known = known || (f.cg == cg && f.bn == bn && f.splits == splits);
    if (!known) {
        set_error("mc_sm100_debug_set_tile_plan: no plan of %u CTAs, %u features, %u slices", cg, bn, splits);
        return MC_E_INVALID_ARGUMENT;
    }
    g_forced.store(cg == 0u ? 0u : (cg << 24) | (splits << 16) | bn);
    return MC_OK;
}

mc_status_t linear_tile(int wb, const void* w, const uint16_t* x, uint32_t x_pitch, uint32_t M, uint32_t N, uint32_t K,
                        const EpiArgs& ep, cudaStream_t stream, bool pdl) {
    TilePlan p = tile_plan(wb, M, N, K, (uint32_t)sm_count());
    if (const uint32_t f = g_forced.load(); f != 0u) p = {f >> 24, f & 0xFFFFu, (f >> 16) & 0xFFu};
    const uint32_t per = kBK * stage_blocks(wb, (int)p.bn), stages = (K + per - 1u) / per;
    while (p.splits > 1u && (p.splits > stages || (p.cg == 2u && p.bn / p.splits < 32u) || p.cg * p.splits > 8u)) p.splits >>= 1;   // a slice is never empty
    TileArgs a{};
    a.ep = ep; a.M = M; a.N = N; a.n_out = ep.gated ? N / 2u : N; a.splits = p.splits;
    a.y_vec = aligned16(ep.y) && (ep.y_stride & 7u) == 0u;
    a.res_vec = aligned16(ep.res) && (ep.res_stride & 7u) == 0u;
    a.status = wait_status_sink();
    const uint32_t key = (uint32_t)wb * 10000u + p.cg * 1000u + p.bn;
    switch (key) {
        case 22256: return launch_tile<2, 2, 256>(w, x, x_pitch, K, a, stream, pdl);
        case 22128: return launch_tile<2, 2, 128>(w, x, x_pitch, K, a, stream, pdl);
        case 21128: return launch_tile<2, 1, 128>(w, x, x_pitch, K, a, stream, pdl);
        case 21064: return launch_tile<2, 1, 64>(w, x, x_pitch, K, a, stream, pdl);
        case 12256: return launch_tile<1, 2, 256>(w, x, x_pitch, K, a, stream, pdl);
        case 12128: return launch_tile<1, 2, 128>(w, x, x_pitch, K, a, stream, pdl);
        case 11128: return launch_tile<1, 1, 128>(w, x, x_pitch, K, a, stream, pdl);
        case 11064: return launch_tile<1, 1, 64>(w, x, x_pitch, K, a, stream, pdl);
        default: set_error("linear_tile: no kernel for plan %u", key); return MC_E_INTERNAL;
    }
}

int linear_tile_take_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tile_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) {
        const int zero = 0;
        (void)cudaMemcpyToSymbol(g_tile_error, &zero, sizeof(int));
    }
    return v;
}

}  // namespace mcl
