// linear_epilogue.cu -- mc_sm100_linear_epilogue: checks, choice of a kernel, and the kernel that takes every shape.
#include "linear_epilogue.cuh"

#include <type_traits>

#include "fast_dispatch.cuh"
#include "linear_rows.cuh"
#include "linear_tile.cuh"
#include "skinny_gemm.cuh"

namespace mcl {

namespace {

// ---- any shape, any stride, any alignment ------------------------------------------------------
// 64 x 64 tiles of y, K in steps of 64, mma.sync m16n8k16 with fp32 accumulators, plain element loads with bounds, a step's
// loads in registers before the step in front of it is multiplied (610 x 5192 e4m3, M = 20: 192 us; element by element 772).
// e4m3 codes are widened to bf16 (exact).  Each warp owns a 32 x 32 quarter.
constexpr uint32_t kAnyTile = 64, kAnyK = 64, kAnyPitch = kAnyK + 8, kAnyThreads = 128;

__device__ __forceinline__ void any_mma(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

template <int WB>
__global__ void __launch_bounds__(kAnyThreads)
linear_any_kernel(const void* __restrict__ w, const uint16_t* __restrict__ x, uint32_t x_stride, uint32_t M, uint32_t N, uint32_t K,
                  uint32_t n_tiles, const EpiArgs e) {
    __shared__ uint16_t sx[kAnyTile][kAnyPitch], sw[kAnyTile][kAnyPitch];
    __shared__ float sz[kAnyTile][kAnyTile + 1];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t m0 = (blockIdx.x / n_tiles) * kAnyTile, n0 = (blockIdx.x % n_tiles) * kAnyTile;
    const uint32_t wm = (warp & 1u) * 32u, wn = (warp >> 1) * 32u;
    pdl_trigger();
    pdl_wait();
    float acc[2][4][4] = {};
    constexpr uint32_t kEach = kAnyTile * kAnyK / kAnyThreads;               // elements of x, and of W, that a thread loads a step
    using W = std::conditional_t<WB == 2, uint16_t, uint8_t>;
    const uint32_t c = tid % kAnyK, r0 = tid / kAnyK;                        // one column, every second row
    const W* wt = static_cast<const W*>(w);
    uint16_t vx[kEach];
    W vw[kEach];
    auto fetch = [&](uint32_t k0) {
        const bool in = k0 + c < K;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t r = r0 + i * (kAnyThreads / kAnyK);
            vx[i] = in && m0 + r < M ? x[(size_t)(m0 + r) * x_stride + k0 + c] : (uint16_t)0;
            vw[i] = in && n0 + r < N ? wt[(size_t)(n0 + r) * K + k0 + c] : (W)0;
        }
    };
    fetch(0);
    for (uint32_t k0 = 0; k0 < K; k0 += kAnyK) {
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t r = r0 + i * (kAnyThreads / kAnyK);
            sx[r][c] = vx[i];
            if constexpr (WB == 2) sw[r][c] = vw[i];
            else sw[r][c] = f32_to_bf16_bits(e4m3_to_f32(vw[i]));
        }
        if (K - k0 > kAnyK) fetch(k0 + kAnyK);
        __syncthreads();
#pragma unroll
        for (uint32_t kk = 0; kk < kAnyK; kk += 16) {
            uint32_t a[2][4], b[4][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 4; ++h)
                    a[i][h] = *reinterpret_cast<const uint32_t*>(&sx[wm + 16 * i + g + 8 * (h & 1)][kk + 2 * t + 8 * (h >> 1)]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) b[j][h] = *reinterpret_cast<const uint32_t*>(&sw[wn + 8 * j + g][kk + 2 * t + 8 * h]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) any_mma(acc[i][j], a[i], b[j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < 4; ++h) sz[wm + 16 * i + g + 8 * (h >> 1)][wn + 8 * j + 2 * t + (h & 1)] = acc[i][j][h];
    __syncthreads();
    const uint32_t cols = e.gated ? kAnyTile / 2 : kAnyTile, c0 = e.gated ? n0 / 2 : n0, n_out = e.gated ? N / 2 : N;
    auto z_of = [&](uint32_t r, uint32_t n_rel) {
        float z = sz[r][n_rel];
        const uint32_t n = n0 + n_rel;
        if (e.scale != nullptr) z *= e.scale[n];
        if (e.bias != nullptr) z += __uint_as_float((uint32_t)e.bias[n] << 16);
        return z;
    };
    for (uint32_t i = tid; i < kAnyTile * cols; i += kAnyThreads) {
        const uint32_t r = i / cols, c = i % cols, m = m0 + r, j = c0 + c;
        if (m >= M || j >= n_out) continue;
        float v = e.gated ? epi_act(z_of(r, 2 * c), e.act) * z_of(r, 2 * c + 1) : epi_act(z_of(r, c), e.act);
        if (e.res != nullptr) v += __uint_as_float((uint32_t)e.res[(size_t)m * e.res_stride + j] << 16);
        e.y[(size_t)m * e.y_stride + j] = f32_to_bf16_bits(v);
    }
}

mc_status_t linear_any(int wb, const void* w, const uint16_t* x, uint32_t x_stride, uint32_t M, uint32_t N, uint32_t K,
                       const EpiArgs& e, cudaStream_t stream, bool pdl) {
    const uint64_t nt = (N + kAnyTile - 1ull) / kAnyTile, mt = (M + kAnyTile - 1ull) / kAnyTile;
    if (nt * mt > 0x7FFFFFFFull) {
        set_error("mc_sm100_linear_epilogue: M=%u N=%u make too many tiles", M, N);
        return MC_E_UNSUPPORTED;
    }
    auto kern = wb == 2 ? linear_any_kernel<2> : linear_any_kernel<1>;
    (void)launch(kern, dim3((uint32_t)(nt * mt)), dim3(kAnyThreads), 0, stream, pdl, w, x, x_stride, M, N, K, (uint32_t)nt, e);
    MCL_CHECK_LAUNCH("linear_any");
    return MC_OK;
}

bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1u)) == 0u; }

}  // namespace

}  // namespace mcl

using namespace mcl;

extern "C" mc_status_t mc_sm100_linear_epilogue(const mc_sm100_linear_epilogue_t* call, void* stream, int32_t pdl) {
    clear_error();
    if (call == nullptr || call->struct_size != sizeof(mc_sm100_linear_epilogue_t) || call->activation > MC_SM100_ACT_SILU || call->gated > 1u ||
        call->reserved != 0u) {
        set_error("mc_sm100_linear_epilogue: invalid call struct (struct_size=%u activation=%u gated=%u)", call ? call->struct_size : 0u,
                  call ? call->activation : 0u, call ? call->gated : 0u);
        return MC_E_INVALID_ARGUMENT;
    }
    const mc_sm100_linear_epilogue_t& d = *call;
    const void* d_w = d.d_w;
    const float* d_scale = d.d_scale;
    const uint16_t* d_x = d.d_x;
    uint16_t* d_y = d.d_y;
    const uint32_t M = d.M, N = d.N, K = d.K;
    const int wb = d_scale == nullptr ? 2 : 1;
    const uint32_t n_out = d.gated ? N / 2u : N;
    const uint32_t xs = d.x_stride ? d.x_stride : K, ys = d.y_stride ? d.y_stride : n_out, rs = d.residual_stride ? d.residual_stride : n_out;
    constexpr uint32_t kMost = 1u << 30;             // row and column numbers stay in 31 bits, with a tile to spare
    if (d_w == nullptr || d_x == nullptr || d_y == nullptr || M == 0 || N == 0 || K == 0 || M > kMost || N > kMost || K > kMost || (d.gated && (N & 1u) != 0) || xs < K ||
        ys < n_out || (d.d_residual != nullptr && rs < n_out) || !aligned_to(d_w, (uintptr_t)wb) || !aligned_to(d_scale, 4) ||
        !aligned_to(d_x, 2) || !aligned_to(d_y, 2) || !aligned_to(d.d_bias, 2) || !aligned_to(d.d_residual, 2)) {
        set_error("mc_sm100_linear_epilogue: invalid args (M=%u N=%u K=%u gated=%u x_stride=%u y_stride=%u residual_stride=%u)", M, N, K,
                  d.gated, xs, ys, rs);
        return MC_E_INVALID_ARGUMENT;
    }
    if (d.d_residual == d_y && rs != ys) {
        set_error("mc_sm100_linear_epilogue: residual and y are one buffer with strides %u and %u", rs, ys);
        return MC_E_INVALID_ARGUMENT;
    }
    const EpiArgs e{d_scale, d.d_bias, d.d_residual, d_y, ys, rs, d.activation, d.gated, pdl != 0 ? 0u : 1u};
    const cudaStream_t st = (cudaStream_t)stream;
    // Every kernel below is launched with the programmatic attribute, so that its launch and set-up run under the end of the
    // previous kernel; what it reads before that end is nothing (e.wait_first), or with `pdl` the weights.
    // rows that a 16-byte unit divides, at aligned addresses: the kernels that stream
    const bool unit = aligned16(d_w) && aligned16(d_x) && ((uint64_t)K * (uint32_t)wb) % 16u == 0u;
    if (M == 1u && unit && fast_fused_fits(wb, d.gated != 0u, N, K)) {       // the activation in shared memory
        RowsArgs a{};
        a.w = d_w; a.scale = d_scale; a.x = d_x; a.y = d_y; a.N = N; a.K = K; a.y_stride = ys; a.kseg = K; a.ep = e;
        const NextWeights nw = take_next_weights();
        a.pf.ptr = static_cast<const uint8_t*>(nw.ptr); a.pf.bytes = nw.bytes;
        return launch_fast_fused(wb, d.gated != 0u, a, st, true);
    }
    const bool tma = unit && (xs & 7u) == 0u;
    // Up to 64 rows the skinny kernel, which splits K eight ways and pads M to 16, 32 or 64.  From 17 rows on the tiled kernel
    // is faster where K is short for the padded M (M = 32, 4096 x 448: 5.0 against 6.4 us; M = 64, 2304 x 1024: 6.0 against 9.1)
    // or, from 33 on, the weights have many rows (M = 33, lm_head 122753 x 2304: 95 against 115; M = 64, 11520 x 3008: 17.4 against
    // 22.1); elsewhere it is slower (M = 32, 11520 x 1536: a third; M = 64, 2304 x 5760: 16.7 against 13.8).  Over 1900 timings
    // (M 17 .. 64, N 480 .. 122753, K 256 .. 5760) the rule is within 1 % of the better one on average, 32 % in the worst case.
    const bool short_k = M > 16u && K <= (M <= 32u ? 640u : 1280u), tall = M > 32u && N >= 4096u && K <= 80u * M;
    const bool tiled = M > 64u || tile_forced() || short_k || tall;
    if (wb == 1 && M <= 16u && tma && !tile_forced() && linear_rows_ok(M, K, xs))
        return linear_rows(static_cast<const uint8_t*>(d_w), d_x, xs, M, N, K, e, st, true);
    if (!tiled && tma) return skinny_gemm_fused(wb == 2 ? SKINNY_W_BF16 : SKINNY_W_E4M3, d_w, d_x, xs, M, N, K, e, st, true);
    (void)take_next_weights();                       // a hint left for this call is consumed
    if (tma) return linear_tile(wb, d_w, d_x, xs, M, N, K, e, st, true);
    return linear_any(wb, d_w, d_x, xs, M, N, K, e, st, true);
}

extern "C" mc_status_t mc_sm100_debug_set_tile_plan(uint32_t cg, uint32_t bn, uint32_t splits) {
    clear_error();
    return tile_force(cg, bn, splits);
}

extern "C" void mc_sm100_debug_tile_plan(int32_t bytes_per_weight, uint32_t M, uint32_t N, uint32_t K, uint32_t sms, uint32_t* cg,
                                         uint32_t* bn, uint32_t* splits) {
    const TilePlan p = tile_plan(bytes_per_weight, M, N, K, sms);
    if (cg != nullptr) *cg = p.cg;
    if (bn != nullptr) *bn = p.bn;
    if (splits != nullptr) *splits = p.splits;
}
