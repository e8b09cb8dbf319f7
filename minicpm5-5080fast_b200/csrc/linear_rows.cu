// linear_rows.cu -- y = epilogue(x W^T) for 2 <= M <= 16 rows and e4m3 weights, streamed through registers.
//
// The skinny tcgen05 kernel moves every code through shared memory three times (raw tile in, raw tile out, widened tile in)
// and hands a K block from role to role four times; at these M that, not HBM, bounds it.  Here a code goes from its 128-bit
// load through the bit placement straight into a mma.sync.m16n8k16 A fragment: lane (g, t) holds 16 consecutive codes of row
// g and of row 8 + g, four mma per 64 codes; the mma's k is only a label, and the B fragment, the same 16 elements of
// activation row g (+ 8 per further column block), is cut up the same way out of shared memory, where the whole activation
// is staged once per CTA (rows an odd number of 16-byte units apart: no bank is met twice).
// Blocks of 16 weight rows are dealt to the CTAs as contiguous near-equal ranges; a CTA works on R blocks at a time, KW = 16 / R
// warps to a block, which take its 64-element K steps round-robin; their partial tiles meet in shared memory and are added in
// warp order.  Bound by latency where N is small, by the bit placement and mma.sync where it is large (lm_head M = 2: 3.4 TB/s).
// Measured (us, this kernel / skinny): 2304 x 5760 M = 8 8.9 / 12.6, M = 16 12.7 / 12.4; 11520 x 2304 M = 8 12.7 / 13.9, M = 16
// 15.3 / 14.6; 20000 x 4096 M = 8 31.4 / 49, M = 16 39 / 50; 122753 x 2304 M = 8 89 / 107, M = 16 114 / 112.  Four column blocks
// (M <= 32) lost: 11520 x 2304 23.8 / 16.4.
#include "linear_rows.cuh"

#include "gemv_fast.cuh"
#include "tcgen05.cuh"

namespace mcl {

namespace {

constexpr uint32_t kWarps = 16, kThreads = 32 * kWarps, kStep = 64, kU = 4;   // kU K steps per register buffer
constexpr size_t kMostShared = 200u * 1024u;

struct RowsFusedArgs {
    const uint8_t* w;
    const uint16_t* x;
    uint32_t M, N, K, x_pitch;
    uint32_t kw, r;
    EpiArgs ep;
};

constexpr size_t shared_bytes(uint32_t mb, uint32_t K) { return (size_t)8u * mb * (2u * K + 16u) + (size_t)kWarps * 16u * 8u * mb * 4u; }

__device__ __forceinline__ uint4 ld_l2(const void* p) {       // what another kernel may have written: read at L2
    uint4 v;
    asm volatile("ld.global.cg.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

}  // namespace

// MB: 8-row blocks of the activation.
template <uint32_t MB>
__global__ void __launch_bounds__(kThreads, 1) linear_rows_kernel(const RowsFusedArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t K = a.K, N = a.N, M = a.M, pitch = 2u * K + 16u;
    uint8_t* xs = smem;                                                        // [8 MB][pitch] bytes
    float* part = reinterpret_cast<float*>(smem + (size_t)8u * MB * pitch);    // [kWarps][16][8 MB]
    const uint32_t S = (K + kStep - 1u) / kStep, KW = a.kw, R = a.r, kwi = warp % KW, slot = warp / KW;
    const uint32_t my_steps = slot < R && S > kwi ? (S - kwi + KW - 1u) / KW : 0u;
    const uint32_t nb = ((S + KW - 1u) / KW + kU - 1u) / kU;                   // batches per block, the same for every warp
    const uint32_t nblk = (N + 15u) / 16u;
    const uint32_t lo = (uint32_t)((uint64_t)nblk * blockIdx.x / gridDim.x), hi = (uint32_t)((uint64_t)nblk * (blockIdx.x + 1u) / gridDim.x);
    const uint32_t T = (hi - lo + R - 1u) / R * nb;
    const uint64_t policy = l2_policy_stream(true);

    uint4 rawA[kU][2], rawB[kU][2];
    auto issue = [&](uint4 (&raw)[kU][2], uint32_t q) {
        const uint32_t rb = lo + q / nb * R + slot, r0 = rb * 16u + g;
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) {
            const uint32_t i = q % nb * kU + u, k = kStep * (kwi + KW * i) + 16u * t;
            const bool in = rb < hi && i < my_steps && k < K;                   // K is a multiple of 16: a lane's codes are all there or none
            raw[u][0] = in && r0 < N ? ld_stream16_hint(a.w + (size_t)r0 * K + k, policy) : make_uint4(0u, 0u, 0u, 0u);
            raw[u][1] = in && r0 + 8u < N ? ld_stream16_hint(a.w + (size_t)(r0 + 8u) * K + k, policy) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    // two sets of accumulators take alternate mma: half the chain of dependent ones
    float2 d01[2][MB], d23[2][MB];
    auto zero = [&]() {
#pragma unroll
        for (uint32_t c = 0; c < 2u * MB; ++c) { d01[c & 1u][c >> 1] = make_float2(0.f, 0.f); d23[c & 1u][c >> 1] = make_float2(0.f, 0.f); }
    };
    auto consume = [&](uint4 (&raw)[kU][2], uint32_t q) {
#pragma unroll
        for (uint32_t u = 0; u < kU; ++u) {
            const uint32_t i = q % nb * kU + u, k = kStep * (kwi + KW * i) + 16u * t;
            if (i >= my_steps) break;                                          // the same for the whole warp
            const bool in = k < K;
            uint4 xa[MB], xb[MB];
#pragma unroll
            for (uint32_t c = 0; c < MB; ++c) {
                const uint4* xp = reinterpret_cast<const uint4*>(xs + (size_t)(8u * c + g) * pitch + 2u * k);
                xa[c] = in ? xp[0] : make_uint4(0u, 0u, 0u, 0u); xb[c] = in ? xp[1] : make_uint4(0u, 0u, 0u, 0u);
            }
            uint32_t w0[8], w1[8];
            const uint32_t v0[4] = {raw[u][0].x, raw[u][0].y, raw[u][0].z, raw[u][0].w}, v1[4] = {raw[u][1].x, raw[u][1].y, raw[u][1].z, raw[u][1].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) { widen4(v0[j], w0[2 * j], w0[2 * j + 1]); widen4(v1[j], w1[2 * j], w1[2 * j + 1]); }
#pragma unroll
            for (uint32_t c = 0; c < MB; ++c) {
                mma16816_bf16(d01[0][c], d23[0][c], w0[0], w1[0], w0[1], w1[1], xa[c].x, xa[c].y);
                mma16816_bf16(d01[1][c], d23[1][c], w0[2], w1[2], w0[3], w1[3], xa[c].z, xa[c].w);
                mma16816_bf16(d01[0][c], d23[0][c], w0[4], w1[4], w0[5], w1[5], xb[c].x, xb[c].y);
                mma16816_bf16(d01[1][c], d23[1][c], w0[6], w1[6], w0[7], w1[7], xb[c].z, xb[c].w);
            }
        }
    };
    auto bf = [](uint16_t b) { return __uint_as_float((uint32_t)b << 16); };
    // the R blocks of pass q / nb are done
    auto flush = [&](uint32_t q) {
        float* mine = part + warp * (16u * 8u * MB);
#pragma unroll
        for (uint32_t c = 0; c < MB; ++c) {
            *reinterpret_cast<float2*>(mine + g * 8u * MB + 8u * c + 2u * t) = make_float2(d01[0][c].x + d01[1][c].x, d01[0][c].y + d01[1][c].y);
            *reinterpret_cast<float2*>(mine + (g + 8u) * 8u * MB + 8u * c + 2u * t) = make_float2(d23[0][c].x + d23[1][c].x, d23[0][c].y + d23[1][c].y);
        }
        zero();
        if (KW > 1u) __syncthreads(); else __syncwarp();
        const uint32_t first = KW > 1u ? tid : lane, step = KW > 1u ? kThreads : 32u, blocks = KW > 1u ? R : 1u;
        const uint32_t gate = a.ep.gated, sh = 4u - gate, per = M << sh;       // a block's outputs: M rows of 16, behind the gate 8
        for (uint32_t idx = first; idx < blocks * per; idx += step) {
            const uint32_t sl = KW > 1u ? idx / per : slot, e = KW > 1u ? idx % per : idx;
            const uint32_t rb = lo + q / nb * R + sl, m = e >> sh, o = e & ((1u << sh) - 1u), j = ((rb * 16u) >> gate) + o;
            if (sl >= R || rb >= hi || j >= N >> gate) continue;
            auto z_of = [&](uint32_t i) {
                float z = 0.f;
                for (uint32_t w = sl * KW; w < (sl + 1u) * KW; ++w) z += part[w * (16u * 8u * MB) + i * 8u * MB + m];
                z *= a.ep.scale[rb * 16u + i];
                return a.ep.bias != nullptr ? z + bf(a.ep.bias[rb * 16u + i]) : z;
            };
            const float r = a.ep.res != nullptr ? bf(a.ep.res[(size_t)m * a.ep.res_stride + j]) : -0.f;
            const float v = epi_act(z_of(o << gate), a.ep.act) * (gate ? z_of(2u * o + 1u) : 1.0f);
            a.ep.y[(size_t)m * a.ep.y_stride + j] = f32_to_bf16_bits(v + r);
        }
        if (KW > 1u) __syncthreads(); else __syncwarp();
    };

    if (a.ep.wait_first) pdl_wait();
    if (T > 0u) issue(rawA, 0u);
    pdl_trigger();
    pdl_wait();
    // the activation, rows beyond M as zeros
    const uint32_t units = K / 8u;                                             // 16-byte units of a row
    for (uint32_t i = tid; i < 8u * MB * units; i += kThreads) {
        const uint32_t m = i / units, u = i - m * units;
        *reinterpret_cast<uint4*>(xs + (size_t)m * pitch + 16u * u) = m < M ? ld_l2(a.x + (size_t)m * a.x_pitch + 8u * u) : make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
    zero();
    for (uint32_t q = 0; q < T;) {
        if (q + 1u < T) issue(rawB, q + 1u);
        consume(rawA, q);
        if (q % nb == nb - 1u) flush(q);
        if (++q >= T) break;
        if (q + 1u < T) issue(rawA, q + 1u);
        consume(rawB, q);
        if (q % nb == nb - 1u) flush(q);
        ++q;
    }
}

bool linear_rows_ok(uint32_t M, uint32_t K, uint32_t x_pitch) {
    return M >= 2u && M <= 16u && (K & 15u) == 0u && (x_pitch & 7u) == 0u && shared_bytes(M <= 8u ? 1u : 2u, K) <= kMostShared;
}

namespace {

template <uint32_t MB>
mc_status_t launch_rows_fused(const RowsFusedArgs& a, uint32_t grid, cudaStream_t stream, bool pdl) {
    const size_t smem = shared_bytes(MB, a.K);
    static SmemOptIn optin;
    const cudaError_t e = optin.ensure(linear_rows_kernel<MB>, smem);
    if (e != cudaSuccess) {
        set_error("linear_rows: cannot raise shared memory to %zu: %s", smem, cudaGetErrorString(e));
        return MC_E_CUDA;
    }
    (void)launch(linear_rows_kernel<MB>, dim3(grid), dim3(kThreads), smem, stream, pdl, a);
    MCL_CHECK_LAUNCH("linear_rows");
    return MC_OK;
}

}  // namespace

mc_status_t linear_rows(const uint8_t* w, const uint16_t* x, uint32_t x_pitch, uint32_t M, uint32_t N, uint32_t K, const EpiArgs& ep,
                        cudaStream_t stream, bool pdl) {
    const uint32_t nblk = (N + 15u) / 16u, sms = (uint32_t)sm_count(), grid = nblk < sms ? nblk : sms;
    const uint32_t most = (nblk + grid - 1u) / grid, S = (K + kStep - 1u) / kStep;
    // blocks at a time: the fewest K steps that the fullest CTA's warps walk through, a pass's end counted as four
    uint32_t r = 1, steps = 0xFFFFFFFFu;
    for (uint32_t c = 1; c <= kWarps; ++c) {
        const uint32_t kw = kWarps / c, n = (most + c - 1u) / c * ((S + kw - 1u) / kw + 4u);
        if (n <= steps) { steps = n; r = c; }
        if (c >= most) break;
    }
    const RowsFusedArgs a{w, x, M, N, K, x_pitch, kWarps / r, r, ep};
    (void)take_next_weights();
    if (M <= 8u) return launch_rows_fused<1>(a, grid, stream, pdl);
    return launch_rows_fused<2>(a, grid, stream, pdl);
}

}  // namespace mcl
