// logits.cu -- the rules a request puts on its logits (penalties, biases, grammar mask) and the token history they read.
#include "common.cuh"

namespace mcl {

namespace {

constexpr uint32_t kLogitsThreads = 256;

struct LogitsArgs {
    const uint16_t* in;
    uint16_t* out;
    uint32_t vocab, row_stride, out_stride;
    int32_t index_base;
    const mc_sm100_logits_config_t* cfg;
    mc_sm100_logits_tables_t t;
};

// A CTA owns kSpan consecutive columns of a row (counted from a 32-byte boundary of the output, so that rows of any length
// and stride move in 32-byte accesses but for their ends), a thread sixteen.  Reading and writing the logits
// is 4 bytes a token; seen bits and masks are 1/16 of that, and counts are gathered for seen tokens only.  At full batches the
// instructions bound it, not the bytes: most tokens are neither seen nor listed and stay the bits that they are, a mask is a
// select on the packed words (64 rows of 122753 with every rule: 36 us with every token through the fp32 path, 24.5 us with
// every piece that holds a touched token, 29.5 us with touched tokens always one a lane; the rule below 16.3 us, 11.4 in a chain, bound by
// instructions and latency alike).
// The rows' first spans go first: the most frequent tokens, seen or listed (twice, too), are a vocabulary's first, and the CTAs
// that hold them take longest (64 rows with 300 biases each, in a chain: 11.4 us; a row's spans one after another 13.8).
// Biases: a token that the list holds once takes its value straight away.  If one of a span's is listed twice, the entries
// that fall into the span are kept in list order in shared memory, where one warp
// adds them up, 32 at a time: a fixed order, no floating-point atomics, any list length (512 entries at a time).  25 rows of 5164,
// 366 biases that repeat tokens: 9.0 us; a thread an entry that looks for the others like it, 12.2.
constexpr uint32_t kOwn = 16, kSpan = kLogitsThreads * kOwn, kBiasBatch = 2 * kLogitsThreads, kFew = 64;

__global__ void __launch_bounds__(kLogitsThreads, 5) logits_process_kernel(const LogitsArgs a) {
    __shared__ __align__(16) uint32_t s_column[kBiasBatch];
    __shared__ __align__(16) float s_sum[kSpan];
    __shared__ float s_value[kBiasBatch];
    __shared__ uint2 s_touched[kLogitsThreads / 32][kFew];
    __shared__ uint32_t s_listed[kSpan / 32], s_once[kSpan / 32], s_warp[kBiasBatch / 32];
    const uint32_t row = blockIdx.x, block = blockIdx.z * gridDim.y + blockIdx.y, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    pdl_trigger();
    for (uint32_t w = tid; w < kSpan / 32; w += kLogitsThreads) s_once[w] = 0u;
    pdl_wait();
    const mc_sm100_logits_config_t c = a.cfg[row];
    const uint16_t* in = a.in + (size_t)row * a.row_stride;
    uint16_t* out = a.out + (size_t)row * a.out_stride;
    // this thread's columns first .. + 15; those below 0 or beyond the row are not there
    const int32_t head = (int32_t)((reinterpret_cast<uintptr_t>(out) & 31u) >> 1), vocab = (int32_t)a.vocab;
    const int32_t span0 = (int32_t)(block * kSpan) - head, first = span0 + (int32_t)(tid * kOwn);
    const bool together = ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 31u) == 0u;
    const bool whole = first >= 0 && first + (int32_t)kOwn <= vocab;
    uint32_t raw[8];
    if (together && whole) {
        asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]), "=r"(raw[4]), "=r"(raw[5]), "=r"(raw[6]), "=r"(raw[7]) : "l"(in + first));
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) raw[k] = 0u;
#pragma unroll
        for (int e = 0; e < (int)kOwn; ++e)
            if (first + e >= 0 && first + e < vocab) raw[e >> 1] |= (uint32_t)in[first + e] << (16 * (e & 1));
    }
    const uint32_t words = (a.t.table_vocab + 31u) / 32u;
    const bool history = c.history_slot >= 0 && (uint32_t)c.history_slot < a.t.n_slots;
    const bool masked = c.mask_row >= 0 && (uint32_t)c.mask_row < a.t.n_masks;
    const uint64_t end64 = (uint64_t)c.bias_begin + c.bias_count;
    if (a.t.d_status != nullptr && block == 0u && tid == 0u &&
        ((c.history_slot >= 0 && !history) || (c.mask_row >= 0 && !masked) || (c.bias_count != 0u && end64 > a.t.n_bias)))
        *a.t.d_status = 1;
    // the bits of a table row that belong to the columns, bit e = column first + e, 0 where there is none
    const int32_t c_lo = first < 0 ? 0 : first, c_hi = first + (int32_t)kOwn < vocab ? first + (int32_t)kOwn : vocab;
    const uint32_t bit0 = (uint32_t)(a.index_base + c_lo), bit1 = (uint32_t)(a.index_base + c_hi - 1);
    auto bits_of = [&](const uint32_t* table_row) -> uint32_t {
        if (c_hi <= c_lo) return 0u;
        const uint32_t w0 = table_row[bit0 >> 5], w1 = table_row[bit1 >> 5];
        return (__funnelshift_r(w0, w1, bit0 & 31u) & ((1u << (c_hi - c_lo)) - 1u)) << (c_lo - first);
    };
    const uint32_t seen = history ? bits_of(a.t.d_seen + (size_t)c.history_slot * words) : 0u;
    const uint32_t allowed = masked ? bits_of(a.t.d_mask + (size_t)c.mask_row * words) : 0xFFFFu;
    uint32_t listed = 0u;
    const uint32_t begin = c.bias_begin, end = (uint32_t)(end64 < a.t.n_bias ? end64 : a.t.n_bias);
    if (begin < end) {                                                               // the same for every thread
        const int32_t lo = span0 < 0 ? 0 : span0, hi = span0 + (int32_t)kSpan < vocab ? span0 + (int32_t)kSpan : vocab;
        const bool one = end - begin <= kBiasBatch;
        uint32_t col[2];
        float value[2];
        auto load = [&](uint32_t j0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t d = (uint32_t)h * kLogitsThreads + tid;
                int32_t column = -1;
                value[h] = 0.f;
                // tokens and index_base are not negative, or the difference is: no overflow
                if (d < end - j0) { const int32_t tok = a.t.d_bias_token[j0 + d]; column = tok < 0 ? -1 : tok - a.index_base; value[h] = a.t.d_bias_value[j0 + d]; }
                col[h] = column >= lo && column < hi ? (uint32_t)(column - span0) : 0xFFFFFFFFu;
            }
        };
        bool several = !one;
        if (one) {
            // no token of the span listed twice, as nearly always: its one entry is its sum
            load(begin);
            __syncthreads();                                                         // s_once is zero
            int twice = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (col[h] != 0xFFFFFFFFu) {
                    const uint32_t bit = 1u << (col[h] & 31u);
                    if (atomicOr(&s_once[col[h] >> 5], bit) & bit) twice = 1;
                    else s_sum[col[h]] = __fadd_rn(0.f, value[h]);
                }
            several = __syncthreads_or(twice) != 0;
        } else {
            for (uint32_t w = tid; w < kSpan / 32; w += kLogitsThreads) s_listed[w] = 0u;
        }
        for (uint32_t j0 = begin; several && j0 < end; j0 = end - j0 > kBiasBatch ? j0 + kBiasBatch : end) {
            uint32_t hits[2];
            if (!one) load(j0);
            for (uint32_t w = tid; w < kSpan / 32; w += kLogitsThreads) s_once[w] = 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                hits[h] = __ballot_sync(0xFFFFFFFFu, col[h] != 0xFFFFFFFFu);
                if (lane == 0) s_warp[h * (kLogitsThreads / 32) + warp] = __popc(hits[h]);
            }
            __syncthreads();
            constexpr uint32_t kCounts = kBiasBatch / 32;
            uint32_t upto = lane < kCounts ? s_warp[lane] : 0u;
#pragma unroll
            for (uint32_t d = 1; d < kCounts; d <<= 1) {
                const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                if (lane >= d) upto += v;
            }
            const uint32_t total = __shfl_sync(0xFFFFFFFFu, upto, kCounts - 1u);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t at = h * (kLogitsThreads / 32) + warp, before = __shfl_sync(0xFFFFFFFFu, upto, at) - __popc(hits[h]);
                if (col[h] != 0xFFFFFFFFu) {
                    const uint32_t k = before + __popc(hits[h] & ((1u << lane) - 1u)), bit = 1u << (col[h] & 31u);
                    s_column[k] = col[h]; s_value[k] = value[h];
                    atomicOr(&s_once[col[h] >> 5], bit);
                    if (one || !(s_listed[col[h] >> 5] & bit)) s_sum[col[h]] = 0.f;  // else the sum of the batches before
                }
            }
            __syncthreads();
            if (warp == 0u)
                for (uint32_t k0 = 0; k0 < total; k0 += 32u) {                       // 32 entries: a token's first lane adds its entries up
                    const bool have = k0 + lane < total;
                    const uint32_t mine = have ? s_column[k0 + lane] : 0xFFFFFFFFu;
                    const float v = have ? s_value[k0 + lane] : 0.f;
                    uint32_t left = __match_any_sync(0xFFFFFFFFu, mine);
                    const bool first_lane = have && (uint32_t)__ffs((int)left) - 1u == lane;
                    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, first_lane ? (uint32_t)__popc(left) : 0u);
                    float sum = first_lane ? s_sum[mine] : 0.f;
                    for (uint32_t i = 0; i < most; ++i) {
                        const float add = __shfl_sync(0xFFFFFFFFu, v, left != 0u ? __ffs((int)left) - 1 : 0);
                        if (left != 0u) sum = __fadd_rn(sum, add);
                        left &= left - 1u;
                    }
                    if (first_lane) s_sum[mine] = sum;
                    __syncwarp();
                }
            __syncthreads();
            if (!one) {
                for (uint32_t w = tid; w < kSpan / 32; w += kLogitsThreads) s_listed[w] |= s_once[w];
                __syncthreads();
            }
        }
        listed = ((one ? s_once : s_listed)[tid >> 1] >> (16u * (tid & 1u))) & 0xFFFFu;
    }
    // one reciprocal a row instead of a division a token: off by 2^-24 of the value, in front of a rounding of 2^-9
    const float grow = c.rep_penalty != 0.f ? c.rep_penalty : 1.f, shrink = __frcp_rn(grow);
    const int32_t* counts = history ? a.t.d_counts + (size_t)c.history_slot * a.t.table_vocab + a.index_base : nullptr;
    auto edit = [&](float l, bool was_seen, int32_t n, bool has_bias, float b) {
        l = was_seen ? __fmul_rn(l, l > 0.f ? shrink : grow) : l;
        l = n > 0 ? __fsub_rn(__fsub_rn(l, __fmul_rn(c.freq_penalty, (float)n)), c.pres_penalty) : l;
        return has_bias ? __fadd_rn(l, b) : l;
    };
    const uint32_t touched = (seen | listed) & allowed;          // a banned token's value does not matter any more
    // Few touched tokens in the warp (nearly everywhere but among a vocabulary's most frequent tokens): every piece goes out
    // under its mask, then the touched tokens are edited one a lane.  Many: each lane edits its own, eight side by side.
    const uint32_t mine = __popc(touched), total = __reduce_add_sync(0xFFFFFFFFu, mine);
    const bool few = total <= kFew;
    uint32_t res[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) res[k] = raw[k];
    if (!few) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t t = touched >> (8u * h), s = seen >> (8u * h), b = listed >> (8u * h);
            if ((t & 0xFFu) == 0u) continue;
            const uint32_t at = tid * kOwn + 8u * h;
            int32_t n_of[8];
            float add[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) n_of[e] = ((s & t) >> e) & 1u ? counts[span0 + (int32_t)at + e] : 0;
            const float4 b0 = *reinterpret_cast<const float4*>(s_sum + at), b1 = *reinterpret_cast<const float4*>(s_sum + at + 4);
            add[0] = b0.x; add[1] = b0.y; add[2] = b0.z; add[3] = b0.w; add[4] = b1.x; add[5] = b1.y; add[6] = b1.z; add[7] = b1.w;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint32_t& word = res[4 * h + (e >> 1)];
                const uint32_t old = (e & 1) ? word >> 16 : word & 0xFFFFu;
                const float l = edit(__uint_as_float(old << 16), (s >> e) & 1u, n_of[e], (b >> e) & 1u, add[e]);
                const uint32_t bits = (t >> e) & 1u ? f32_to_bf16_bits(l) : old;
                word = (e & 1) ? (word & 0xFFFFu) | (bits << 16) : (word & 0xFFFF0000u) | bits;
            }
        }
    }
    if (masked) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t keep = ((allowed >> (2 * k)) & 1u) * 0xFFFFu + ((allowed >> (2 * k + 1)) & 1u) * 0xFFFF0000u;
            res[k] = (res[k] & keep) | (0xFF80FF80u & ~keep);                        // -infinity
        }
    }
    if (whole) {
        uint32_t changed = in != out ? 1u : 0u;                  // in place, what stays as it was is not written
#pragma unroll
        for (int k = 0; k < 8; ++k) changed |= res[k] ^ raw[k];
        if (changed != 0u)
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + first), "r"(res[0]), "r"(res[1]), "r"(res[2]), "r"(res[3]),
                         "r"(res[4]), "r"(res[5]), "r"(res[6]), "r"(res[7]) : "memory");
    } else {
#pragma unroll
        for (int e = 0; e < (int)kOwn; ++e)
            if (first + e >= 0 && first + e < vocab) out[first + e] = (uint16_t)(res[e >> 1] >> (16 * (e & 1)));
    }
    if (!few || total == 0u) return;
    uint32_t upto = mine;
#pragma unroll
    for (uint32_t d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, upto, d);
        if (lane >= d) upto += v;
    }
    uint32_t at = upto - mine;
    for (uint32_t t = touched; t != 0u; t &= t - 1u, ++at) {
        const uint32_t e = (uint32_t)__ffs((int)t) - 1u, q = e >> 1;
        const uint32_t w4 = q & 4u ? (q & 2u ? (q & 1u ? raw[7] : raw[6]) : (q & 1u ? raw[5] : raw[4])) : (q & 2u ? (q & 1u ? raw[3] : raw[2]) : (q & 1u ? raw[1] : raw[0]));
        s_touched[warp][at] = make_uint2((tid * kOwn + e) | (((seen >> e) & 1u) << 30) | (((listed >> e) & 1u) << 31), e & 1u ? w4 & 0xFFFF0000u : w4 << 16);
    }
    __syncwarp();                                                // the list, and what was stored above, are the whole warp's
    for (uint32_t k = lane; k < total; k += 32u) {
        const uint2 t = s_touched[warp][k];
        const uint32_t in_span = t.x & 0x3FFFFFFFu;
        const int32_t col = span0 + (int32_t)in_span;
        const bool was_seen = (t.x >> 30) & 1u;
        out[col] = f32_to_bf16_bits(edit(__uint_as_float(t.y), was_seen, was_seen ? counts[col] : 0, t.x >> 31, s_sum[in_span]));
    }
}

struct HistoryArgs {
    int32_t* counts;
    uint32_t* seen;
    uint32_t n_slots, vocab;
    const int32_t* tokens;
    uint32_t n_tokens;
    const uint32_t* offsets;
    const uint32_t* prompt_len;
    const int32_t* slots;
    int32_t* status;
};

// Sequence `seq`: its slot and its tokens; false (and the status word raised) when they lie outside the tables.
__device__ __forceinline__ bool history_seq(const HistoryArgs& a, uint32_t seq, uint32_t& slot, uint32_t& lo, uint32_t& hi) {
    const int32_t s = a.slots != nullptr ? a.slots[seq] : (int32_t)seq;
    lo = a.offsets != nullptr ? a.offsets[seq] : seq;
    hi = a.offsets != nullptr ? a.offsets[seq + 1u] : seq + 1u;
    slot = (uint32_t)s;
    const bool ok = s >= 0 && slot < a.n_slots && lo <= hi && hi <= a.n_tokens;
    if (!ok && a.status != nullptr && threadIdx.x == 0u) *a.status = 1;
    return ok;
}

// Rebuild: a CTA owns `span` tokens of the vocabulary of one slot.  It counts in shared memory over the slot's tokens and
// writes each count and seen bit once: no clearing pass, no global atomics, one launch; the token
// list is read once per span (from L2 after the first).  Of several sequences that name a slot the first owns it and the
// others add to its counts.
constexpr uint32_t kHistThreads = 256;

__global__ void __launch_bounds__(kHistThreads, 4) history_rebuild_kernel(const HistoryArgs a, uint32_t n_seqs, uint32_t span) {
    extern __shared__ __align__(16) int32_t s_hist[];            // [span + 4] counts, [span / 32] seen bits
    __shared__ uint32_t s_same[kHistThreads / 32];
    pdl_trigger();
    pdl_wait();
    const uint32_t seq = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    uint32_t slot, lo, hi;
    const bool valid = history_seq(a, seq, slot, lo, hi);
    for (uint32_t i = tid; i < (span + 4u + span / 32u + 3u) / 4u; i += kHistThreads) reinterpret_cast<uint4*>(s_hist)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (!valid) return;
    const uint32_t t0 = blockIdx.y * span, t1 = min(a.vocab, t0 + span);
    // counts stand in shared memory as far from a 16-byte boundary as in the table: rows of any length go out 16 bytes at a time
    int32_t* row = a.counts + (size_t)slot * a.vocab + t0;
    const uint32_t shift = (uint32_t)((reinterpret_cast<uintptr_t>(row) & 15u) >> 2);
    int32_t* s_count = s_hist + shift;
    uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_hist + span + 4u);
    auto add = [&](uint32_t which, uint32_t l, uint32_t h) {
        const uint32_t n = h - l, prompt = a.prompt_len != nullptr ? a.prompt_len[which] : 0u;
        const int32_t* src = a.tokens + l;
        for (uint32_t k0 = tid; k0 < n; k0 += kHistThreads * 16u) {
            uint32_t tok[16];
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) tok[e] = k0 + e * kHistThreads < n ? (uint32_t)src[k0 + e * kHistThreads] : 0xFFFFFFFFu;
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) {
                if (tok[e] < t0 || tok[e] >= t1) continue;
                const uint32_t t = tok[e] - t0;
                atomicOr(s_seen + t / 32u, 1u << (t & 31u));
                if (k0 + e * kHistThreads >= prompt) atomicAdd(s_count + t, 1);
            }
        }
    };
    if (a.slots == nullptr) {
        __syncthreads();
        add(seq, lo, hi);
    } else {
        // one look over the sequences: does an earlier one own the slot, which later ones join
        bool counted = false;
        for (uint32_t j0 = 0; j0 < n_seqs; j0 += kHistThreads) {
            const uint32_t j = j0 + tid;
            uint32_t s, l, h;
            const bool same = j != seq && j < n_seqs && history_seq(a, j, s, l, h) && s == slot;
            const uint32_t hits = __ballot_sync(0xFFFFFFFFu, same);
            if (lane == 0) s_same[warp] = hits;
            if (__syncthreads_or(same && j < seq ? 1 : 0)) return;
            if (!counted && j0 + kHistThreads > seq) { add(seq, lo, hi); counted = true; }
            for (uint32_t w = 0; w < kHistThreads / 32u; ++w)
                for (uint32_t m = s_same[w]; m != 0u; m &= m - 1u) {
                    const uint32_t other = j0 + w * 32u + (uint32_t)__ffs((int)m) - 1u;
                    (void)history_seq(a, other, s, l, h);
                    add(other, l, h);
                }
            __syncthreads();
        }
    }
    __syncthreads();
    const uint32_t words = (a.vocab + 31u) / 32u;
    const uint32_t n = t1 - t0, upto = shift + n;                 // shared entries [shift, upto) are the table's
    int32_t* table = row - shift;
    for (uint32_t i = tid * 4u; i < upto; i += kHistThreads * 4u) {
        const int4 v = *reinterpret_cast<const int4*>(s_hist + i);
        if (i >= shift && i + 4u <= upto) {
            *reinterpret_cast<int4*>(table + i) = v;
        } else {
            const int32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (i + k >= shift && i + k < upto) table[i + k] = e[k];
        }
    }
    for (uint32_t i = tid; i < (n + 31u) / 32u; i += kHistThreads) a.seen[(size_t)slot * words + t0 / 32u + i] = s_seen[i];
}

// Append: integer atomics, whose order does not show in the result.
__global__ void __launch_bounds__(kLogitsThreads) history_add_kernel(const HistoryArgs a) {
    pdl_trigger();
    pdl_wait();
    uint32_t slot, lo, hi;
    if (!history_seq(a, blockIdx.x, slot, lo, hi)) return;
    const uint32_t words = (a.vocab + 31u) / 32u, n = hi - lo, prompt = a.prompt_len != nullptr ? a.prompt_len[blockIdx.x] : 0u;
    for (uint32_t j = blockIdx.y * kLogitsThreads + threadIdx.x; j < n; j += gridDim.y * kLogitsThreads) {
        const uint32_t tok = (uint32_t)a.tokens[lo + j];
        if (tok >= a.vocab) continue;
        atomicOr(a.seen + (size_t)slot * words + tok / 32u, 1u << (tok & 31u));
        if (j >= prompt) atomicAdd(a.counts + (size_t)slot * a.vocab + tok, 1);
    }
}

// Tables are words: misaligned ones are refused, not read.
template <typename... P> bool words_aligned(const P*... p) { return ((reinterpret_cast<uintptr_t>(p) | ...) & 3u) == 0u; }

}  // namespace

}  // namespace mcl

using namespace mcl;

extern "C" {

// The kernels of this file wait for the previous kernel before they read anything; they are always launched with the
// programmatic attribute, which lets their launch and set-up run under its end.
mc_status_t mc_sm100_logits_process(const mc_sm100_logits_process_t* call, const mc_sm100_logits_tables_t* tables, void* stream, int32_t) {
    clear_error();
    const char* who = "mc_sm100_logits_process";
    if (call == nullptr || call->struct_size != sizeof(mc_sm100_logits_process_t)) {
        set_error("%s: invalid call struct (struct_size=%u)", who, call ? call->struct_size : 0u);
        return MC_E_INVALID_ARGUMENT;
    }
    const uint32_t n_rows = call->n_rows, vocab = call->vocab, row_stride = call->row_stride, out_stride = call->out_stride;
    const int32_t index_base = call->index_base;
    if (call->d_logits == nullptr || call->d_out == nullptr || call->d_cfg == nullptr || tables == nullptr || n_rows == 0 || n_rows > 65535u ||
        vocab == 0 || row_stride < vocab || out_stride < vocab || index_base < 0 ||
        (call->d_logits == call->d_out && row_stride != out_stride) || ((reinterpret_cast<uintptr_t>(call->d_logits) | reinterpret_cast<uintptr_t>(call->d_out)) & 1u) != 0u) {
        set_error("%s: invalid args (rows=%u vocab=%u strides=%u,%u index_base=%d)", who, n_rows, vocab, row_stride, out_stride, index_base);
        return MC_E_INVALID_ARGUMENT;
    }
    const mc_sm100_logits_tables_t& t = *tables;
    if (t.struct_size != sizeof(mc_sm100_logits_tables_t) || t.reserved != 0u || t.table_vocab > 0x10000000u ||
        (uint64_t)index_base + vocab > t.table_vocab || (t.n_slots != 0u && (t.d_counts == nullptr || t.d_seen == nullptr)) ||
        (t.n_masks != 0u && t.d_mask == nullptr) || (t.n_bias != 0u && (t.d_bias_token == nullptr || t.d_bias_value == nullptr)) ||
        !words_aligned(call->d_cfg, t.d_counts, t.d_seen, t.d_mask, t.d_bias_token, t.d_bias_value, t.d_status)) {
        set_error("%s: invalid tables (struct_size=%u table_vocab=%u slots=%u masks=%u biases=%u) for columns %d..%llu", who, t.struct_size,
                  t.table_vocab, t.n_slots, t.n_masks, t.n_bias, index_base, (unsigned long long)((uint64_t)index_base + vocab));
        return MC_E_INVALID_ARGUMENT;
    }
    const LogitsArgs a{call->d_logits, call->d_out, vocab, row_stride, out_stride, index_base, call->d_cfg, t};
    const uint32_t spans = (vocab + kOwn - 1u + kSpan - 1u) / kSpan, deep = (spans + 65534u) / 65535u;
    (void)launch(logits_process_kernel, dim3(n_rows, (spans + deep - 1u) / deep, deep), dim3(kLogitsThreads), 0,
                 (cudaStream_t)stream, true, a);
    MCL_CHECK_LAUNCH("logits_process");
    return MC_OK;
}

mc_status_t mc_sm100_token_history(const mc_sm100_token_history_t* call, void* stream, int32_t) {
    clear_error();
    if (call == nullptr || call->struct_size != sizeof(mc_sm100_token_history_t) || call->rebuild > 1u) {
        set_error("mc_sm100_token_history: invalid call struct (struct_size=%u rebuild=%u)", call ? call->struct_size : 0u, call ? call->rebuild : 0u);
        return MC_E_INVALID_ARGUMENT;
    }
    const mc_sm100_token_history_t& d = *call;
    const uint32_t n_seqs = d.n_seqs, table_vocab = d.table_vocab;
    if (d.d_counts == nullptr || d.d_seen == nullptr || d.n_slots == 0 || d.n_slots > 0x7FFFFFFFu || table_vocab == 0 || table_vocab > 0x10000000u ||
        (d.d_tokens == nullptr && d.n_tokens != 0u) || n_seqs == 0 || n_seqs > 0x7FFFFFFFu || (d.d_offsets == nullptr && d.n_tokens < n_seqs) ||
        (d.d_slots == nullptr && n_seqs > d.n_slots) || d.n_tokens > 0x7FFFFFFFu ||
        !words_aligned(d.d_counts, d.d_seen, d.d_tokens, d.d_offsets, d.d_prompt_len, d.d_slots, d.d_status)) {
        set_error("mc_sm100_token_history: invalid args (slots=%u vocab=%u tokens=%u sequences=%u)", d.n_slots, table_vocab, d.n_tokens, n_seqs);
        return MC_E_INVALID_ARGUMENT;
    }
    const HistoryArgs a{d.d_counts, d.d_seen, d.n_slots, table_vocab, d.d_tokens, d.n_tokens, d.d_offsets, d.d_prompt_len, d.d_slots, d.d_status};
    if (d.rebuild != 0u) {
        // One round of CTAs, four to an SM (56 KB each) where the batch allows it: spans of 2048 to 13664 tokens.
        // 64 slots of 122753: 9 spans, 576 CTAs in one round: 10.9 us; with spans of 16384 (three CTAs to an SM, two rounds) 13.5 us.
        const uint64_t spans = 4ull * (uint32_t)sm_count() / n_seqs;
        uint64_t span = spans == 0 ? table_vocab : ((uint64_t)table_vocab + spans - 1u) / spans;
        span = span < 2048u ? 2048u : (span > 13664u ? 13664u : (span + 31u) & ~(uint64_t)31u);
        const size_t bytes = ((size_t)span + 4u) * 4u + (size_t)span / 8u + 16u;
        static SmemOptIn optin;
        const cudaError_t e = optin.ensure(history_rebuild_kernel, bytes);
        if (e != cudaSuccess) {
            set_error("mc_sm100_token_history: cannot raise shared memory to %zu: %s", bytes, cudaGetErrorString(e));
            return MC_E_CUDA;
        }
        (void)launch(history_rebuild_kernel, dim3(n_seqs, (uint32_t)((table_vocab + span - 1u) / span)), dim3(kHistThreads), bytes,
                     (cudaStream_t)stream, true, a, n_seqs, (uint32_t)span);
        MCL_CHECK_LAUNCH("history_rebuild");
        return MC_OK;
    }
    (void)launch(history_add_kernel, dim3(n_seqs, d.d_offsets != nullptr ? 8 : 1), dim3(kLogitsThreads), 0, (cudaStream_t)stream, true, a);
    MCL_CHECK_LAUNCH("history_add");
    return MC_OK;
}

}  // extern "C"
