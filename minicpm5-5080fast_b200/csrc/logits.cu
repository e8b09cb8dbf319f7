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

// A CTA owns kSpan consecutive columns of a row (counted from a 16-byte boundary of the output, so that rows of any length
// and stride are stored in 16-byte pieces but for their ends), a thread one piece of eight.  What costs is reading and
// writing the logits, 4 bytes a token; seen bits and mask are 1/16 of that, and the counts are gathered for seen tokens only.
// The bias list is read once per CTA, 256 entries at a time: those that fall into the span are kept in list order in shared
// memory, and each thread adds up the ones of its own tokens: a fixed order, no atomics, any list length.
constexpr uint32_t kPiece = 8, kSpan = kLogitsThreads * kPiece;

struct BiasEntry { uint32_t column; float value; };

__global__ void __launch_bounds__(kLogitsThreads) logits_process_kernel(const LogitsArgs a) {
    __shared__ BiasEntry s_bias[kLogitsThreads];
    __shared__ uint32_t s_warp[kLogitsThreads / 32];
    const uint32_t row = blockIdx.y, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    pdl_trigger();
    pdl_wait();
    const mc_sm100_logits_config_t c = a.cfg[row];
    const uint16_t* in = a.in + (size_t)row * a.row_stride;
    uint16_t* out = a.out + (size_t)row * a.out_stride;
    // columns [first, first + 8) of this thread; those below 0 or beyond the row are not there
    const uint32_t head = (uint32_t)((reinterpret_cast<uintptr_t>(out) & 15u) >> 1);
    const int32_t first = (int32_t)(blockIdx.x * kSpan + tid * kPiece) - (int32_t)head;
    const int32_t lo = first < 0 ? 0 : first, hi = first + (int32_t)kPiece < (int32_t)a.vocab ? first + (int32_t)kPiece : (int32_t)a.vocab;
    const bool whole = hi - lo == (int32_t)kPiece;
    uint32_t raw[4] = {0u, 0u, 0u, 0u};
    if (whole && ((reinterpret_cast<uintptr_t>(in + first)) & 15u) == 0u) {
        const uint4 v = *reinterpret_cast<const uint4*>(in + first);
        raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
    } else {
#pragma unroll
        for (int e = 0; e < (int)kPiece; ++e)
            if (first + e >= lo && first + e < hi) raw[e >> 1] |= (uint32_t)in[first + e] << (16 * (e & 1));
    }
    const uint32_t words = (a.t.table_vocab + 31u) / 32u;
    const bool history = c.history_slot >= 0 && (uint32_t)c.history_slot < a.t.n_slots;
    const bool masked = c.mask_row >= 0 && (uint32_t)c.mask_row < a.t.n_masks;
    const uint64_t end64 = (uint64_t)c.bias_begin + c.bias_count;
    if (a.t.d_status != nullptr && blockIdx.x == 0u && tid == 0u &&
        ((c.history_slot >= 0 && !history) || (c.mask_row >= 0 && !masked) || (c.bias_count != 0u && end64 > a.t.n_bias)))
        *a.t.d_status = 1;
    // the eight bits of a table row that belong to columns lo .. hi - 1, bit e = column first + e
    auto bits_of = [&](const uint32_t* table_row) -> uint32_t {
        if (hi <= lo) return 0u;
        const uint32_t t0 = (uint32_t)a.index_base + (uint32_t)lo, t1 = (uint32_t)a.index_base + (uint32_t)hi - 1u;
        const uint32_t w0 = table_row[t0 >> 5], w1 = (t1 >> 5) != (t0 >> 5) ? table_row[t1 >> 5] : 0u;
        return (__funnelshift_r(w0, w1, t0 & 31u) & ((1u << (hi - lo)) - 1u)) << (lo - first);
    };
    const uint32_t seen = history ? bits_of(a.t.d_seen + (size_t)c.history_slot * words) : 0u;
    const uint32_t allowed = masked ? bits_of(a.t.d_mask + (size_t)c.mask_row * words) : 0xFFu;

    float bias[kPiece];
    uint32_t listed = 0u;
    const uint64_t end = end64 < a.t.n_bias ? end64 : a.t.n_bias;
    for (uint64_t j0 = c.bias_begin; j0 < end; j0 += kLogitsThreads) {               // the same for every thread
        const int32_t span0 = (int32_t)(blockIdx.x * kSpan) - (int32_t)head;
        uint32_t col = 0xFFFFFFFFu;
        float value = 0.f;
        if (j0 + tid < end) {
            const int64_t column = (int64_t)a.t.d_bias_token[j0 + tid] - a.index_base;
            if (column >= 0 && column < (int64_t)a.vocab && column >= span0 && column < (int64_t)span0 + kSpan) {
                col = (uint32_t)(column - span0);
                value = a.t.d_bias_value[j0 + tid];
            }
        }
        const uint32_t hits = __ballot_sync(0xFFFFFFFFu, col != 0xFFFFFFFFu);
        if (lane == 0) s_warp[warp] = __popc(hits);
        __syncthreads();
        uint32_t before = 0u, total = 0u;
#pragma unroll
        for (uint32_t w = 0; w < kLogitsThreads / 32; ++w) { const uint32_t n = s_warp[w]; before += w < warp ? n : 0u; total += n; }
        if (col != 0xFFFFFFFFu) s_bias[before + __popc(hits & ((1u << lane) - 1u))] = BiasEntry{col, value};
        __syncthreads();
        for (uint32_t k = 0; k < total; ++k) {
            const BiasEntry b = s_bias[k];
            if ((b.column / kPiece) == tid) {
#pragma unroll
                for (uint32_t e = 0; e < kPiece; ++e)
                    if ((b.column & (kPiece - 1u)) == e) { bias[e] = (listed >> e) & 1u ? __fadd_rn(bias[e], b.value) : __fadd_rn(0.f, b.value); listed |= 1u << e; }
            }
        }
        __syncthreads();
    }
    const bool repeat = c.rep_penalty != 1.f && c.rep_penalty != 0.f;
    const int32_t* counts = history ? a.t.d_counts + (size_t)c.history_slot * a.t.table_vocab + a.index_base : nullptr;
    uint32_t res[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < (int)kPiece; ++e) {
        float l = (e & 1) ? bf16hi(raw[e >> 1]) : bf16lo(raw[e >> 1]);
        if ((seen >> e) & 1u) {
            if (repeat) l = l > 0.f ? __fdiv_rn(l, c.rep_penalty) : __fmul_rn(l, c.rep_penalty);
            const int32_t n = counts[first + e];
            if (n > 0) l = __fsub_rn(__fsub_rn(l, __fmul_rn(c.freq_penalty, (float)n)), c.pres_penalty);
        }
        if ((listed >> e) & 1u) l = __fadd_rn(l, bias[e]);
        if (!((allowed >> e) & 1u)) l = -INFINITY;
        res[e >> 1] |= (uint32_t)f32_to_bf16_bits(l) << (16 * (e & 1));
    }
    if (in == out && res[0] == raw[0] && res[1] == raw[1] && res[2] == raw[2] && res[3] == raw[3]) return;   // in place, nothing to say
    if (whole) *reinterpret_cast<uint4*>(out + first) = make_uint4(res[0], res[1], res[2], res[3]);
    else {
#pragma unroll
        for (int e = 0; e < (int)kPiece; ++e)
            if (first + e >= lo && first + e < hi) out[first + e] = (uint16_t)(res[e >> 1] >> (16 * (e & 1)));
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

// Rebuild: a CTA owns `span` tokens of the vocabulary of one slot.  It counts in shared memory (bit 31: seen in the prompt)
// over the slot's tokens and writes each count and seen bit once: no clearing pass, no global atomics, one launch; the token
// list is read once per span (from L2 after the first).  Of several sequences that name a slot the first owns it and the
// others add to its counts.
constexpr uint32_t kHistThreads = 512;

__global__ void __launch_bounds__(kHistThreads) history_rebuild_kernel(const HistoryArgs a, uint32_t n_seqs, uint32_t span) {
    extern __shared__ uint32_t s_count[];
    __shared__ uint32_t s_same[kHistThreads / 32];
    pdl_trigger();
    pdl_wait();
    const uint32_t seq = blockIdx.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    uint32_t slot, lo, hi;
    if (!history_seq(a, seq, slot, lo, hi)) return;
    for (uint32_t i = tid; i < span; i += kHistThreads) s_count[i] = 0u;
    auto same_slot = [&](uint32_t other) {
        uint32_t s, l, h;
        return other < n_seqs && history_seq(a, other, s, l, h) && s == slot;
    };
    if (a.slots != nullptr) {
        bool taken = false;
        for (uint32_t j = tid; j < seq; j += kHistThreads) taken = taken || same_slot(j);
        if (__syncthreads_or(taken ? 1 : 0)) return;
    } else {
        __syncthreads();
    }
    const uint32_t t0 = blockIdx.y * span, t1 = min(a.vocab, t0 + span);
    auto add = [&](uint32_t which) {
        uint32_t s, l, h;
        (void)history_seq(a, which, s, l, h);
        const uint32_t n = h - l, prompt = a.prompt_len != nullptr ? a.prompt_len[which] : 0u;
        for (uint32_t k = tid; k < n; k += kHistThreads) {
            const uint32_t tok = (uint32_t)a.tokens[l + k];
            if (tok < t0 || tok >= t1) continue;
            if (k < prompt) atomicOr(s_count + (tok - t0), 0x80000000u);
            else atomicAdd(s_count + (tok - t0), 1u);
        }
    };
    add(seq);
    if (a.slots != nullptr) {
        for (uint32_t j0 = seq + 1u; j0 < n_seqs; j0 += kHistThreads) {
            const uint32_t hits = __ballot_sync(0xFFFFFFFFu, same_slot(j0 + tid));
            if (lane == 0) s_same[warp] = hits;
            __syncthreads();
            for (uint32_t w = 0; w < kHistThreads / 32u; ++w)
                for (uint32_t m = s_same[w]; m != 0u; m &= m - 1u) add(j0 + w * 32u + (uint32_t)__ffs((int)m) - 1u);
            __syncthreads();
        }
    }
    __syncthreads();
    const uint32_t words = (a.vocab + 31u) / 32u;
    for (uint32_t i = tid; t0 + (i & ~31u) < t1; i += kHistThreads) {              // whole warps stay together: span % 32 = 0
        const uint32_t c = t0 + i < t1 ? s_count[i] : 0u;
        if (t0 + i < t1) a.counts[(size_t)slot * a.vocab + t0 + i] = (int32_t)(c & 0x7FFFFFFFu);
        const uint32_t bits = __ballot_sync(0xFFFFFFFFu, c != 0u);
        if (lane == 0) a.seen[(size_t)slot * words + (t0 + i) / 32u] = bits;
    }
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

}  // namespace

}  // namespace mcl

using namespace mcl;

extern "C" {

mc_status_t mc_sm100_logits_process(const uint16_t* d_logits, uint16_t* d_out, uint32_t n_rows, uint32_t vocab, uint32_t row_stride,
                                    uint32_t out_stride, int32_t index_base, const mc_sm100_logits_config_t* d_cfg,
                                    const mc_sm100_logits_tables_t* tables, void* stream, int32_t pdl) {
    clear_error();
    const char* who = "mc_sm100_logits_process";
    if (d_logits == nullptr || d_out == nullptr || d_cfg == nullptr || tables == nullptr || n_rows == 0 || n_rows > 65535u || vocab == 0 ||
        vocab > 0x40000000u || row_stride < vocab || out_stride < vocab || index_base < 0 || (d_logits == d_out && row_stride != out_stride)) {
        set_error("%s: invalid args (rows=%u vocab=%u strides=%u,%u index_base=%d)", who, n_rows, vocab, row_stride, out_stride, index_base);
        return MC_E_INVALID_ARGUMENT;
    }
    const mc_sm100_logits_tables_t& t = *tables;
    if (t.struct_size != sizeof(mc_sm100_logits_tables_t) || t.reserved != 0u || t.table_vocab > 0x7FFFFFFFu ||
        (uint64_t)index_base + vocab > t.table_vocab || (t.n_slots != 0u && (t.d_counts == nullptr || t.d_seen == nullptr)) ||
        (t.n_masks != 0u && t.d_mask == nullptr) || (t.n_bias != 0u && (t.d_bias_token == nullptr || t.d_bias_value == nullptr))) {
        set_error("%s: invalid tables (struct_size=%u table_vocab=%u slots=%u masks=%u biases=%u) for columns %d..%llu", who, t.struct_size,
                  t.table_vocab, t.n_slots, t.n_masks, t.n_bias, index_base, (unsigned long long)((uint64_t)index_base + vocab));
        return MC_E_INVALID_ARGUMENT;
    }
    const LogitsArgs a{d_logits, d_out, vocab, row_stride, out_stride, index_base, d_cfg, t};
    (void)launch(logits_process_kernel, dim3((vocab + kPiece - 1u + kSpan - 1u) / kSpan, n_rows), dim3(kLogitsThreads), 0,
                 (cudaStream_t)stream, pdl != 0, a);
    MCL_CHECK_LAUNCH("logits_process");
    return MC_OK;
}

mc_status_t mc_sm100_token_history(int32_t* d_counts, uint32_t* d_seen, uint32_t n_slots, uint32_t table_vocab, const int32_t* d_tokens,
                                   uint32_t n_tokens, const uint32_t* d_offsets, const uint32_t* d_prompt_len, const int32_t* d_slots,
                                   uint32_t n_seqs, int32_t rebuild, int32_t* d_status, void* stream, int32_t pdl) {
    clear_error();
    if (d_counts == nullptr || d_seen == nullptr || n_slots == 0 || n_slots > 0x7FFFFFFFu || table_vocab == 0 || table_vocab > 0x40000000u ||
        (d_tokens == nullptr && n_tokens != 0u) || n_seqs == 0 || n_seqs > 0x7FFFFFFFu || (d_offsets == nullptr && n_tokens < n_seqs) ||
        (d_slots == nullptr && n_seqs > n_slots)) {
        set_error("mc_sm100_token_history: invalid args (slots=%u vocab=%u tokens=%u sequences=%u)", n_slots, table_vocab, n_tokens, n_seqs);
        return MC_E_INVALID_ARGUMENT;
    }
    const HistoryArgs a{d_counts, d_seen, n_slots, table_vocab, d_tokens, n_tokens, d_offsets, d_prompt_len, d_slots, d_status};
    if (rebuild != 0) {
        // Spans of 2048 to 16384 tokens: as many CTAs as two rounds of SMs, and no more (each reads the whole token list).
        const uint64_t spans = (2ull * (uint32_t)sm_count() + n_seqs - 1u) / n_seqs;
        uint64_t span = ((uint64_t)table_vocab + spans - 1u) / spans;
        span = span < 2048u ? 2048u : (span > 16384u ? 16384u : (span + 31u) & ~(uint64_t)31u);
        static SmemOptIn optin;
        const cudaError_t e = optin.ensure(history_rebuild_kernel, span * 4u);
        if (e != cudaSuccess) {
            set_error("mc_sm100_token_history: cannot raise shared memory to %u: %s", (uint32_t)span * 4u, cudaGetErrorString(e));
            return MC_E_CUDA;
        }
        (void)launch(history_rebuild_kernel, dim3(n_seqs, (uint32_t)((table_vocab + span - 1u) / span)), dim3(kHistThreads), (size_t)span * 4u,
                     (cudaStream_t)stream, pdl != 0, a, n_seqs, (uint32_t)span);
        MCL_CHECK_LAUNCH("history_rebuild");
        return MC_OK;
    }
    (void)launch(history_add_kernel, dim3(n_seqs, d_offsets != nullptr ? 8 : 1), dim3(kLogitsThreads), 0, (cudaStream_t)stream, pdl != 0, a);
    MCL_CHECK_LAUNCH("history_add");
    return MC_OK;
}

}  // extern "C"
