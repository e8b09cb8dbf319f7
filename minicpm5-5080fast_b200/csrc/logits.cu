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

// One token per thread.
__global__ void __launch_bounds__(kLogitsThreads) logits_process_kernel(const LogitsArgs a) {
    pdl_trigger();
    pdl_wait();
    const uint32_t row = blockIdx.y, i = blockIdx.x * kLogitsThreads + threadIdx.x;
    const mc_sm100_logits_config_t c = a.cfg[row];
    const uint32_t words = (a.t.table_vocab + 31u) / 32u;
    const bool bad_slot = c.history_slot >= 0 && (uint32_t)c.history_slot >= a.t.n_slots;
    const bool bad_mask = c.mask_row >= 0 && (uint32_t)c.mask_row >= a.t.n_masks;
    const uint64_t end = (uint64_t)c.bias_begin + c.bias_count;
    if (a.t.d_status != nullptr && i == 0u && (bad_slot || bad_mask || (c.bias_count != 0u && end > a.t.n_bias))) *a.t.d_status = 1;
    if (i >= a.vocab) return;
    const uint32_t tok = (uint32_t)a.index_base + i;
    float l = __uint_as_float((uint32_t)a.in[(size_t)row * a.row_stride + i] << 16);
    if (c.history_slot >= 0 && !bad_slot) {
        if ((a.t.d_seen[(size_t)c.history_slot * words + tok / 32u] >> (tok & 31u)) & 1u) {
            if (c.rep_penalty != 1.f && c.rep_penalty != 0.f) l = l > 0.f ? __fdiv_rn(l, c.rep_penalty) : __fmul_rn(l, c.rep_penalty);
            const int32_t n = a.t.d_counts[(size_t)c.history_slot * a.t.table_vocab + tok];
            if (n > 0) l = __fsub_rn(__fsub_rn(l, __fmul_rn(c.freq_penalty, (float)n)), c.pres_penalty);
        }
    }
    float bias = 0.f;
    bool listed = false;
    for (uint64_t j = c.bias_begin; j < end && j < a.t.n_bias; ++j)
        if ((uint32_t)a.t.d_bias_token[j] == tok) { bias += a.t.d_bias_value[j]; listed = true; }
    if (listed) l = __fadd_rn(l, bias);
    if (c.mask_row >= 0 && !bad_mask && !((a.t.d_mask[(size_t)c.mask_row * words + tok / 32u] >> (tok & 31u)) & 1u)) l = -INFINITY;
    a.out[(size_t)row * a.out_stride + i] = f32_to_bf16_bits(l);
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

// Every slot that a sequence names starts from nothing.
__global__ void __launch_bounds__(kLogitsThreads) history_clear_kernel(const HistoryArgs a) {
    pdl_trigger();
    pdl_wait();
    uint32_t slot, lo, hi;
    if (!history_seq(a, blockIdx.x, slot, lo, hi)) return;
    const uint32_t words = (a.vocab + 31u) / 32u, first = blockIdx.y * kLogitsThreads + threadIdx.x, step = gridDim.y * kLogitsThreads;
    for (uint32_t i = first; i < a.vocab; i += step) a.counts[(size_t)slot * a.vocab + i] = 0;
    for (uint32_t i = first; i < words; i += step) a.seen[(size_t)slot * words + i] = 0u;
}

// Integer atomics: the order does not show in the result.
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
        vocab > 0x7FFFFFFFu || row_stride < vocab || out_stride < vocab || index_base < 0 || (d_logits == d_out && row_stride != out_stride)) {
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
    (void)launch(logits_process_kernel, dim3((vocab + kLogitsThreads - 1u) / kLogitsThreads, n_rows), dim3(kLogitsThreads), 0,
                 (cudaStream_t)stream, pdl != 0, a);
    MCL_CHECK_LAUNCH("logits_process");
    return MC_OK;
}

mc_status_t mc_sm100_token_history(int32_t* d_counts, uint32_t* d_seen, uint32_t n_slots, uint32_t table_vocab, const int32_t* d_tokens,
                                   uint32_t n_tokens, const uint32_t* d_offsets, const uint32_t* d_prompt_len, const int32_t* d_slots,
                                   uint32_t n_seqs, int32_t rebuild, int32_t* d_status, void* stream, int32_t pdl) {
    clear_error();
    if (d_counts == nullptr || d_seen == nullptr || n_slots == 0 || n_slots > 0x7FFFFFFFu || table_vocab == 0 || table_vocab > 0x7FFFFFFFu ||
        (d_tokens == nullptr && n_tokens != 0u) || n_seqs == 0 || n_seqs > 0x7FFFFFFFu || (d_offsets == nullptr && n_tokens < n_seqs) ||
        (d_slots == nullptr && n_seqs > n_slots)) {
        set_error("mc_sm100_token_history: invalid args (slots=%u vocab=%u tokens=%u sequences=%u)", n_slots, table_vocab, n_tokens, n_seqs);
        return MC_E_INVALID_ARGUMENT;
    }
    const HistoryArgs a{d_counts, d_seen, n_slots, table_vocab, d_tokens, n_tokens, d_offsets, d_prompt_len, d_slots, d_status};
    if (rebuild != 0) {
        (void)launch(history_clear_kernel, dim3(n_seqs, 16), dim3(kLogitsThreads), 0, (cudaStream_t)stream, pdl != 0, a);
        MCL_CHECK_LAUNCH("history_clear");
    }
    (void)launch(history_add_kernel, dim3(n_seqs, d_offsets != nullptr ? 8 : 1), dim3(kLogitsThreads), 0, (cudaStream_t)stream, pdl != 0, a);
    MCL_CHECK_LAUNCH("history_add");
    return MC_OK;
}

}  // extern "C"
