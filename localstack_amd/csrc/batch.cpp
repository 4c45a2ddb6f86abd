// batch.cpp - C entries of the operators of a decode step of many sequences: lstk_attn_paged and lstk_sample
// (include/lstk_qwen3.h) and lstk_moe_select (include/lstk_moe.h). They hold no state: the caller owns every buffer, the
// workspaces among them.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/lstk_qwen3.h"
#include "batch.h"
#include "forward.h"
#include "internal.h"

namespace {

using lstk::set_error;

int hip_fail(hipError_t e, const char *what) { return set_error(LSTK_E_DEVICE, std::string(what) + ": " + hipGetErrorString(e)); }
int bad(const std::string &msg) { return set_error(LSTK_E_INVALID, msg); }
bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// A launch has fewer than 2^32 threads along x, in work-groups of up to 1024.
constexpr int64_t kMostGrid = (int64_t(1) << 22) - 1;
constexpr int kMostHeads = 65535;
constexpr int kMostTokens = 1 << 24;

// Shapes of a paged attention call, checked, and its plan.
int paged_plan(int n_seq, int n_head, int n_head_kv, int head_dim, int max_len, int window, int n_sink, lstk::PagedAttnParams &P,
               size_t &bytes) {
    if (n_seq < 0) return bad("n_seq must be >= 0");
    if (n_head < 1 || n_head_kv < 1 || n_head % n_head_kv) return bad("n_head must be a positive multiple of n_head_kv");
    if (!lstk::attn_supported(head_dim)) return bad("head_dim must be 64, 128 or 256");
    if (max_len < 0 || n_sink < 0) return bad("max_len and n_sink must be >= 0");
    P.n_seq = n_seq;
    P.n_head = n_head;
    P.n_kv = n_head_kv;
    P.hd = head_dim;
    P.max_len = max_len;
    P.window = window > 0 ? window : 0;
    P.n_sink = n_sink;
    const int row_blocks = (n_head / n_head_kv - 1) / 16 + 1;
    if (n_head > kMostHeads || (int64_t) n_seq * n_head_kv * row_blocks > kMostGrid)
        return bad("too many sequences or heads for one launch");
    bytes = lstk::paged_attn_plan(P);
    return LSTK_OK;
}

}  // namespace

extern "C" {

size_t lstk_attn_paged_work_bytes(int n_seq, int n_head, int n_head_kv, int head_dim, int max_len, int window, int n_sink) {
    lstk::PagedAttnParams P{};
    size_t bytes = 0;
    return paged_plan(n_seq, n_head, n_head_kv, head_dim, max_len, window, n_sink, P, bytes) == LSTK_OK ? bytes : 0;
}

int lstk_attn_paged(const lstk_paged_cache *cache, const lstk_paged_seqs *seqs, const uint16_t *d_q, int n_head, int window,
                    int n_sink, float scale, uint16_t *d_out, void *d_work, size_t work_bytes, lstk_stream_t stream) {
    if (!cache || !seqs) return bad("null argument");
    lstk::PagedAttnParams P{};
    size_t bytes = 0;
    const int rc = paged_plan(seqs->n_seq, n_head, cache->n_head_kv, cache->head_dim, seqs->max_len, window, n_sink, P, bytes);
    if (rc != LSTK_OK) return rc;
    if (cache->kv_size < lstk::kPageCells || cache->kv_size % lstk::kPageCells || cache->kv_size > lstk::kPagedMaxCells)
        return bad("kv_size must be a positive multiple of 32, at most 2^27");
    if (seqs->n_table < 0) return bad("n_table must be >= 0");
    if (!std::isfinite(scale)) return bad("scale must be finite");
    if (P.n_seq == 0) return LSTK_OK;
    if (!cache->d_k || !cache->d_v || !seqs->d_len || !seqs->d_first || (!seqs->d_blocks && seqs->n_table > 0) || !d_q || !d_out)
        return bad("null argument");
    if (!aligned(cache->d_k, 16) || !aligned(cache->d_v, 16) || !aligned(d_q, 16) || !aligned(d_out, 16))
        return bad("k, v, q and out must be 16-byte aligned");
    if (!cache->d_cell_seq != !seqs->d_seq) return bad("d_cell_seq and d_seq go together");
    if (!aligned(seqs->d_len, 4) || !aligned(seqs->d_first, 4) || !aligned(seqs->d_blocks, 4) || !aligned(seqs->d_seq, 4) ||
        !aligned(cache->d_cell_seq, 4))
        return bad("len, first, blocks, seq and cell_seq must be 4-byte aligned");
    if (bytes > 0 && (!d_work || !aligned(d_work, 16) || work_bytes < bytes))
        return bad("the workspace must be 16-byte aligned and hold " + std::to_string(bytes) + " bytes");
    P.q = d_q;
    P.kc = cache->d_k;
    P.vc = cache->d_v;
    P.kv_size = cache->kv_size;
    P.len = seqs->d_len;
    P.first = seqs->d_first;
    P.blocks = seqs->d_blocks;
    P.n_table = seqs->n_table;
    P.cell_seq = cache->d_cell_seq;
    P.seq = seqs->d_seq;
    P.scale = scale * 1.44269504088896341f;
    lstk::paged_attn_work(P, d_work);
    P.out = d_out;
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e = lstk::launch_paged_attn(P, st, nullptr);
    if (e == hipSuccess) e = lstk::launch_paged_attn_join(P, st, nullptr);
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "paged attention launch");
}

size_t lstk_sample_work_bytes(int n_rows, int n_vocab) {
    if (n_rows < 1 || n_vocab < 1 || n_vocab >= lstk::kSampleMaxVocab) return 0;
    lstk::SampleParams P{};
    P.n_rows = n_rows;
    P.n_vocab = n_vocab;
    return lstk::sample_plan(P, nullptr);
}

int lstk_sample(const float *d_logits, int64_t ld_logits, int n_rows, int n_vocab, const lstk_sampling *how, const float *d_u,
                int32_t *d_tokens, float *d_probs, void *d_work, size_t work_bytes, lstk_stream_t stream) {
    if (n_rows < 0) return bad("n_rows must be >= 0");
    if (n_vocab < 1 || n_vocab >= lstk::kSampleMaxVocab) return bad("n_vocab must be in [1, 2^20)");
    if (ld_logits < n_vocab) return bad("ld_logits must be at least n_vocab");
    if (n_rows == 0) return LSTK_OK;
    if (!d_logits || !how || !d_u || !d_tokens) return bad("null argument");
    if (!aligned(d_logits, 4) || !aligned(how->d_temperature, 4) || !aligned(how->d_top_k, 4) || !aligned(how->d_top_p, 4) ||
        !aligned(how->d_min_p, 4) || !aligned(d_u, 4) || !aligned(d_tokens, 4) || !aligned(d_probs, 4))
        return bad("every array must be 4-byte aligned");
    lstk::SampleParams P{};
    P.n_rows = n_rows;
    P.n_vocab = n_vocab;
    const size_t bytes = lstk::sample_plan(P, d_work);
    if (!d_work || !aligned(d_work, 16) || work_bytes < bytes)
        return bad("the workspace must be 16-byte aligned and hold " + std::to_string(bytes) + " bytes");
    if ((int64_t) n_rows * P.slices > kMostGrid) return bad("too many rows for one launch");
    P.logits = d_logits;
    P.ld = ld_logits;
    P.temperature = how->d_temperature;
    P.top_k = how->d_top_k;
    P.top_p = how->d_top_p;
    P.min_p = how->d_min_p;
    P.u = d_u;
    P.tokens = d_tokens;
    P.probs = d_probs;
    const hipError_t e = lstk::launch_sample(P, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "sample launch");
}

int lstk_moe_select(const lstk_router_rule *rule, const float *d_logits, int64_t ld_logits, const float *d_bias, int n_tokens,
                    int n_expert, int n_expert_used, int32_t *d_ids, float *d_weights, lstk_stream_t stream) {
    const int rc = lstk::check_rule(rule, n_expert, n_expert_used);
    if (rc != LSTK_OK) return rc;
    if (n_tokens < 0 || n_tokens > kMostTokens) return bad("n_tokens must be in [0, 2^24]");
    if (ld_logits < n_expert) return bad("ld_logits must be at least n_expert");
    if (n_tokens == 0) return LSTK_OK;
    if (!d_logits || !d_ids || !d_weights) return bad("null argument");
    if (!aligned(d_logits, 4) || !aligned(d_bias, 4) || !aligned(d_ids, 4) || !aligned(d_weights, 4))
        return bad("every array must be 4-byte aligned");
    const hipError_t e = lstk::launch_select(lstk::select_params(*rule, d_logits, ld_logits, d_bias, n_tokens, n_expert,
                                                                 n_expert_used, d_ids, d_weights),
                                             static_cast<hipStream_t>(stream), nullptr);
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "select launch");
}

}  // extern "C"

namespace lstk {

int check_rule(const lstk_router_rule *rule, int n_expert, int n_expert_used) {
    if (!rule) return bad("null rule");
    if (n_expert < 1 || n_expert > 256) return bad("n_expert must be in [1, 256]");
    if (n_expert_used < 1 || n_expert_used > n_expert || n_expert_used > 64) return bad("n_expert_used must be in [1, min(n_expert, 64)]");
    if (rule->score != LSTK_SCORE_SOFTMAX && rule->score != LSTK_SCORE_SIGMOID) return bad("unknown score function");
    if (rule->n_group < 1 || n_expert % rule->n_group) return bad("n_group must divide n_expert");
    if (rule->n_group_used < 1 || rule->n_group_used > rule->n_group) return bad("n_group_used must be in [1, n_group]");
    const int per = n_expert / rule->n_group;
    if (rule->group_top < 1 || rule->group_top > 2 || rule->group_top > per) return bad("group_top must be 1 or 2 and at most a group's experts");
    if ((int64_t) rule->n_group_used * per < n_expert_used) return bad("the groups kept hold fewer than n_expert_used experts");
    if (!std::isfinite(rule->scale)) return bad("scale must be finite");
    return LSTK_OK;
}

SelectParams select_params(const lstk_router_rule &rule, const float *logits, int64_t ld, const float *bias, int T, int E, int k,
                           int32_t *ids, float *weights) {
    return {logits, ld, bias, T, E, k, rule.score == LSTK_SCORE_SIGMOID, rule.n_group, rule.n_group_used, rule.group_top,
            rule.renorm != 0, rule.scale, ids, weights};
}

}  // namespace lstk
