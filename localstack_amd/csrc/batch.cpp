// batch.cpp - C entries of the operators of a decode step of many sequences: attention over pages (lstk_attn_paged, _q8, lstk_attn_shared,
// _q8), the quantised cache (lstk_cache_q8_store, _load), lstk_sample and lstk_token_logprobs (include/lstk_qwen3.h) and
// lstk_moe_select (include/lstk_moe.h). They hold no state: the caller owns every buffer, the workspaces among them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "../../include/lstk_qwen3.h"
#include "batch.h"
#include "cache_q8.h"
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
constexpr float kLog2e = 1.44269504088896341f;

// Shapes of a paged attention call, checked, and its plan.
int paged_plan(bool q8, int n_seq, int n_head, int n_head_kv, int head_dim, int max_len, int window, int n_sink, lstk::PagedAttnParams &P,
               size_t &bytes) {
    P.in_q8 = q8;
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

// What a call of attention over pages has beyond its shapes: the sequences, their cache and the buffers.
int paged_inputs(const lstk_paged_seqs *seqs, const int32_t *d_cell_seq, const uint16_t *d_q, float scale, uint16_t *d_out, const void *d_work,
                 size_t work_bytes, size_t bytes, lstk::PagedAttnParams &P) {
    if (!seqs->d_len || !seqs->d_first || (!seqs->d_blocks && seqs->n_table > 0) || !d_q || !d_out) return bad("null argument");
    if (!aligned(d_q, 16) || !aligned(d_out, 16)) return bad("k, v, q and out must be 16-byte aligned");
    if (!d_cell_seq != !seqs->d_seq) return bad("d_cell_seq and d_seq go together");
    if (!aligned(seqs->d_len, 4) || !aligned(seqs->d_first, 4) || !aligned(seqs->d_blocks, 4) || !aligned(seqs->d_seq, 4) ||
        !aligned(d_cell_seq, 4))
        return bad("len, first, blocks, seq and cell_seq must be 4-byte aligned");
    if (bytes > 0 && (!d_work || !aligned(d_work, 16) || work_bytes < bytes))
        return bad("the workspace must be 16-byte aligned and hold " + std::to_string(bytes) + " bytes");
    P.q = d_q;
    P.len = seqs->d_len;
    P.first = seqs->d_first;
    P.blocks = seqs->d_blocks;
    P.n_table = seqs->n_table;
    P.cell_seq = d_cell_seq;
    P.seq = seqs->d_seq;
    P.scale = scale * kLog2e;
    P.out = d_out;
    return LSTK_OK;
}
int fp16_cache(const lstk_paged_cache *cache, bool used, const uint16_t *&k, const uint16_t *&v, int64_t &kv_size) {
    if (cache->kv_size < lstk::kPageCells || cache->kv_size % lstk::kPageCells || cache->kv_size > lstk::kPagedMaxCells)
        return bad("kv_size must be a positive multiple of 32, at most 2^27");
    if (used && (!cache->d_k || !cache->d_v)) return bad("null argument");
    if (used && (!aligned(cache->d_k, 16) || !aligned(cache->d_v, 16))) return bad("k, v, q and out must be 16-byte aligned");
    k = cache->d_k;
    v = cache->d_v;
    kv_size = cache->kv_size;
    return LSTK_OK;
}
int q8_cache(const lstk_q8_cache *cache, bool used) {
    if (cache->n_head_kv < 1 || cache->n_head_kv > kMostHeads) return bad("n_head_kv must be in [1, 65535]");
    if (!lstk::attn_supported(cache->head_dim)) return bad("head_dim must be 64, 128 or 256");
    if (cache->n_pages < 1 || cache->n_pages > lstk::kPagedMaxCells / lstk::kPageCells) return bad("n_pages must be in [1, 2^22]");
    if (used && !cache->d_pages) return bad("null argument");
    if (used && !aligned(cache->d_pages, 16)) return bad("the cache must be 16-byte aligned");
    return LSTK_OK;
}
hipError_t run_paged(const lstk::PagedAttnParams &P, hipStream_t st) {
    const hipError_t e = P.q8 ? lstk::launch_paged_attn_q8(P, st, nullptr) : lstk::launch_paged_attn(P, st, nullptr);
    return e == hipSuccess ? lstk::launch_paged_attn_join(P, st, nullptr) : e;
}

// A call over a prefix and the sequences' own cells. The workspace: the prefix's parts, then that of the own cells.
int prefix_plan(int n_seq, int n_head, int n_head_kv, int head_dim, int max_prefix, lstk::PrefixAttnParams &X, size_t &bytes) {
    if (max_prefix < 0) return bad("the prefix's max_len must be >= 0");
    X.n_seq = n_seq;
    X.n_head = n_head;
    X.n_kv = n_head_kv;
    X.hd = head_dim;
    X.max_len = max_prefix;
    bytes = (lstk::prefix_attn_plan(X) + 15) / 16 * 16;
    if (((int64_t) X.n_chunk * X.n_kv + 7) / 8 * 8 * X.n_rowblk > kMostGrid) return bad("too many sequences or heads for one launch");
    return LSTK_OK;
}
template <typename Cache>
int run_shared(const lstk_prefix *prefix, const Cache *cache, const lstk_paged_seqs *seqs, const uint16_t *d_q, int n_head, float scale,
               uint16_t *d_out, void *d_work, size_t work_bytes, lstk_stream_t stream) {
    constexpr bool q8 = std::is_same_v<Cache, lstk_q8_cache>;
    if (!prefix || !prefix->cache || !cache || !seqs) return bad("null argument");
    lstk::PagedAttnParams P{};
    lstk::PrefixAttnParams X{};
    size_t own = 0, pre = 0;
    int rc = paged_plan(q8, seqs->n_seq, n_head, cache->n_head_kv, cache->head_dim, seqs->max_len, 0, 0, P, own);
    if (rc == LSTK_OK) rc = prefix_plan(seqs->n_seq, n_head, cache->n_head_kv, cache->head_dim, prefix->max_len, X, pre);
    if (rc != LSTK_OK) return rc;
    if (prefix->cache->n_head_kv != cache->n_head_kv || prefix->cache->head_dim != cache->head_dim)
        return bad("the prefix's cache must have the heads of the sequences'");
    if (prefix->cache->d_cell_seq) return bad("the cells of a prefix have no owner: its d_cell_seq must be NULL");
    if (seqs->n_table < 0 || prefix->n_table < 0) return bad("n_table must be >= 0");
    if (!std::isfinite(scale)) return bad("scale must be finite");
    const bool used = P.n_seq > 0;
    if constexpr (q8) {
        rc = q8_cache(cache, used);
        P.q8 = cache->d_pages;
        P.kv_size = cache->n_pages * lstk::kPageCells;
    } else {
        rc = fp16_cache(cache, used, P.kc, P.vc, P.kv_size);
    }
    if (rc == LSTK_OK) rc = fp16_cache(prefix->cache, used && X.n_chunk > 0, X.kc, X.vc, X.kv_size);
    if (rc != LSTK_OK || !used) return rc;
    if (X.n_chunk > 0 && (!prefix->d_len || (!prefix->d_blocks && prefix->n_table > 0))) return bad("null argument");
    if (!aligned(prefix->d_len, 4) || !aligned(prefix->d_blocks, 4)) return bad("len, first, blocks, seq and cell_seq must be 4-byte aligned");
    if ((rc = paged_inputs(seqs, cache->d_cell_seq, d_q, scale, d_out, d_work, work_bytes, pre + own, P)) != LSTK_OK) return rc;
    X.q = d_q;
    X.len = prefix->d_len;
    X.blocks = prefix->d_blocks;
    X.n_table = prefix->n_table;
    X.scale = P.scale;
    X.part = static_cast<float *>(d_work);
    lstk::paged_attn_work(P, static_cast<uint8_t *>(d_work) + pre);
    P.pre = X.part;
    P.n_pre = X.n_chunk;
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e = lstk::launch_prefix_attn(X, st, nullptr);
    if (e == hipSuccess) e = run_paged(P, st);
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "shared attention launch");
}

int cache_rows(const lstk_q8_cache *cache, const void *d_k, const void *d_v, int type, int64_t ld_k, int64_t ld_v, const int32_t *d_cells,
               int n_rows, bool writes_rows, lstk::CacheRowsParams &P) {
    if (!cache) return bad("null argument");
    if (n_rows < 0 || n_rows > kMostTokens) return bad("n_rows must be in [0, 2^24]");
    const int rc = q8_cache(cache, n_rows > 0);
    if (rc != LSTK_OK) return rc;
    if (type != LSTK_TYPE_F16 && type != LSTK_TYPE_F32) return bad("rows must be of LSTK_TYPE_F16 or LSTK_TYPE_F32");
    const int64_t least = writes_rows && n_rows > 1 ? (int64_t) cache->n_head_kv * cache->head_dim : 0;
    if (ld_k < least || ld_v < least || ld_k % 8 || ld_v % 8) return bad("ld_k and ld_v must be multiples of 8, and hold a row where rows are written");
    if ((int64_t) ((n_rows + 38) / 32) * cache->n_head_kv > kMostGrid) return bad("too many rows for one launch");
    if (n_rows == 0) return LSTK_OK;
    if (!d_k || !d_v || !d_cells) return bad("null argument");
    if (!aligned(d_k, 16) || !aligned(d_v, 16) || !aligned(d_cells, 4)) return bad("k and v must be 16-byte aligned, cells 4-byte");
    P = {cache->d_pages, cache->n_pages * lstk::kPageCells, cache->n_head_kv, cache->head_dim, d_cells, n_rows, type == LSTK_TYPE_F32,
         d_k, d_v, ld_k, ld_v};
    return LSTK_OK;
}

}  // namespace

extern "C" {

size_t lstk_attn_paged_work_bytes(int n_seq, int n_head, int n_head_kv, int head_dim, int max_len, int window, int n_sink) {
    lstk::PagedAttnParams P{};
    size_t bytes = 0;
    return paged_plan(false, n_seq, n_head, n_head_kv, head_dim, max_len, window, n_sink, P, bytes) == LSTK_OK ? bytes : 0;
}

int lstk_attn_paged(const lstk_paged_cache *cache, const lstk_paged_seqs *seqs, const uint16_t *d_q, int n_head, int window,
                    int n_sink, float scale, uint16_t *d_out, void *d_work, size_t work_bytes, lstk_stream_t stream) {
    if (!cache || !seqs) return bad("null argument");
    lstk::PagedAttnParams P{};
    size_t bytes = 0;
    int rc = paged_plan(false, seqs->n_seq, n_head, cache->n_head_kv, cache->head_dim, seqs->max_len, window, n_sink, P, bytes);
    if (rc != LSTK_OK) return rc;
    if (seqs->n_table < 0) return bad("n_table must be >= 0");
    if (!std::isfinite(scale)) return bad("scale must be finite");
    rc = fp16_cache(cache, P.n_seq > 0, P.kc, P.vc, P.kv_size);
    if (rc != LSTK_OK || P.n_seq == 0) return rc;
    rc = paged_inputs(seqs, cache->d_cell_seq, d_q, scale, d_out, d_work, work_bytes, bytes, P);
    if (rc != LSTK_OK) return rc;
    lstk::paged_attn_work(P, d_work);
    const hipError_t e = run_paged(P, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "paged attention launch");
}

size_t lstk_attn_paged_q8_work_bytes(int n_seq, int n_head, int n_head_kv, int head_dim, int max_len, int window, int n_sink) {
    lstk::PagedAttnParams P{};
    size_t bytes = 0;
    return paged_plan(true, n_seq, n_head, n_head_kv, head_dim, max_len, window, n_sink, P, bytes) == LSTK_OK ? bytes : 0;
}

int lstk_attn_paged_q8(const lstk_q8_cache *cache, const lstk_paged_seqs *seqs, const uint16_t *d_q, int n_head, int window, int n_sink,
                       float scale, uint16_t *d_out, void *d_work, size_t work_bytes, lstk_stream_t stream) {
    if (!cache || !seqs) return bad("null argument");
    lstk::PagedAttnParams P{};
    size_t bytes = 0;
    int rc = paged_plan(true, seqs->n_seq, n_head, cache->n_head_kv, cache->head_dim, seqs->max_len, window, n_sink, P, bytes);
    if (rc != LSTK_OK) return rc;
    if (seqs->n_table < 0) return bad("n_table must be >= 0");
    if (!std::isfinite(scale)) return bad("scale must be finite");
    rc = q8_cache(cache, P.n_seq > 0);
    if (rc != LSTK_OK || P.n_seq == 0) return rc;
    rc = paged_inputs(seqs, cache->d_cell_seq, d_q, scale, d_out, d_work, work_bytes, bytes, P);
    if (rc != LSTK_OK) return rc;
    P.q8 = cache->d_pages;
    P.kv_size = cache->n_pages * lstk::kPageCells;
    lstk::paged_attn_work(P, d_work);
    const hipError_t e = run_paged(P, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "paged attention launch");
}

// What serves both kinds of caches.
size_t lstk_attn_shared_work_bytes(int n_seq, int n_head, int n_head_kv, int head_dim, int max_len, int max_prefix) {
    lstk::PagedAttnParams P{};
    lstk::PrefixAttnParams X{};
    size_t own = 0, own_q8 = 0, pre = 0;
    return paged_plan(false, n_seq, n_head, n_head_kv, head_dim, max_len, 0, 0, P, own) == LSTK_OK &&
                   paged_plan(true, n_seq, n_head, n_head_kv, head_dim, max_len, 0, 0, P, own_q8) == LSTK_OK &&
                   prefix_plan(n_seq, n_head, n_head_kv, head_dim, max_prefix, X, pre) == LSTK_OK
               ? pre + std::max(own, own_q8)
               : 0;
}

int lstk_attn_shared(const lstk_prefix *prefix, const lstk_paged_cache *cache, const lstk_paged_seqs *seqs, const uint16_t *d_q, int n_head,
                     float scale, uint16_t *d_out, void *d_work, size_t work_bytes, lstk_stream_t stream) {
    return run_shared(prefix, cache, seqs, d_q, n_head, scale, d_out, d_work, work_bytes, stream);
}

int lstk_attn_shared_q8(const lstk_prefix *prefix, const lstk_q8_cache *cache, const lstk_paged_seqs *seqs, const uint16_t *d_q, int n_head,
                        float scale, uint16_t *d_out, void *d_work, size_t work_bytes, lstk_stream_t stream) {
    return run_shared(prefix, cache, seqs, d_q, n_head, scale, d_out, d_work, work_bytes, stream);
}

int lstk_cache_q8_store(const lstk_q8_cache *cache, const void *d_k, const void *d_v, int type, int64_t ld_k, int64_t ld_v,
                        const int32_t *d_cells, int n_rows, lstk_stream_t stream) {
    lstk::CacheRowsParams P{};
    const int rc = cache_rows(cache, d_k, d_v, type, ld_k, ld_v, d_cells, n_rows, false, P);
    if (rc != LSTK_OK || n_rows == 0) return rc;
    const hipError_t e = lstk::launch_cache_store(P, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "cache store launch");
}

int lstk_cache_q8_load(const lstk_q8_cache *cache, void *d_k, void *d_v, int type, int64_t ld_k, int64_t ld_v, const int32_t *d_cells,
                       int n_rows, lstk_stream_t stream) {
    lstk::CacheRowsParams P{};
    const int rc = cache_rows(cache, d_k, d_v, type, ld_k, ld_v, d_cells, n_rows, true, P);
    if (rc != LSTK_OK || n_rows == 0) return rc;
    const hipError_t e = lstk::launch_cache_load(P, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "cache load launch");
}

size_t lstk_token_logprobs_work_bytes(int n_rows, int n_vocab, int n_top) {
    if (n_rows < 1 || n_vocab < 1 || n_vocab > lstk::kLogpMaxVocab || n_top < 0 || n_top > lstk::kLogpMaxTop) return 0;
    lstk::LogpParams P{};
    P.n_rows = n_rows;
    P.n_vocab = n_vocab;
    P.n_top = n_top;
    return lstk::logp_plan(P, nullptr);
}

int lstk_token_logprobs(const float *d_logits, int64_t ld_logits, int n_rows, int n_vocab, const int32_t *d_tokens, int n_top,
                        float *d_logprobs, float *d_entropy, int32_t *d_top_ids, float *d_top_logprobs, void *d_work, size_t work_bytes,
                        lstk_stream_t stream) {
    if (n_rows < 0) return bad("n_rows must be >= 0");
    if (n_vocab < 1 || n_vocab > lstk::kLogpMaxVocab) return bad("n_vocab must be in [1, 2^20 - 16]");
    if (n_top < 0 || n_top > lstk::kLogpMaxTop) return bad("n_top must be in [0, 32]");
    if (ld_logits < n_vocab) return bad("ld_logits must be at least n_vocab");
    if (n_rows == 0) return LSTK_OK;
    if (!d_logits || !d_tokens || !d_logprobs || (n_top > 0 && (!d_top_ids || !d_top_logprobs))) return bad("null argument");
    if (!aligned(d_logits, 4) || !aligned(d_tokens, 4) || !aligned(d_logprobs, 4) || !aligned(d_entropy, 4) || !aligned(d_top_ids, 4) ||
        !aligned(d_top_logprobs, 4))
        return bad("every array must be 4-byte aligned");
    lstk::LogpParams P{};
    P.n_rows = n_rows;
    P.n_vocab = n_vocab;
    P.n_top = n_top;
    const size_t bytes = lstk::logp_plan(P, d_work);
    if (bytes > 0 && (!d_work || !aligned(d_work, 16) || work_bytes < bytes))
        return bad("the workspace must be 16-byte aligned and hold " + std::to_string(bytes) + " bytes");
    if ((int64_t) n_rows * P.slices > kMostGrid) return bad("too many rows for one launch");
    P.logits = d_logits;
    P.ld = ld_logits;
    P.tokens = d_tokens;
    P.logp = d_logprobs;
    P.entropy = d_entropy;
    P.top_ids = d_top_ids;
    P.top_logp = d_top_logprobs;
    const hipError_t e = lstk::launch_logp(P, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? LSTK_OK : hip_fail(e, "log probability launch");
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
