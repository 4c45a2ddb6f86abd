// batch.h - launchers of the operators of a decode step of many sequences: attention of one new token per sequence over the paged
// cache in fp16 (paged_attn.hip) or 8 bits (paged_attn_q8.hip) and over a prefix that they share (prefix_attn.hip), rows into and out of
// the 8-bit cache (cache_q8.hip), log probabilities (logp.hip), sampling (sample.hip) and routing by a rule (select.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels.h"

namespace lstk {

constexpr int64_t kPagedMaxCells = int64_t(1) << 27; // of a cache: the attention kernel's 32-bit offsets
constexpr int kPageCells = 32; // cells of a page: the cache's block (KvCache::block_size, src/kv_cache.h:27)

// Attention of one query token per sequence over one layer's cache in the cell layouts of forward.h. Logical cell i of
// sequence b is cell blocks[first[b] + i / 32] * 32 + i % 32; cells [0, len[b]) exist, and of those the last `window` and
// the first `n_sink` are visible (window <= 0: all). A page whose table entry or block number is out of range is not.
struct PagedAttnSplit { // the work-group that began a task, and how many others went on with it
    int wg, more;
};
struct PagedAttnParams {
    const uint16_t *q; // [n_seq][n_head][hd] fp16
    const uint16_t *kc, *vc;
    const int32_t *len, *first, *blocks;
    const int32_t *cell_seq, *seq; // both or neither
    int64_t kv_size;
    int n_seq, n_head, n_kv, hd, n_table, max_len, window, n_sink;
    float scale; // of the scores, times log2(e)
    int n_rowblk, n_wg;    // blocks of 16 query heads per KV head; work-groups of equal shares, 0: one per task (paged_attn_plan)
    PagedAttnSplit *split; // [n_seq][n_kv * n_rowblk], a task each
    float *part;           // [n_wg][2][min(16, heads per KV head)][hd + 4]: max, sum, 2 unused, unnormalised output of a part of a task
    uint16_t *out;         // [n_seq][n_head][hd] fp16
    bool in_q8 = false;           // the cache is a quantised one (set before paged_attn_plan):
    const uint8_t *q8 = nullptr;  // its records (cache_q8.h) in place of kc and vc, kv_size / 32 pages
    float *pre = nullptr;         // [n_pre + 1][n_seq][n_head][hd + 4]: what parts of a prefix left, in the form of `part`, and room
    int n_pre = 0;
};
// Fills n_rowblk and n_wg; returns the bytes of workspace (16-byte aligned) that calls of these shapes with this max_len or a
// smaller one take (0 where every task has a work-group), which paged_attn_work points at.
size_t paged_attn_plan(PagedAttnParams &P);
void paged_attn_work(PagedAttnParams &P, void *work);
hipError_t launch_paged_attn(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm);
hipError_t launch_paged_attn_q8(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm);
hipError_t launch_paged_attn_join(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm);

// Attention of the query tokens of all sequences over one list of pages that they share: what each of n_chunk shares of the list
// leaves, [n_chunk][n_seq * n_head][hd + 4] (max, sum, 2 unused, unnormalised output), for PagedAttnParams::pre.
struct PrefixAttnParams {
    const uint16_t *q; // [n_seq][n_head][hd] fp16
    const uint16_t *kc, *vc;
    const int32_t *len, *blocks; // len: one number, cells of the prefix
    int64_t kv_size;
    int n_seq, n_head, n_kv, hd, n_table, max_len;
    float scale; // of the scores, times log2(e)
    int n_chunk, n_rowblk; // prefix_attn_plan
    bool shared;           // the wavefronts of a work-group share pages; otherwise each takes its own
    float *part;
};
// Fills n_chunk, n_rowblk and shared; returns the bytes of `part` with room for one more (0: no prefix).
size_t prefix_attn_plan(PrefixAttnParams &P);
hipError_t launch_prefix_attn(const PrefixAttnParams &P, hipStream_t st, const LaunchTiming *tm);

// Rows into and out of a quantised cache (cache_q8.hip).
struct CacheRowsParams {
    uint8_t *cache;
    int64_t n_cells; // of the cache
    int n_kv, hd;
    const int32_t *cells; // [n] cell of each row; one outside the cache is left alone (read: zeros)
    int n;
    bool f32;        // rows are f32, otherwise fp16
    const void *k, *v; // [n][n_kv][hd], rows ld_k and ld_v values apart; written to when reading back
    int64_t ld_k, ld_v;
};
hipError_t launch_cache_store(const CacheRowsParams &P, hipStream_t st);
hipError_t launch_cache_load(const CacheRowsParams &P, hipStream_t st);

// Log probabilities of one token per row of logits, entropy and the largest values.
constexpr int kLogpMaxTop = 32;
constexpr int kLogpMaxVocab = (1 << 20) - 16; // 64 slices of what a work-group holds
struct LogpParams {
    const float *logits;
    int64_t ld;
    int n_rows, n_vocab, n_top;
    const int32_t *tokens;
    float *logp, *entropy; // entropy may be null
    int32_t *top_ids;      // [n_rows][n_top]
    float *top_logp;
    int slices, slice;     // work-groups per row and 16-byte quads per slice (logp_plan)
    float *sums;           // [n_rows][slices][4]: max, values alike it, sum of e^(x - max) of the others, sum of (x - max) e^(x - max)
    unsigned long long *best; // [n_rows][slices][n_top] (value, lowest index), largest first
};
size_t logp_plan(LogpParams &P, void *work);
hipError_t launch_logp(const LogpParams &P, hipStream_t st);

// Sampling of one token per row of logits.
constexpr int kSampleBins = 2048;
constexpr int kSampleMaxVocab = 1 << 20;
struct SampleParams {
    const float *logits;
    int64_t ld;
    int n_rows, n_vocab;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *u;
    int32_t *tokens;
    float *probs;
    bool by_row;       // one work-group per row, one launch (sample_plan)
    int slices, slice; // work-groups per row and 16-byte quads per slice
    unsigned long long *best; // [n_rows][slices] largest (logit, lowest index) of a slice
    unsigned long long *mass; // [n_rows][kSampleBins]
    uint32_t *count;          // [n_rows][kSampleBins]
    uint32_t *n_list;         // [n_rows] entries of list
    uint32_t *n_done;         // [n_rows] work-groups of the last launch that are through
    unsigned long long *list; // [n_rows][n_vocab] (logit, index) of the values in the bins where a cut may fall
};
// Fills slices and slice, and the workspace pointers from `work`; returns the workspace's bytes.
size_t sample_plan(SampleParams &P, void *work);
hipError_t launch_sample(const SampleParams &P, hipStream_t st);

// Routing by a rule from logits.
struct SelectParams {
    const float *logits;
    int64_t ld;
    const float *bias;
    int T, E, k;
    int sigmoid, n_group, n_group_used, group_top, renorm;
    float scale;
    int32_t *ids;
    float *weights;
};
hipError_t launch_select(const SelectParams &P, hipStream_t st, const LaunchTiming *tm);

}  // namespace lstk
