// batch.h - launchers of the operators of a decode step of many sequences: attention of one new token per
// sequence over the paged cache (paged_attn.hip), sampling (sample.hip) and routing by a rule (select.hip).
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
};
// Fills n_rowblk and n_wg; returns the bytes of workspace (16-byte aligned) that calls of these shapes with this max_len or a
// smaller one take (0 where every task has a work-group), which paged_attn_work points at.
size_t paged_attn_plan(PagedAttnParams &P);
void paged_attn_work(PagedAttnParams &P, void *work);
hipError_t launch_paged_attn(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm);
hipError_t launch_paged_attn_join(const PagedAttnParams &P, hipStream_t st, const LaunchTiming *tm);

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
