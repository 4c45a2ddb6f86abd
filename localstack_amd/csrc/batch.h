// batch.h - launchers of the operators of a decode step of many sequences: attention of one new token per
// sequence over the paged cache (paged_attn.hip), sampling (sample.hip) and routing by a rule (select.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels.h"

namespace lstk {

constexpr int kPageCells = 32; // cells of a page: the cache's block (KvCache::block_size, src/kv_cache.h:27)

// Attention of one query token per sequence over one layer's cache in the cell layouts of forward.h. Logical cell i of
// sequence b is cell blocks[first[b] + i / 32] * 32 + i % 32; cells [0, len[b]) exist, and of those the last `window` and
// the first `n_sink` are visible (window <= 0: all). A page whose table entry or block number is out of range is not.
struct PagedAttnParams {
    const uint16_t *q; // [n_seq][n_head][hd] fp16
    const uint16_t *kc, *vc;
    const int32_t *len, *first, *blocks;
    const int32_t *cell_seq, *seq; // both or neither
    int64_t kv_size;
    int n_seq, n_head, n_kv, hd, n_table, max_len, window, n_sink;
    float scale; // of the scores, times log2(e)
    int chunk, n_chunk, n_rowblk; // pages per work-group, chunks of the longest sequence, 16-row blocks (paged_attn_plan)
    float *part;                  // [n_seq][n_head][n_chunk][hd + 4]: max, sum, 2 unused, unnormalised output
    uint16_t *out;                // [n_seq][n_head][hd] fp16
};
// Fills chunk, n_chunk and n_rowblk; returns the bytes of `part` that calls of these shapes with this max_len or a smaller
// one take (0 where every sequence takes one chunk).
size_t paged_attn_plan(PagedAttnParams &P);
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
    int slices, slice; // work-groups per row and 16-byte quads per slice (sample_plan)
    unsigned long long *best; // [n_rows][slices] largest (logit, lowest index) of a slice
    unsigned long long *mass; // [n_rows][kSampleBins]
    uint32_t *count;          // [n_rows][kSampleBins]
    uint32_t *n_list;         // [n_rows] entries of list
    uint32_t *n_done;         // [n_rows] work-groups of the last launch that are through
    int *list;                // [n_rows][n_vocab] indices of the values in the bins where a cut may fall
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
