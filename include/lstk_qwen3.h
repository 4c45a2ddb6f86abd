/* lstk_qwen3.h - C ABI of the Qwen3-MoE forward pass that surrounds the MoE path on MI355X.
 *
 * The MoE block (include/lstk_moe.h) needs the rest of the model around it to produce logits. This
 * is that rest, on the same device and stream:
 *   qwen3_build_graph()   src/qwen3.cpp:223-259 (embedding, per-layer attention + MoE, final norm,
 *                         output head; the last layer's FFN runs on the output row only)
 *   attn_block()          src/qwen3.cpp:128-171 (RMSNorm, Q/K/V, QK-norm, NEOX RoPE, KV set_rows,
 *                         attention with fp32 accumulation over fp16 K/V, o-proj, residual)
 *   Engine::decode/step   src/engine.cpp:250-278 (chunks of n_batch tokens, logits of the last token)
 *   Engine::step_resident / step_streaming  src/engine.cpp:282-341 (router trace; streaming pools
 *                         acquire the experts each layer selected before running them)
 *   KvCache               src/kv_cache.cpp:59-150 (block table per sequence, cell_seq / cell_pos,
 *                         visibility = same sequence and cell_pos <= token position)
 * Dense (non-MoE) FFNs and Qwen2's Q/K/V biases are not part of this path.
 *
 * Conventions are those of lstk_moe.h: 0 or a negative LSTK_E_* code, lstk_last_error() for the
 * message, caller-owned device pointers and stream, one host thread and one stream per model.
 * Weight layouts are ggml's: an F16 matrix of ggml shape [n_in, n_out] is n_out rows of n_in
 * contiguous fp16 values.
 */
#ifndef LSTK_QWEN3_H
#define LSTK_QWEN3_H

#include "lstk_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct lstk_model lstk_model;

/* Qwen3HParams (src/qwen3.h:22-46), the fields the MoE forward pass reads. */
typedef struct lstk_qwen3_hparams {
    int32_t n_layer;
    int32_t n_embd;
    int32_t n_head;
    int32_t n_head_kv;
    int32_t head_dim;
    int32_t n_vocab;
    int32_t n_expert;
    int32_t n_expert_used;
    int32_t n_ff_exp;
    int32_t n_ctx_train; /* carried for RoPE; inert without context extension */
    float rms_eps;
    float rope_freq_base;
} lstk_qwen3_hparams;

/* One layer's dense tensors on the device (Qwen3Layer, src/qwen3.h:49-73). Norm weights are f32;
 * q_norm / k_norm may be NULL (no QK-norm). The experts live in the lstk_pool passed at creation. */
typedef struct lstk_qwen3_layer {
    const float *attn_norm;  /* [n_embd] */
    const uint16_t *wq;      /* F16 [n_head * head_dim][n_embd] */
    const uint16_t *wk;      /* F16 [n_head_kv * head_dim][n_embd] */
    const uint16_t *wv;      /* F16 [n_head_kv * head_dim][n_embd]; when wk starts where wq ends and wv
                                where wk ends (one [q | k | v] block), multi-token steps take one
                                library product for all three instead of three */
    const uint16_t *wo;      /* F16 [n_embd][n_head * head_dim] */
    const float *q_norm;     /* [head_dim] or NULL */
    const float *k_norm;     /* [head_dim] or NULL */
    const float *ffn_norm;   /* [n_embd] */
    const void *gate_inp;    /* router, [n_expert][n_embd] of gate_inp_type */
    int32_t gate_inp_type;   /* LSTK_TYPE_F16 or LSTK_TYPE_F32 */
} lstk_qwen3_layer;

/* Model-wide tensors (Qwen3Weights, src/qwen3.h:75-82). output == NULL ties the head to tok_embd,
 * as the reference's loader does when the GGUF has no output.weight (src/qwen3.cpp:55-57). */
typedef struct lstk_qwen3_weights {
    const uint16_t *tok_embd;    /* F16 [n_vocab][n_embd] */
    const float *output_norm;    /* [n_embd] */
    const uint16_t *output;      /* F16 [n_vocab][n_embd] or NULL */
    const lstk_qwen3_layer *layers; /* n_layer entries, copied at creation */
} lstk_qwen3_weights;

/* Creates the forward pass over `pool` (whose dims must match hp) with a KV cache of kv_size cells
 * (a multiple of 256, like the reference's n_ctx) and steps of at most n_batch tokens
 * (EngineParams::n_batch, at most the pool's n_batch). head_dim must be 64, 128 or 256;
 * n_embd and n_head * head_dim multiples of 8 and at most 8192. The KV cache (fp16,
 * 2 * n_layer * kv_size * n_head_kv * head_dim * 2 bytes) and the step scratch are allocated here, on
 * the current device. The pool is not owned and must outlive the model. */
int lstk_model_create(const lstk_qwen3_hparams *hp, const lstk_qwen3_weights *w, lstk_pool *pool, uint32_t kv_size,
                      uint32_t n_batch, lstk_model **out);
void lstk_model_destroy(lstk_model *model);

/* Engine::decode (src/engine.cpp:250-260) for one sequence: appends `n_tokens` host token ids to
 * sequence `seq` in steps of at most n_batch tokens and writes the logits of the last token,
 * [n_vocab] f32, to the device pointer d_logits. When d_trace is not NULL it receives the router's
 * expert ids of every layer for the last step, [n_layer][n_step_tokens][n_expert_used] int32, where the
 * last layer has only its output row (the others are -1), like the reference's trace
 * (src/engine.cpp:299-316). Token ids out of [0, n_vocab) are rejected before anything runs.
 * Fails with LSTK_E_EXHAUSTED when the KV cache has no room ("KV cache is full"). */
int lstk_model_decode(lstk_model *model, int32_t seq, const int32_t *tokens, int n_tokens, float *d_logits,
                      int32_t *d_trace, lstk_stream_t stream);

/* lstk_model_decode in two halves, for callers that replay a step as a HIP graph.
 * prepare: Engine::make_step_inputs (src/engine.cpp:200-243) - reserves the KV cells of n_tokens
 *   (<= n_batch) host tokens of `seq`, queues their upload to the model's input buffer on `stream` and
 *   returns the number of attended cells in *n_cells.
 * forward: the step's kernels over those inputs, writing the last token's logits (and the trace, as
 *   lstk_model_decode). With a resident pool it makes no host synchronisation and no allocation, so it
 *   may be captured; a captured forward replays correctly after each prepare of the same seq,
 *   n_tokens and n_cells (n_cells changes only when the sequence crosses a multiple of 256 cells),
 *   wherever the new cells lie: while the stream is capturing, attention covers cells [0, n_cells)
 *   (an eager forward starts at the sequence's lowest cache block instead).
 *   Where the step last prepared is a batch step (below) it is refused, unless it is being captured.
 *   With a streaming pool it synchronises the stream once per layer (the router's ids go to the host),
 *   unless the pool was created with LSTK_POOL_DEVICE_LRU: then the experts are acquired on the device
 *   (lstk_pool_acquire_device), nothing waits on the host and the forward may be captured too. */
int lstk_model_prepare(lstk_model *model, int32_t seq, const int32_t *tokens, int n_tokens, int32_t *n_cells,
                       lstk_stream_t stream);
int lstk_model_forward(lstk_model *model, int32_t seq, int n_tokens, int32_t n_cells, float *d_logits,
                       int32_t *d_trace, lstk_stream_t stream);

/* One new token for each of n_seq distinct sequences in one step (no counterpart in the reference, whose steps take one
 * sequence): appends tokens[i] to sequence seqs[i] and writes the logits of every row, [n_seq][n_vocab] f32, to d_logits.
 * 1 <= n_seq <= n_batch. With window > 0 each token attends its sequence's last `window` cells and first n_sink cells, else
 * all of them (lstk_attn_paged); prompts run through lstk_model_decode attend everything. d_trace, when not NULL, receives the
 * router's ids [n_layer][n_seq][n_expert_used]; a trace file (lstk_model_set_trace) gets the step like any other.
 * Nothing is appended when the arguments are rejected or the cache has no room for all of them. The cache may have at most
 * 2^27 cells. */
int lstk_model_decode_batch(lstk_model *model, int n_seq, const int32_t *seqs, const int32_t *tokens, int window, int n_sink,
                            float *d_logits, int32_t *d_trace, lstk_stream_t stream);
/* The same in two halves, like lstk_model_prepare / lstk_model_forward. prepare_batch returns the longest sequence's cells in
 * *max_len. forward_batch takes the step last prepared (n_seq as there) and any max_len that holds its sequences; captured,
 * it replays correctly after each later prepare_batch of n_seq sequences, whichever they are, none longer than max_len. */
int lstk_model_prepare_batch(lstk_model *model, int n_seq, const int32_t *seqs, const int32_t *tokens, int32_t *max_len,
                             lstk_stream_t stream);
int lstk_model_forward_batch(lstk_model *model, int n_seq, int32_t max_len, int window, int n_sink, float *d_logits,
                             int32_t *d_trace, lstk_stream_t stream);

/* Attention of one new token per sequence over one layer's paged cache, on caller-owned device memory (the model's batch
 * step runs it on its own cache):
 *   out[b][h] = sum_i softmax_i(scale q[b][h] . k[i][h / (n_head / n_head_kv)]) v[i][..]   over the visible cells i of row b
 * K is [n_head_kv][head_dim / 4][kv_size][4] fp16 (4 dims of a cell together, cells side by side), V
 * [n_head_kv][kv_size / 4][head_dim][4] (4 cells of a dim together); head_dim 64, 128 or 256, kv_size a multiple of 32, at most 2^27.
 * Pages are runs of 32 cells: logical cell i of row b is cell d_blocks[d_first[b] + i / 32] * 32 + i % 32, 0 <= i < d_len[b];
 * rows may share pages. Visible are the cells i < min(d_len[b], max_len), of them with window > 0 only the last `window` and
 * the first n_sink (counted in cells the row holds). A page whose table index (outside [0, n_table)) or block number (outside the cache) is out of range is
 * not visible; with d_cell_seq [kv_size] and d_seq [n_seq] given (both or neither), nor is a cell whose d_cell_seq entry is
 * not d_seq[b]. What the cache holds in cells that are not visible is never used, whatever it is; a row with no visible cell
 * gets zeros. A NaN or an infinity in a visible cell can make its head's output NaN. Sums are fp32; a weight enters them as two fp16
 * parts, good to 2^-22 (to 2^-40 of the largest where it is below 2^-18 of it). */
typedef struct lstk_paged_cache {
    const uint16_t *d_k, *d_v;
    int64_t kv_size;
    int32_t n_head_kv, head_dim;
    const int32_t *d_cell_seq; /* or NULL */
} lstk_paged_cache;
typedef struct lstk_paged_seqs {
    int32_t n_seq;
    int32_t max_len;         /* bound of the lengths: sizes the launch and the workspace */
    const int32_t *d_len;    /* [n_seq] */
    const int32_t *d_first;  /* [n_seq] index of a row's first page in d_blocks */
    const int32_t *d_blocks; /* [n_table] block numbers */
    int32_t n_table;
    const int32_t *d_seq;    /* [n_seq] or NULL */
} lstk_paged_seqs;
/* d_q and d_out are [n_seq][n_head][head_dim] fp16; d_work holds at least lstk_attn_paged_work_bytes (0 for shapes that need
 * none or are rejected; what serves one max_len serves smaller ones) and belongs to one call at a time: calls that may overlap, captured ones among them, take one each.
 * Results do not depend on what else runs and repeat bit for bit. */
size_t lstk_attn_paged_work_bytes(int n_seq, int n_head, int n_head_kv, int head_dim, int max_len, int window, int n_sink);
int lstk_attn_paged(const lstk_paged_cache *cache, const lstk_paged_seqs *seqs, const uint16_t *d_q, int n_head, int window,
                    int n_sink, float scale, uint16_t *d_out, void *d_work, size_t work_bytes, lstk_stream_t stream);

/* The next token of each row of logits (the reference's Sampler works on host logits, src/sampler.cpp:20-82; its repeat
 * penalty is not part of this). Per row, with the values in descending order (equal values: the lower index first; NaN counts
 * as -inf, +inf as the largest float) and w = e^((x - x_max) / temperature):
 *   the first top_k values stay (<= 0: all), of those the ones with w >= min_p (<= 0: all; the largest always);
 *   of those the shortest run from the top that holds top_p of their sum (>= 1: all; the largest always);
 *   the token is the first whose running sum exceeds u times the sum of what stays, u in [0, 1); its probability is w over
 *   that sum. temperature <= 0 or NaN: the largest value, probability 1.
 * w is held as a whole multiple of 2^-44 (from a series good to 1.8e-14), so that sums are exact and the same in any order: a value
 * whose w is below 2^-45 is never drawn.
 * A row with nothing above -inf gives token -1 and probability 0. The four setting arrays are on the device, [n_rows] each;
 * a NULL one means temperature 1 / no cut; a NaN top_p or min_p means no cut. Row r of the logits is at
 * d_logits + r * ld_logits; n_vocab < 2^20. d_probs may be NULL. The workspace is as lstk_attn_paged's. */
typedef struct lstk_sampling {
    const float *d_temperature;
    const int32_t *d_top_k;
    const float *d_top_p, *d_min_p;
} lstk_sampling;
size_t lstk_sample_work_bytes(int n_rows, int n_vocab);
int lstk_sample(const float *d_logits, int64_t ld_logits, int n_rows, int n_vocab, const lstk_sampling *how, const float *d_u,
                int32_t *d_tokens, float *d_probs, void *d_work, size_t work_bytes, lstk_stream_t stream);

/* KvCache::remove_seq / truncate_seq / length (src/kv_cache.cpp:97-150, src/engine.h:75-80). */
int lstk_model_remove_seq(lstk_model *model, int32_t seq);
int lstk_model_truncate_seq(lstk_model *model, int32_t seq, int32_t keep);
int32_t lstk_model_seq_len(const lstk_model *model, int32_t seq);

/* Appends n_cells positions to sequence `seq` without running tokens: their K and V cells hold seeded
 * pseudo-random fp16 values in [-1, 1). A synthetic context of a given length, for measuring decode
 * at that KV length without a prefill; it has no counterpart in the reference. */
int lstk_model_fill_context(lstk_model *model, int32_t seq, int n_cells, uint64_t seed, lstk_stream_t stream);

/* Test hook (no counterpart in the reference): with d_states set, every forward also copies the residual
 * stream after each layer l, [T][n_embd] f32, to d_states + l * T * n_embd (a device buffer of at least
 * n_layer * n_batch * n_embd floats) on its stream, so a test can compare the model layer by layer with
 * a reference fed the same layer inputs; NULL turns it off. After the last layer only the output row has
 * been through the MoE block. */
int lstk_model_debug_capture(lstk_model *model, float *d_states);

/* Test hook (no counterpart in the reference): with d_moe_in set, every forward also copies the residual
 * stream entering layer l's MoE block (after attention, o-proj and residual; the input of ffn_norm and the
 * router), [T][n_embd] f32, to d_moe_in + l * T * n_embd, so a test can run a reference router on exactly
 * the device's router input; NULL turns it off. */
int lstk_model_debug_capture_moe_in(lstk_model *model, float *d_moe_in);

/* Test hook (no counterpart in the reference): options of the model's later forwards. Bit 0 set: a
 * single-token step runs RoPE and the new cell's K / V store in a launch of their own before the
 * attention, whose chunks then take several 64-cell passes, instead of inside the attention launch with
 * one-pass chunks (the plan steps of more tokens and contexts past 65536 cells always take), so a test can
 * compare the two plans on the same cache. 0 restores the default. */
int lstk_model_debug_options(lstk_model *model, int flags);

/* Test hook (no counterpart in the reference): the attention launch plan a step of n_tokens takes (host
 * arithmetic only, no device call), for n_head query / n_kv KV heads of head_dim over cells
 * [cell_begin, n_cells) of a kv_size-cell cache; rope_in asks for RoPE inside the launch (one token).
 * out[0..5] = query rows per work-group, row blocks, cells per chunk, chunks, RoPE kept inside the launch
 * (0 / 1), work-groups of the attention launch. Fails with LSTK_E_INVALID on arguments a model would
 * never pass. */
int lstk_debug_attn_plan(int n_tokens, int n_head, int n_kv, int head_dim, int kv_size, int n_cells, int cell_begin,
                         int rope_in, int32_t out[6]);
/* Test hook: whether such a step's attention (no RoPE inside) splits the cells over a work-group's wavefronts (1) or the
 * query rows (0); n_live = cells of the range that belong to the sequence (0: all). */
int lstk_debug_attn_split(int n_tokens, int n_head, int n_kv, int head_dim, int kv_size, int n_cells, int cell_begin,
                          int n_live, int32_t *split);

/* Engine::set_routing_trace (src/engine.cpp:179-186): with a path, creates the file and writes the
 * trace header ("LSTKRTE1", n_layer, n_expert, n_expert_used as little-endian int32); every later step
 * of lstk_model_decode then appends its token count and its router ids ([n_layer][n_tokens][k] int32,
 * -1 for rows the last layer skips), read back from the device after the step (a synchronisation per
 * step, as the reference's). NULL closes the file. Steps run through prepare / forward are not traced. */
int lstk_model_set_trace(lstk_model *model, const char *path);

/* Per-stage device time of the forward pass's own kernels, recorded like lstk_pool_timing:
 * stage 0 = norms + embedding, 1 = Q/K/V + QK-norm + RoPE + KV store, 2 = attention,
 * 3 = o-proj + residual, 4 = output head. The MoE block's stages are read with lstk_pool_timing. */
int lstk_model_set_timing(lstk_model *model, int enable);
int lstk_model_timing(lstk_model *model, double ms[5], int64_t launches[5]);

#ifdef __cplusplus
}
#endif

#endif /* LSTK_QWEN3_H */
