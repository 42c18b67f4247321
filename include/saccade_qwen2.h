/*
 * saccade_qwen2.h -- C ABI of the Qwen2 decoder glue that surrounds the C-TARQ linears
 * (libsaccade_ctarq.so).  Each entry point is one step of saccade-runner's model, run on the GPU:
 *
 *   sc_qwen2_embed         <- Embedding::forward            saccade-runner/src/model.rs:512
 *   sc_qwen2_add_rmsnorm   <- residual add + RmsNorm::forward  model.rs:92-98, 295-304
 *   sc_qwen2_rope_append   <- RotaryEmbedding::apply + the KV-cache concat  model.rs:111-154, 225-236
 *   sc_qwen2_attention     <- scores, softmax, attn . v (GQA)  model.rs:238-257
 *   sc_qwen2_silu_mul      <- Mlp::forward's silu(gate) * up    model.rs:295-299
 *   sc_qwen2_add_rmsnorm_route, sc_qwen2_silu_mul_route
 *                          <- the two above with the next linears' router (op.rs:64-73,
 *                             heuristics.rs:3-14) in their epilogue, consumed by
 *                             sc_forward_group_routed
 *   sc_qwen2_f16_to_f32    <- ProjectionLayer::forward's to_dtype back to f32  model.rs:61
 *   sc_qwen2_paged_append, sc_qwen2_paged_attention
 *                          <- the two cache steps on a paged cache of f32, f16 or bf16 shared by ragged
 *                             sequences (the reference concatenates one f32 tensor per sequence)
 *   sc_qwen2_process_logits
 *                          <- penalties, biases and grammar masks before the argmax of
 *                             saccade-runner/src/bin/verify.rs:98-130 (the reference has the argmax only)
 *
 * The linears themselves are sc_forward / sc_forward_group calls (saccade_ctarq.h).  Everything is
 * f32 except the inputs of the linears, which these kernels write as f16 (the projection layer's
 * to_dtype(F16), model.rs:58-60).  Calls are asynchronous on `stream` and allocate nothing.
 */
#ifndef SACCADE_QWEN2_H
#define SACCADE_QWEN2_H

#include <stddef.h>
#include <stdint.h>

#include "saccade_ctarq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* out[t] = f32(table[ids[t]]) for an f16 embedding table [vocab, hidden]; an id outside the table
 * records SC_EDEVICE in *status (nullable device word) and reads row 0. */
SC_API sc_status sc_qwen2_embed(const int64_t* ids, int64_t tokens, const uint16_t* table, int64_t vocab,
                                int64_t hidden, float* out, uint32_t* status, void* stream);

/* resid [tokens, hidden] += delta (nullable); out = resid / sqrt(mean(resid^2) + eps) * w, written as
 * f16 (SC_F16: the input of the next linears) or f32 (SC_F32: the final norm before lm_head).  The
 * mean is a fixed-order f32 sum (256 strided partial sums, then those in order).  hidden <= 16384
 * (the row is staged in shared memory); SC_EINVAL otherwise. */
SC_API sc_status sc_qwen2_add_rmsnorm(float* resid, const float* delta, const float* weight, int64_t tokens,
                                      int64_t hidden, float eps, void* out, int out_dtype, void* stream);

/* q [tokens, num_heads, head_dim] rotated in place; k rotated and, with v, written at cache slot
 * slot[t], position pos[t] of k_cache / v_cache [slots, num_kv_heads, max_pos, head_dim]. */
SC_API sc_status sc_qwen2_rope_append(float* q, const float* k, const float* v, const float* cos_table,
                                      const float* sin_table, const int32_t* slot, const int32_t* pos, int64_t tokens,
                                      int num_heads, int num_kv_heads, int head_dim, int max_pos, float* k_cache,
                                      float* v_cache, void* stream);

/* Scratch bytes sc_qwen2_attention needs for `tokens` queries. */
SC_API size_t sc_qwen2_attention_scratch(int64_t tokens, int num_heads, int num_kv_heads, int head_dim, int max_pos);

/* Causal GQA attention: token t attends the keys 0..pos[t] of its cache slot; out_f16 [tokens,
 * num_heads * head_dim].  max_query_pos bounds every pos[t] (it sizes the key blocks launched).
 * Limits (SC_EINVAL otherwise): head_dim 32, 64 or 128; at most 8 query heads per KV head and 128
 * query heads; max_query_pos < 8192.  Keys go in blocks of 256: per block the scores (per-lane
 * partial dot products over head_dim, then a 32-lane xor butterfly), its max, exp evaluated in f64
 * and rounded to f32, the lane-strided sum, p . v over the keys in order; blocks are combined in
 * order, so the result is a fixed function of the inputs. */
SC_API sc_status sc_qwen2_attention(const float* q, const float* k_cache, const float* v_cache, const int32_t* slot,
                                    const int32_t* pos, int64_t tokens, int num_heads, int num_kv_heads, int head_dim,
                                    int max_pos, int max_query_pos, float* scratch, size_t scratch_bytes,
                                    uint16_t* out_f16, void* stream);

/* out_f16[i] = f16(silu(f32(gate[i])) * f32(up[i])), silu(g) = g / (1 + exp(-g)). */
SC_API sc_status sc_qwen2_silu_mul(const uint16_t* gate, const uint16_t* up, int64_t n, uint16_t* out_f16,
                                   void* stream);

/* out[i] = f32(x[i]) for f16 x. */
/* The router of the linears that read the output, fused into the kernel that writes it.  Each
 * kernel is one CTA per token: it writes the token's f16 row exactly as the plain kernel does
 * (same bits), keeps it in shared memory, and routes the token for every layer of `group`
 * (heuristics.rs:3-14, op.rs:64-73: f64 sums decide when the thresholds lie outside the f32 error
 * band, else the reference's f32 chains are replayed), writing mask[l][t] (0/1); the last CTA to
 * finish writes the ascending routed list routed_idx[l][0..n) and n_routed[l][0] of each layer.
 * These are the routing sc_forward_group would compute on the same row, and sc_forward_group_routed
 * takes them instead of routing again.  `counter` is one uint32 in device memory that is zero
 * before the call (the kernel leaves it zero).  The group's layers must read the whole row:
 * in_features == hidden (norm) or width (silu); set_bypass_c_tarq routes every token.
 * add_rmsnorm_route: resid += delta (nullable), out_f16 = f16 RMSNorm as sc_qwen2_add_rmsnorm
 * (hidden <= 16384).  silu_mul_route: out_f16 [tokens, width] = f16(silu(gate) * up) as
 * sc_qwen2_silu_mul (width a multiple of 8, width <= 65536).  No reference counterpart: the
 * reference routes inside each projection (op.rs:64-73). */
SC_API sc_status sc_qwen2_add_rmsnorm_route(float* resid, const float* delta, const float* weight, int64_t tokens,
                                            int64_t hidden, float eps, uint16_t* out_f16, const sc_group* group,
                                            uint8_t* const* mask, int32_t* const* routed_idx,
                                            int32_t* const* n_routed, uint32_t* counter, void* stream);
SC_API sc_status sc_qwen2_silu_mul_route(const uint16_t* gate, const uint16_t* up, int64_t tokens, int64_t width,
                                         uint16_t* out_f16, const sc_group* group, uint8_t* const* mask,
                                         int32_t* const* routed_idx, int32_t* const* n_routed, uint32_t* counter,
                                         void* stream);

/* ---- A paged cache.  k_pages / v_pages hold num_pages pages of [num_kv_heads][page_size][head_dim]
 * elements of cache_dtype (SC_F32, SC_F16, SC_BF16), page p at element p * page_stride (each page's
 * own elements contiguous).  Row b of block_table [num_seqs][max_pages] lists sequence b's pages in
 * order: its position p is row p % page_size of page block_table[b][p / page_size].  Sequence b owns
 * token rows cu_q[b] .. cu_q[b + 1] (cu_q [num_seqs + 1], ascending from 0; rows from cu_q[num_seqs] on
 * belong to no sequence and their outputs are left as they were) and kv_len[b] positions counting those
 * tokens: its i-th new token sits at position kv_len[b] - (cu_q[b + 1] - cu_q[b]) + i.  All of these are
 * device arrays read by the kernels, so a captured graph replays with new lengths and pages.
 * Limits (SC_EINVAL otherwise): head_dim 64 or 128; page_size a power of two in 8..256; num_heads a
 * multiple of num_kv_heads with at most 64 query heads per KV head.  Nothing of a page is read or
 * written that the lengths do not cover, except that attention may load the rest of a sequence's
 * last page, whatever it holds.  A position, page or length outside the tables records SC_EDEVICE in
 * *status (nullable device word; see sc_layer_check's codes) and is skipped, never followed. */

/* Rotates q and k (out[d] = x[d] cos[d] - x[d + hd/2] sin[d], out[d + hd/2] = x[d + hd/2] cos[d + hd/2] +
 * x[d] sin[d + hd/2] in f32, with row `position` of cos_table / sin_table [max_pos][head_dim]), writes
 * the rotated k and v into the pages and the rotated q to q_out [tokens][num_heads][head_dim], all as
 * cache_dtype with one rounding.  q, k, v: in_dtype rows (heads contiguous) q_stride, k_stride and
 * v_stride elements apart, so slices of one projection buffer serve.  in_dtype is SC_F32 or
 * cache_dtype.  q_out may be q itself (same type, q_stride = num_heads * head_dim) and must not lie over q, k or v
 * otherwise.  A token whose
 * position lies outside the rotation tables is left out; one without a page gets its q only. */
SC_API sc_status sc_qwen2_paged_append(const void* q, const void* k, const void* v, int in_dtype, int64_t q_stride,
                                       int64_t k_stride, int64_t v_stride, int64_t tokens, const float* cos_table,
                                       const float* sin_table, int64_t max_pos, int num_heads, int num_kv_heads,
                                       int head_dim, void* k_pages, void* v_pages, int cache_dtype, int64_t num_pages,
                                       int64_t page_stride, int page_size, const int32_t* block_table,
                                       int64_t max_pages, const int32_t* cu_q, const int32_t* kv_len, int64_t num_seqs,
                                       void* q_out, uint32_t* status, void* stream);

/* Scratch bytes sc_qwen2_paged_attention needs with these arguments (no initial contents; one call uses it at
 * a time); 0 for short sequences of few new tokens, and for arguments it refuses. */
SC_API size_t sc_qwen2_paged_attention_scratch(int64_t num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                               int64_t max_q_len, int64_t max_kv_len, int cache_dtype);

/* Causal attention of each sequence's new tokens over its pages: the token at position p attends
 * positions 0..p, o = sum softmax(scale * q . k) v per query head (grouped onto the KV heads), f32
 * sums and softmax statistics.  q [tokens][num_heads][head_dim] of cache_dtype, rows q_stride elements
 * apart; out [tokens][num_heads][head_dim] contiguous, out_dtype = cache_dtype (an f32 cache may also
 * write SC_F16, the linears' input); it may be q itself (same type, q_stride = num_heads * head_dim), or none of its
 * bytes.  lse (nullable, f32 [tokens][num_heads]) = log sum exp(scale * q . k).
 * A token at a negative position attends nothing: its output is 0, its lse -inf.  max_q_len and max_kv_len bound
 * every sequence's new tokens and positions and choose the kernels (a sequence with more new tokens is skipped and
 * recorded; more positions are attended all the same).  q, the pages, their strides and out are 16-byte aligned.
 * 16-bit caches run on the tensor cores.  With more than 16 rows (max_q_len x query heads of a KV head) each softmax
 * weight is rounded once to the cache's type there (f16: at worst to steps of 2^-30 of the row's largest), with fewer
 * it is held in two such parts; the softmax's sums are of the unrounded weights.  Whatever lies behind a token's
 * position, NaN and infinities too, does not touch its output; one that attends a key that is NaN or a value that is
 * not finite gets no finite result from it (nor may one of a bf16 cache with values above 2^64). */
SC_API sc_status sc_qwen2_paged_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages,
                                          int cache_dtype, int64_t num_pages, int64_t page_stride, int page_size,
                                          const int32_t* block_table, int64_t max_pages, const int32_t* cu_q,
                                          const int32_t* kv_len, int64_t num_seqs, int64_t tokens, int num_heads,
                                          int num_kv_heads, int head_dim, int64_t max_q_len, int64_t max_kv_len,
                                          float scale, void* out, int out_dtype, float* lse, void* scratch,
                                          size_t scratch_bytes, uint32_t* status, void* stream);

/* Scratch bytes sc_qwen2_process_logits needs for best / best_value (no initial contents; one call uses
 * it at a time); without both it needs none. */
SC_API size_t sc_qwen2_process_logits_scratch(int64_t rows, int64_t vocab);

/* Logits [rows][vocab] of dtype (SC_F32, SC_F16, SC_BF16), rows `stride` apart, of the tokens vocab_begin ..
 * vocab_begin + vocab (a tensor-parallel rank's slice; every id below is of the whole vocabulary) ->
 * out (out_stride apart; may be logits itself with the same stride, or none of its elements).  Per row and
 * token v, in f32 and rounded once:
 *   x = logits[v]
 *   v among the row's history: x = x > 0 ? x / repetition : x * repetition
 *   x = x - frequency * n - (n > 0 ? presence : 0), n = times v occurs among the generated tokens
 *   x = x + the last bias entry of v;   x = -inf where the row's grammar mask does not allow v
 * history [rows][history_stride] (ids; others than the slice's are passed over): the first hist_len[r]
 * are the row's, of these the first prompt_len[r] its prompt (null prompt_len: all generated).
 * repetition, presence, frequency: f32 per row (null: 1, 0, 0).  bias entries bias_ptr[r] .. bias_ptr[r + 1]
 * of bias_ids / bias_vals [num_bias], at most 4095 a row.  mask [mask_rows][mask_words] of bits, bit v % 32
 * of word v / 32: 1 allows v; mask_row[r] is the row's mask, negative for none (null mask_row: mask r).
 * best (nullable int64 [rows]) and best_value (nullable, dtype [rows]): the id and value of the largest
 * output, the first of equals, NaN above all as torch.argmax has it.  A length, mask row or number of
 * bias entries out of range records SC_EDEVICE in *status (nullable) and is cut to what there is (a
 * mask row: no mask).  history_stride <= 524287, rows <= 2^20 and vocab_begin + vocab <= 2^30, SC_EINVAL
 * otherwise. */
SC_API sc_status sc_qwen2_process_logits(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t stride,
                                         int64_t vocab_begin, const int32_t* history, int64_t history_stride,
                                         const int32_t* prompt_len, const int32_t* hist_len, const float* repetition,
                                         const float* presence, const float* frequency, const int32_t* bias_ptr,
                                         const int32_t* bias_ids, const float* bias_vals, int64_t num_bias,
                                         const int32_t* mask, int64_t mask_words, int64_t mask_rows,
                                         const int32_t* mask_row, void* out, int64_t out_stride, int64_t* best,
                                         void* best_value, void* scratch, size_t scratch_bytes, uint32_t* status,
                                         void* stream);

SC_API sc_status sc_qwen2_f16_to_f32(const uint16_t* x, int64_t n, float* out, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SACCADE_QWEN2_H */
