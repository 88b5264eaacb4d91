/*
 * jinf MI355X kernels: drafted tokens and bounded KV caches.
 *
 * Four operators around the K / V caches that jinf_attention_decode reads and
 * jinf_rmsnorm_qkv_rope_batch writes (kernels_ext.h):
 *   - attention of a tree of drafted tokens over a cache, to check several
 *     guessed continuations in one step;
 *   - the accepted tokens' K / V rows into the caches;
 *   - decode attention that also adds up the attention weight each cached
 *     position receives;
 *   - the positions of least accumulated weight out of the caches.
 * The reference decodes one token per step over an ever-growing cache
 * (src/engine.cpp:684-805, cuda/attention_kernel.cu:25-96) and has none of
 * them; scores, softmax and GQA head mapping are those of its attention.
 *
 * Common rules (those of kernels_ext.h):
 *   - pointers are DEVICE pointers on the stream's device, which is current;
 *     all work is asynchronous on `stream`; nothing allocates, frees or
 *     synchronizes; calls can be captured in a HIP graph;
 *   - cache element (sequence s, position t, kv head j, dim d) is at
 *     s * ld_seq + t * ld_pos + j * head_dim + d in k_cache / v_cache, of
 *     kv_type JINF_HIP_F32 or JINF_HIP_F16; ld_pos >= n_heads_kv * head_dim and,
 *     with more than one sequence, ld_seq >= max_ctx * ld_pos (or 0 where a
 *     function says so: every sequence reads one cache); head_dim <= 1024;
 *   - accumulated weights are fp32, (s, j, t) at s * ld_w_seq + j * ld_w + t,
 *     ld_w >= max_ctx and, with more than one sequence, ld_w_seq >=
 *     n_heads_kv * ld_w;
 *   - lens: device array of n_seq int32, values clamped to [0, max_ctx];
 *   - outputs overlap no other argument unless a function says so;
 *   - JINF_HIP_OK, JINF_HIP_ERR_INVALID (nothing enqueued) or
 *     JINF_HIP_ERR_DEVICE (a launch failed); no sequences is JINF_HIP_OK with
 *     nothing enqueued;
 *   - a workspace is device memory of any contents, 16-byte aligned, free for
 *     other use after the call's work; concurrent calls need one each, and so
 *     do captured graphs that may be replayed at the same time.
 *
 * This header includes no HIP or CUDA header.
 */
#ifndef JINF_KV_HIP_H
#define JINF_KV_HIP_H

#include <stddef.h>
#include <stdint.h>
#include "../kernels_ext.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most drafted tokens per sequence. */
#define JINF_HIP_MAX_NODES 256

/* GQA attention of up to max_nodes (<= JINF_HIP_MAX_NODES) drafted tokens per
 * sequence.  Node i of sequence s attends to the cached positions t < lens[s]
 * and to the drafted tokens j whose bit is set in its mask row:
 *   out[s, i, h] = sum softmax(scale * q[s,i,h] . k) v   over those rows,
 * kv head h / (n_heads / n_heads_kv).  A node with no row gets zeros, one with a
 * NaN score NaN (an infinite key may make a score NaN).  A non-finite V value makes
 * its dim non-finite in the nodes that attend to it; non-finite values in rows that a
 * node does not attend to do not reach it.
 *   - q, out: fp32; node (s, i) at s * ld_q_seq + i * ld_q (ld_out alike).
 *   - k_draft, v_draft: the nodes' K (rotated to their positions) and V rows,
 *     (s, i) at s * ld_draft_seq + i * ld_draft, of draft_type F32 or F16; used
 *     as the cache would hold them (rounded once to an fp16 cache's type).
 *   - mask: [n_seq][max_nodes][ceil(max_nodes / 64)] words, bit j % 64 of word
 *     j / 64 for node j (itself included, if it is to be).  Any relation may be
 *     given; bits at or past the sequence's node count are ignored.
 *   - n_nodes: nodes of each sequence (device int32, clamped to [0,
 *     max_nodes]), or NULL: max_nodes.  Output rows past it are not written; what
 *     the other rows past it hold does not matter.
 *   - ld_seq may be 0 (all sequences share one cached prefix).
 *   - scale as in jinf_attention_decode (0: 1 / sqrt(head_dim)).
 * Fast path: head_dim 64 or 128, q, caches and their strides 16-byte aligned;
 * an fp16 cache then needs |q * scale| < 45000.  Any other layout runs one
 * wave per (node, head), much slower.
 * Workspace (optional: NULL or too small runs every context in one piece):
 * jinf_attention_tree_workspace_bytes(...) bytes. */
int jinf_attention_tree(float* out, int ld_out, int64_t ld_out_seq, const float* q, int ld_q,
                        int64_t ld_q_seq, const void* k_cache, const void* v_cache, int kv_type,
                        int64_t ld_pos, int64_t ld_seq, const int32_t* lens, const void* k_draft,
                        const void* v_draft, int draft_type, int ld_draft, int64_t ld_draft_seq,
                        const uint64_t* mask, const int32_t* n_nodes, int max_nodes, int n_seq,
                        int max_ctx, int head_dim, int n_heads, int n_heads_kv, float scale,
                        void* workspace, size_t workspace_bytes, hipStream_t stream);

/* Workspace bytes jinf_attention_tree can use (0 for an empty shape). */
size_t jinf_attention_tree_workspace_bytes(int n_seq, int max_nodes, int n_heads, int n_heads_kv,
                                           int head_dim, int max_ctx);

/* Appends rows to the caches: for a < counts[s], row index[s * n_take + a] of
 * sequence s's n_rows rows (k_rows / v_rows, (s, i) at s * ld_rows_seq + i *
 * ld_rows, of rows_type) becomes position lens[s] + a, rounded once where the
 * cache is fp16 and the rows are not.
 *   - index NULL: row a itself (n_take <= n_rows).  A row may be named twice.
 *     An index outside [0, n_rows) stores +0.0.
 *   - counts NULL: n_take rows for every sequence; values are clamped to [0,
 *     n_take].  Positions at or past max_ctx are not stored.
 *   - weights (may be NULL): the appended positions' accumulated weights are
 *     set to 0.
 *   - lens_out (may be NULL; not lens itself): the new lengths. */
int jinf_cache_append(void* k_cache, void* v_cache, int kv_type, int64_t ld_pos, int64_t ld_seq,
                      float* weights, int64_t ld_w, int64_t ld_w_seq, const int32_t* lens,
                      int32_t* lens_out, const void* k_rows, const void* v_rows, int rows_type,
                      int ld_rows, int64_t ld_rows_seq, int n_rows, const int32_t* index,
                      const int32_t* counts, int n_take, int n_seq, int max_ctx, int head_dim,
                      int n_heads_kv, hipStream_t stream);

/* jinf_attention_decode (same q, out, caches, lens, scale and results; each
 * within its tolerance) that also adds each position's attention weight to
 * its sum:
 *   weights[s, j, t] += sum over the query heads h of kv head j of
 *                       softmax_t(scale * q[s,h] . k[s,t,j]),   t < lens[s].
 * Weights at or past lens[s] are neither read nor written.  ld_seq may be 0.
 * Fast path as jinf_attention_tree's.
 * Workspace (required): jinf_attention_scored_workspace_bytes(...) bytes. */
int jinf_attention_decode_scored(float* out, int ld_out, const float* q, int ld_q,
                                 const void* k_cache, const void* v_cache, int kv_type,
                                 int64_t ld_pos, int64_t ld_seq, float* weights, int64_t ld_w,
                                 int64_t ld_w_seq, const int32_t* lens, int n_seq, int max_ctx,
                                 int head_dim, int n_heads, int n_heads_kv, float scale,
                                 void* workspace, size_t workspace_bytes, hipStream_t stream);

size_t jinf_attention_scored_workspace_bytes(int n_seq, int n_heads, int n_heads_kv, int head_dim,
                                             int max_ctx);

/* Takes each (sequence, kv head) down to at most `budget` positions.  Where
 * lens[s] > budget, the first n_first and the last n_recent positions stay, and
 * of those between them the budget - n_first - n_recent with the largest
 * accumulated weight (the lowest position first among equal ones; NaN counts as
 * larger than any number, -0 as 0).  The kept positions move together, in their
 * order, to rows 0 .. budget - 1 of k_out / v_out and of weights_out; each kv
 * head keeps positions of its own.  Where lens[s] <= budget everything stays.
 * Rows at or past the new length keep what they held.
 *   - In place: k_out == k_cache, v_out == v_cache, weights_out == weights, each
 *     with its input's strides.  Otherwise no output may overlap an input;
 *     out strides are those of caches of min(budget, max_ctx) positions or more.
 *   - kept (may be NULL): [n_seq][n_heads_kv][budget] int32, the old position of
 *     each row, -1 at or past the new length.
 *   - lens_out (may be NULL; may be lens): min(lens[s], budget).
 *   - budget >= 0, n_first >= 0, n_recent >= 0, n_first + n_recent <= budget.
 *   - ld_seq may not be 0 with more than one sequence.
 * Workspace (required): jinf_cache_evict_workspace_bytes(...) bytes. */
int jinf_cache_evict(void* k_out, void* v_out, int64_t ld_pos_out, int64_t ld_seq_out,
                     const void* k_cache, const void* v_cache, int kv_type, int64_t ld_pos,
                     int64_t ld_seq, float* weights_out, int64_t ld_wo, int64_t ld_wo_seq,
                     const float* weights, int64_t ld_w, int64_t ld_w_seq, const int32_t* lens,
                     int32_t* lens_out, int32_t* kept, int budget, int n_first, int n_recent,
                     int n_seq, int max_ctx, int head_dim, int n_heads_kv, void* workspace,
                     size_t workspace_bytes, hipStream_t stream);

size_t jinf_cache_evict_workspace_bytes(int n_seq, int n_heads_kv, int budget);

#ifdef __cplusplus
}
#endif

#endif /* JINF_KV_HIP_H */
