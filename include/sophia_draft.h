/*
 * sophia_draft.h -- C ABI of the drafted-token kernels: one step that runs a
 * tree of candidate tokens of each sequence through the decoder, and the parts
 * around it.  The reference decodes one token per step
 * (ml/runtime/generation/decode.py:68-79); its caches, whose contents these
 * kernels read and advance, are those of sophia_kda.h and sophia_decoder.h.
 *
 * Conventions as in sophia_kda.h: device pointers, strides in elements, an
 * explicit hipStream_t passed as void*, an int status.  Nothing here
 * allocates, synchronises or reads device data on the host.
 *
 * Trees.  The nodes of n_trees trees are packed rows.  Tree s is rows
 * cu_nodes[s] .. cu_nodes[s + 1) (int32, device), at most max_nodes <=
 * SOPHIA_TREE_NODES of them; parents[row] (int32, device) is the index of the
 * node's parent within its tree.  A node comes after its parent; a parent that
 * is not an earlier node of the tree makes the node a root, which follows the
 * cached tokens.  Rows of no tree are left as they are.
 */
#ifndef SOPHIA_DRAFT_H
#define SOPHIA_DRAFT_H

#include <stddef.h>
#include <stdint.h>

#include "sophia_kda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SOPHIA_TREE_NODES 64

/*
 * The KDA recurrence along every path of the trees, from the cached state, which
 * is not changed (beside sophia_kda_decode_conv_step, whose arguments it takes:
 * attention.py:226-258, 330-348 of the reference for each node).  With anc(i) =
 * node i and its ancestors:
 *   q, k, v = silu(conv) of the q | k | v channels, whose earlier samples are the
 *             node's ancestors and then the cached history (rounded to x's type, as the
 *             decode step rounds it); q, k normalised (flag), q times scale
 *   G_i = sum over anc(i) of the log-decay (below -104, where e^x is 0 in fp32: -104)
 *   u_i = beta_i (v_i - S^T (k_i e^G_i) - sum_{j in anc(i), j != i} (k_i . k_j e^(G_i - G_j)) u_j)
 *   o_i = S^T (q_i e^G_i) + sum_{j in anc(i)} (q_i . k_j e^(G_i - G_j)) u_j
 * All of it in fp32; o is rounded once.
 *   x_q, x_k, x_v : [rows, heads, 128] before the conv, one row stride.
 *   conv_weight   : [3 * heads * 128, kernel_size] fp32, kernel_size 1 .. 4;
 *   conv_state    : [n_slots, 3 * heads * 128, kernel_size - 1] fp32 (NULL when kernel_size is 1).
 *   g [rows, heads, 128], beta [rows, heads], A_log [heads], dt_bias [heads * 128].
 *   state         : [n_slots, heads, 128, 128] fp32; tree s uses slot slots[s]
 *                   (NULL: s).  A tree whose slot is out of range gets zeros.
 *   o             : [rows, heads, 128] of x's type.
 *   tape          : [rows, heads, 3, 128] fp32: u, k and G of each node, for sophia_tree_commit.
 * flags: SOPHIA_KDA_QK_L2NORM, SOPHIA_KDA_GATE_IN_KERNEL, SOPHIA_KDA_BETA_SIGMOID.
 * x, g and o: 16-byte aligned, row strides multiples of 8; state, tape and dt_bias 16-byte aligned.
 */
int sophia_kda_tree_step(const void *x_q, const void *x_k, const void *x_v, int64_t x_row_stride, int x_dtype,
                         const float *conv_weight, const float *conv_state, int kernel_size, const void *g,
                         int64_t g_row_stride, int g_dtype, const void *beta, int64_t beta_row_stride, int beta_dtype,
                         const float *A_log, const float *dt_bias, float scale, float lower_bound, unsigned flags,
                         const float *state, int n_slots, const int32_t *slots, const int32_t *cu_nodes,
                         const int32_t *parents, int n_trees, int64_t rows, int max_nodes, int num_heads, int head_dim,
                         void *o, int64_t o_row_stride, float *tape, void *stream);

/*
 * An accepted path of every tree into the caches of all layers, in one launch (for
 * each SOPHIA_COMMIT_KDA / SOPHIA_COMMIT_MLA layers).  The nodes of tree s are
 * path[s, 0 .. n_path[s]) (int32, device; row stride path_stride), from a root
 * downwards; an index that is no node of the tree ends the path.  With j over the
 * path and a its last node, for each KDA layer
 *   S = Diag(e^G_a) S + sum_j (k_j e^(G_a - G_j)) u_j^T, history = the last samples of (history, x of the path)
 * and for each MLA layer  cache[slot, cached[s] + t] = latent[path[s, t]]  (positions
 * past max_seq are left out).  An empty path changes nothing.  Trees of one call
 * have different slots; a slot out of range is left out.
 *   kda[l] : tape, state and conv_state as above (conv_state NULL when kernel_size is 1),
 *            x the pre-conv rows [rows, 3 * heads * 128] of x_dtype, row stride x_stride.
 *   mla[l] : latent [rows, rank] of latent_dtype, row stride latent_stride; cache
 *            [n_slots, max_seq, rank] fp32 with slot_stride; rank a multiple of 4, 16-byte
 *            aligned rows of cache, rows of latent aligned to 4 elements.
 */
#define SOPHIA_COMMIT_KDA 48
#define SOPHIA_COMMIT_MLA 24
typedef struct {
  const float *tape;
  const void *x;
  int64_t x_stride;
  float *conv_state;
  float *state;
} sophia_commit_kda;
typedef struct {
  const void *latent;
  int64_t latent_stride;
  float *cache;
  int64_t slot_stride;
} sophia_commit_mla;
int sophia_tree_commit(const int32_t *path, int64_t path_stride, const int32_t *n_path, int max_path,
                       const int32_t *cu_nodes, int n_trees, int64_t rows, const int32_t *slots, int n_slots,
                       const sophia_commit_kda *kda, int n_kda, int num_heads, int head_dim, int kernel_size, int x_dtype,
                       const sophia_commit_mla *mla, int n_mla, const int64_t *cached, int max_seq, int rank,
                       int latent_dtype, void *stream);

/*
 * The same for trees of which only the first max_nodes nodes were looked at (the step's
 * max_nodes; sophia_tree_commit: SOPHIA_TREE_NODES): the tape holds nothing of the
 * others, and an index of one of them ends the path too.
 */
int sophia_tree_commit_within(const int32_t *path, int64_t path_stride, const int32_t *n_path, int max_path,
                              const int32_t *cu_nodes, int n_trees, int64_t rows, int max_nodes, const int32_t *slots,
                              int n_slots, const sophia_commit_kda *kda, int n_kda, int num_heads, int head_dim,
                              int kernel_size, int x_dtype, const sophia_commit_mla *mla, int n_mla, const int64_t *cached,
                              int max_seq, int rank, int latent_dtype, void *stream);

/*
 * MLA attention in latent space of every node of the trees over the cached latents
 * of its sequence and the drafted ones of itself and its ancestors (beside
 * sophia_mla_decode_attn, attention.py:609-657 of the reference):
 *   out[i, h] = sum_k softmax_k(scale qa[i, h] . key_k) key_k,
 *   keys: cache[slot, 0 .. cached[s]) and latent[j], j in anc(i).
 *   qa, latent, out : [rows, heads, rank], [rows, rank], [rows, heads, rank] of one type.
 *   cache           : [n_slots, max_seq, rank] fp32, slot_stride between slots; tree s uses
 *                     slot slots[s] (NULL: s).  A tree whose slot is out of range gets zeros.
 *   cached          : [n_trees] int64, taken into [0, max_seq].
 * bf16: the cached latents are rounded to bf16, the probabilities enter the value product
 * to 2^-16; fp32: fp32 products.  Scores, softmax and sums are fp32; out is rounded once.
 * rank in {32, 64, 128, 256}; heads <= 16; scale > 0; row strides multiples of 8, every
 * pointer 16-byte aligned.  With splits > 1 a tree's keys are divided into equal
 * ranges of split_keys (a multiple of 64) or more, as long as keeps the chip full, at most
 * `splits` of them; this needs a workspace of sophia_mla_tree_workspace_size(n_trees,
 * max_nodes, rank, dtype, splits) bytes.
 */
size_t sophia_mla_tree_workspace_size(int n_trees, int max_nodes, int rank, int dtype, int splits);
int sophia_mla_tree_attn(const void *qa, int64_t qa_stride, const void *latent, int64_t latent_stride, int dtype,
                         const float *cache, int64_t slot_stride, int n_slots, int max_seq, const int32_t *slots,
                         const int64_t *cached, const int32_t *cu_nodes, const int32_t *parents, int n_trees,
                         int64_t rows, int max_nodes, float scale, void *out, int64_t out_stride, int heads, int rank,
                         int splits, int split_keys, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Penalties, biases and masks on the logits of the next tokens.  With row r of
 * sequence s (cu_nodes NULL: s = r; else the tree that holds r):
 *   seen(v):  v is in history[s, 0 .. history_len[s]), or the token of a node of anc(r)
 *   count(v): how often, from history[s, prompt_len[s]] on (NULL: 0) and in anc(r)
 *   y = seen ? (x > 0 ? x / repetition[s] : x repetition[s]) - frequency[s] count - presence[s] (count > 0) : x
 *   out = allowed ? y + sum of bias[s, j] with bias_ids[s, j] = v : -inf
 *   logits, out : [rows, vocab] of one type, out may be logits itself.
 *   history     : [n_seqs, history_stride] int64 or NULL, with trees without the nodes' tokens
 *                 (node 0's neither); ids outside the vocabulary are not
 *                 looked at, in bias_ids neither; history_len is taken into [0, history_max].
 *   repetition (> 0), presence, frequency : [n_seqs] fp32 or NULL (1, 0, 0).
 *   bias_ids, bias : [n_seqs, n_bias].
 *   allowed     : [n_masks, (vocab + 31) / 32] int32 or NULL, bit v % 32 of word v / 32; row r
 *                 has mask allowed_rows[r] (NULL: r); out of range: every token is allowed.
 * Any alignment is taken; 16-byte aligned rows are faster.  NaN stays NaN where allowed.
 */
int sophia_adjust_logits(const void *logits, int64_t logits_stride, void *out, int64_t out_stride, int dtype,
                         int64_t rows, int vocab, const int64_t *history, int64_t history_stride,
                         const int32_t *history_len, const int32_t *prompt_len, int history_max,
                         const float *repetition, const float *presence, const float *frequency,
                         const int64_t *bias_ids, const float *bias, int n_bias, const int32_t *allowed, int n_masks,
                         const int32_t *allowed_rows, const int32_t *cu_nodes, const int32_t *parents,
                         const int64_t *tokens, int n_seqs, int max_nodes, void *stream);

/*
 * The model's choice at every node, and the walk along the drafted tokens that
 * agree with it:
 *   chosen[r]   = the index of row r's greatest logit, of equal ones the lowest (NaN is
 *                 never chosen; a row without a value above -inf gives 0); of all rows
 *   path[s]     = node 0, then again and again the first child whose token is the choice of
 *                 the node before it; -1 behind the path (max_nodes entries, stride path_stride)
 *   n_path[s]   = its length (0 for a tree without nodes)
 *   next_token[s] = the choice of its last node (-1 for a tree without nodes)
 *   logits [rows, vocab] of any alignment, tokens [rows] int64.  Needs a workspace of sophia_tree_accept_workspace_size(rows, vocab) bytes.
 */
size_t sophia_tree_accept_workspace_size(int64_t rows, int vocab);
int sophia_tree_accept(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab,
                       const int64_t *tokens, const int32_t *cu_nodes, const int32_t *parents, int n_trees,
                       int max_nodes, int32_t *path, int64_t path_stride, int32_t *n_path, int64_t *next_token,
                       int64_t *chosen, void *workspace, size_t workspace_bytes, void *stream);

/*
 * The same, but a row without a value above -inf (its mask allows nothing, or it is NaN)
 * has no choice: chosen is -1, a path ends at such a node, and next_token is -1 there.
 */
int sophia_tree_accept_strict(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab,
                              const int64_t *tokens, const int32_t *cu_nodes, const int32_t *parents, int n_trees,
                              int max_nodes, int32_t *path, int64_t path_stride, int32_t *n_path, int64_t *next_token,
                              int64_t *chosen, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SOPHIA_DRAFT_H */
