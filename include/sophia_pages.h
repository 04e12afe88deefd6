/*
 * sophia_pages.h -- C ABI of the kernels for latents in pages and for beams: the
 * MLA layers' latents in pages that sequences share, the choice of the best
 * continuations, and the moves of caches that follow from it.  The reference keeps
 * a rectangular cache and one sequence per row of it
 * (ml/runtime/model/attention.py:122-143, 560-583).
 *
 * Conventions as in sophia_kda.h: device pointers, strides in elements, an
 * explicit hipStream_t passed as void*, an int status.  Nothing here
 * allocates, synchronises or reads device data on the host.
 *
 * Pages.  A layer's pool is [n_pages, page_size, rank] of one type (bf16 or fp32),
 * page_stride elements from page to page, page_size a power of two.  A sequence's
 * key j is row j % page_size of page table[slot, j / page_size] (int32, device,
 * [table_rows, max_pages], table_stride).  A page id out of [0, n_pages) is no page:
 * its keys are not there, what would be written to it is left out.  Sequence s uses
 * row slots[s] of the table (NULL: s); a row out of range has no pages.
 *
 * New tokens.  The last tokens of the sequences are packed rows: sequence s has rows
 * cu_seqlens[s] .. cu_seqlens[s + 1) (int32, device), n of them, and kv_len[s] (int64,
 * device) tokens in all, those included: row i of it is at position kv_len[s] - n + i.
 */
#ifndef SOPHIA_PAGES_H
#define SOPHIA_PAGES_H

#include <stddef.h>
#include <stdint.h>

#include "sophia_kda.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * MLA attention in latent space over paged latents (beside sophia_mla_decode_attn,
 * attention.py:609-657 of the reference): for each new row at position p and each head
 *   out[h] = sum_{j <= p} softmax_j(scale qa[h] . c_j) c_j   over the keys j that there are.
 * A row without keys gets zeros.  Rows of no sequence, and rows of a sequence past its
 * first max_new, are left as they are.
 *   qa, out : [rows, heads, rank] of `dtype`, the type of the pages; 16-byte aligned, row
 *             strides multiples of 8.  heads 1 .. 128, rank 32, 64, 128 or 256.
 *   max_new, max_len : bounds (host) on the new tokens and on kv_len of a sequence; max_new
 *             sizes the launch, max_len only the division of work, not the result.
 *   splits  : key ranges of a sequence at most (0: chosen here), the same in both calls.
 * A latent that is not finite does not reach the rows before its position; a row at or after
 * it is not finite in at least one value.  Scores, softmax and sums are fp32; in bf16, a
 * probability enters the value product as two bf16 numbers.
 */
size_t sophia_mla_paged_workspace_size(int n_seqs, int64_t rows, int max_new, int64_t max_len, int heads, int rank,
                                       int dtype, int splits);
int sophia_mla_paged_attn(const void *qa, int64_t qa_stride, int dtype, const void *pages, int64_t page_stride,
                          int64_t n_pages, int page_size, const int32_t *table, int64_t table_stride, int table_rows,
                          int max_pages, const int32_t *slots, const int32_t *cu_seqlens, const int64_t *kv_len,
                          int n_seqs, int64_t rows, int max_new, int64_t max_len, float scale, void *out,
                          int64_t out_stride, int heads, int rank, int splits, void *workspace, size_t workspace_bytes,
                          void *stream);

/*
 * sophia_mla_latent_norms with paged latents: q_lat and kv_lat [rows, q_rank] and
 * [rows, kv_rank] normalised in place, and each new token's latent written to its place in
 * the pages (of the rows' type).  Rows of no sequence are normalised too, and written nowhere.
 */
int sophia_mla_latent_norms_paged(void *q_lat, int64_t q_stride, void *kv_lat, int64_t kv_stride, int64_t rows,
                                  int q_rank, int kv_rank, int dtype, const float *q_norm_weight, float q_eps,
                                  const float *kv_norm_weight, float kv_eps, void *pages, int64_t page_stride,
                                  int64_t n_pages, int page_size, const int32_t *table, int64_t table_stride,
                                  int table_rows, int max_pages, const int32_t *slots, const int32_t *cu_seqlens,
                                  const int64_t *kv_len, int n_seqs, void *stream);

/*
 * The best continuations of each group of `beams` rows of logits [groups * beams, vocab]:
 * of the candidates scores[b] + log_softmax(logits[b])[v] of its beams the `keep` greatest,
 * sorted, equal ones by beam, then by their logits, then by token.  ended[b] != 0: the beam's only candidate is its own score
 * with pad_token.  Logits and sums that are NaN or infinite are no candidates (and a row with a
 * logit of +inf or a score that is not finite has none): places without one hold score -inf,
 * parent -1, token -1.  Exponentials are of logits less the greatest one of their part of a row (8,192
 * logits), in fp32, and summed in fp32 2,048 at a time; these sums are joined, and candidates formed and
 * compared, in double precision.  A score below fp32's range is returned as -inf.
 *   out_scores fp32, out_parent int32 (a beam of the group), out_token int64: [groups, keep].
 *   beams, keep 1 .. SOPHIA_BEAMS.
 */
#define SOPHIA_BEAMS 64
size_t sophia_beam_select_workspace_size(int64_t rows, int vocab, int keep);
int sophia_beam_select(const void *logits, int64_t logits_stride, int dtype, int64_t rows, int vocab,
                       const float *scores, const uint8_t *ended, int64_t pad_token, int beams, int keep,
                       float *out_scores, int32_t *out_parent, int64_t *out_token, void *workspace,
                       size_t workspace_bytes, void *stream);

/*
 * Moves of cache slots, in place and as if all at once: slot dst[i] becomes what slot
 * src[i] was (int32, device), i < n <= SOPHIA_MOVES.  A move from or to a slot out of
 * [0, n_slots), or to itself, changes nothing; of several moves to one slot the last one
 * counts.  For each KDA layer its state [n_slots, state_elems] and conv history [n_slots,
 * conv_elems] (fp32, dense).  With cached[i] (int64, device), the tokens that move i takes along:
 *   mla[l]  : latents [n_slots, max_seq, rank] fp32 with slot_stride, positions below cached[i];
 *   table, pools[l] : the ids of the pages that cached[i] tokens fill, and the tokens of the page that they
 *             fill in part, from the source's page into the one that dst[i] has there.  The pages of
 *             different slots at that place are different ones.
 * The workspace holds the plan of the call.
 */
#define SOPHIA_MOVES 4096
#define SOPHIA_FORK_KDA 48
#define SOPHIA_FORK_MLA 24
size_t sophia_move_workspace_size(int n);
int sophia_cache_fork(const int32_t *src, const int32_t *dst, const int64_t *cached, int n, int n_slots,
                      float *const *states, int64_t state_elems, float *const *convs, int64_t conv_elems, int n_kda,
                      float *const *mla, int64_t slot_stride, int max_seq, int n_mla, void *const *pools,
                      int64_t page_stride, int64_t n_pages, int page_size, int n_pools, int32_t *table,
                      int64_t table_stride, int max_pages, int rank, int pool_dtype, void *workspace,
                      size_t workspace_bytes, void *stream);

/*
 * pages[dst[i]] = pages[src[i]] in every pool, under the same rules (in place, as if at once).
 */
int sophia_page_copy(const int32_t *src, const int32_t *dst, int n, void *const *pools, int n_pools,
                     int64_t page_stride, int64_t page_elems, int64_t n_pages, int dtype, void *workspace,
                     size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SOPHIA_PAGES_H */
