/*
 * dflash_logits.h — what a request asks of the logits before a token is taken
 * from them: penalties for repeated tokens, biases and grammar masks.
 * Conventions (return codes, streams, no allocation, no synchronisation) are
 * those of dflash_gdn.h.
 *
 * A state of B sequences over a vocabulary of V tokens:
 *
 *   counts     int32 [B, V]   how often a token was generated (bits 0 .. 30);
 *                             the sign bit: the prompt has it
 *   known      uint32 [B, ceil(V / 32)]  bit v % 32 of word v / 32: token v has
 *                             a count or a bias.  Where the bit is 0 both are 0,
 *                             so that a pass over the logits reads V / 8 bytes
 *                             of a sequence's state and the few entries that
 *                             there are
 *   bias       fp32 [B, V]
 *   penalties  fp32 [B, 3]    repetition (> 0), presence, frequency
 *
 * Row i of a sequence's N rows knows the counted tokens and the draft tokens
 * 0 .. i - 1.  With c(v) the times v was generated, those drafts included, the
 * processed logit of token v is, every step in fp32,
 *
 *   l = logit
 *   l = l > 0 ? l / repetition : l * repetition  if c(v) > 0 or the prompt has v
 *   l = l - frequency * c(v) - presence          if c(v) > 0
 *   l = l + bias(v)
 *   l = -inf                                     if the mask's bit of v is 0
 *
 * A mask (bit v % 32 of word v / 32 set: v is allowed) overrides whatever the
 * logit is, a NaN too.
 */
#ifndef DFLASH_LOGITS_H
#define DFLASH_LOGITS_H

#include "dflash_gdn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Every array contiguous and 4-byte aligned. */
typedef struct {
  int32_t* counts;
  uint32_t* known;
  float* bias;
  float* penalties;
  int32_t B, V;
} dflash_logits_state;

/* Most rows of a sequence that draft tokens are counted for (N - 1 drafts). */
#define DFLASH_LOGITS_MAX_DRAFT 64
/* Most biases of one call. */
#define DFLASH_LOGITS_MAX_BIAS 4096

/* No counts and biases, penalties 1, 0, 0.  Only the known entries are written:
 * a state whose arrays are not yet those of a state is made with zeros. */
int dflash_logits_state_reset(const dflash_logits_state* state, void* stream);

/* Count tokens: sequence b's are tokens[b * row_stride .. + n), the first lens[b] of
 * them with lens (null: all).  Ids outside [0, V) are passed over.  prompt: the
 * prompt's sign bit is set; else each is counted once more. */
int dflash_logits_state_add(const dflash_logits_state* state, const int32_t* tokens, int64_t row_stride,
                            int n, const int32_t* lens, int prompt, void* stream);

/* bias(ids[b][j]) = values[b][j], j < n <= DFLASH_LOGITS_MAX_BIAS; of an id given
 * twice the last counts, ids outside [0, V) are passed over. */
int dflash_logits_state_set_bias(const dflash_logits_state* state, const int32_t* ids, int64_t ids_stride,
                                 const float* values, int64_t values_stride, int n, void* stream);

/* Processed logits [B, N, V] to out, rounded once to the logits' type (logits_dtype: a
 * dflash_gdn.h tag).  Strides in elements; a row's V entries are contiguous.  out may be
 * the logits themselves with the same strides: entries that nothing changes then keep their
 * values, and eights of a row (from a multiple of 8 on) that hold no masked and no known token
 * are not touched.  state null: only the mask.  draft [B, n_draft]: draft token i is known to the
 * rows from i + 1 on.  mask: words, batch and row stride in words (0: shared), or null. */
int dflash_logits_process(const void* logits, int logits_dtype, int64_t batch_stride, int64_t row_stride,
                          const dflash_logits_state* state, const int32_t* draft, int64_t draft_stride,
                          int n_draft, const uint32_t* mask, int64_t mask_batch_stride,
                          int64_t mask_row_stride, void* out, int64_t out_batch_stride,
                          int64_t out_row_stride, int B, int N, int V, void* stream);

/* dflash_greedy_accept of the processed logits, which are not stored: the greedy token of
 * a row is that of the largest fp32 value, the lowest on ties (a row that its mask leaves
 * nothing: token 0).  workspace: dflash_greedy_accept_processed_workspace_bytes(B, N, V)
 * bytes, 8-byte aligned. */
size_t dflash_greedy_accept_processed_workspace_bytes(int B, int N, int V);
int dflash_greedy_accept_processed(const void* logits, int logits_dtype, int64_t batch_stride,
                                   int64_t row_stride, const int32_t* draft, int64_t draft_stride,
                                   int n_draft, const dflash_logits_state* state, const uint32_t* mask,
                                   int64_t mask_batch_stride, int64_t mask_row_stride,
                                   int32_t* posterior, int32_t* matched, int32_t* bonus, int B, int N,
                                   int V, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
