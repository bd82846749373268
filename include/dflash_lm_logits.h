/*
 * dflash_lm_logits.h — the LM head's logits in fp32, for an accept that something is to
 * change before it (dflash_logits.h).  Conventions (return codes, streams, no
 * allocation, no synchronisation) are those of dflash_gdn.h.
 *
 * logits[m][v] = hidden[m] . weight[v], the fp32 sums that dflash_lm_head_greedy_accept
 * (of a fragment-tiled weight: dflash_lm_head_greedy_accept_tiled) compares, to the bit:
 * their greedy tokens are the fused accept's.  hidden: bf16 [M, H], M <= 64, rows
 * hidden_row_stride elements apart; the weight and the limits are those of the two
 * accepts; logits: fp32, rows logits_row_stride elements apart (at least V), 4-byte
 * aligned.
 */
#ifndef DFLASH_LM_LOGITS_H
#define DFLASH_LM_LOGITS_H

#include "dflash_gdn.h"

#ifdef __cplusplus
extern "C" {
#endif

int dflash_lm_head_logits(const void* hidden, int64_t hidden_row_stride, const void* weight,
                          int64_t weight_row_stride, int H, int V, float* logits,
                          int64_t logits_row_stride, int M, void* stream);
int dflash_lm_head_logits_tiled(const void* hidden, int64_t hidden_row_stride, const void* weight_tiled,
                                int H, int V, float* logits, int64_t logits_row_stride, int M,
                                void* stream);

#ifdef __cplusplus
}
#endif
#endif
