/*
 * sera_logprobs.h - C ABI of what a program reads off rows of logits on MI355X
 * (gfx950): log probabilities of given tokens, the distribution's entropy and
 * its most likely tokens. The logits are those of the LM head
 * (q3_cuda_q4k_linear over the vocabulary) or any other rows.
 *
 * The conventions are those of sera_q4k.h: plain C types, device pointers, a
 * stream is a hipStream_t passed as void* (NULL = the null stream). The call
 * enqueues on the given stream, does not synchronize and allocates nothing, so
 * it can be captured into a graph. Return codes: 0 success, -1 invalid
 * arguments, -3 launch failed; sera_q4k_last_error() gives the message. No
 * other set-up call is needed.
 */
#ifndef SERA_LOGPROBS_H
#define SERA_LOGPROBS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SERA_LOGPROBS_MAX_TOP 64

/* Scratch for sera_logprobs with these sizes on the current device: what rows
 * that are split over workgroups leave (0: none is needed, or the arguments are
 * refused by the call as well). Not monotone in the rows: ask for every size
 * that is used and keep the largest, at most 0.3 MB on 256 compute units. */
size_t sera_logprobs_workspace_bytes(int rows, int vocab, int top);

/* Of each row x of logits ([rows][vocab] of `type`: 0 F32, 1 F16, 30 BF16,
 * GGUF's ids; `stride` elements from one row to the next, aligned as their
 * elements are), with log Z = log(sum_j e^x_j):
 *
 *   token_logprobs[r][i] = x[tokens[r][i]] - log Z     i < per_row
 *   entropy[r]           = log Z - sum_j p_j x_j       (nats, p_j = e^x_j / Z)
 *   top_ids[r][i], top_logprobs[r][i]                  i < top (0..64, <= vocab)
 *
 * the top tokens by falling logit, of equal ones the lower id first (-0 and 0
 * are equal). per_row may be 0, entropy NULL and top 0 for what is not wanted.
 * Logits of -inf are tokens of no probability: their log probability is -inf,
 * and they are among the top only where there are too few others. A token
 * outside 0..vocab-1 has log probability NaN. A row that holds a NaN or +inf,
 * or nothing but -inf, has no distribution: NaN everywhere, and top ids of -1.
 *
 * Sums are around a maximum, in fp32 of 16 elements and in 64 bits of those.
 * One or two launches; results repeat bit for bit. workspace: 16-byte aligned,
 * sera_logprobs_workspace_bytes(), used by one call at a time. */
int sera_logprobs(uint32_t type, const void *logits, int64_t stride, int rows, int vocab, const int32_t *tokens,
                  int per_row, float *token_logprobs, float *entropy, int top, int32_t *top_ids, float *top_logprobs,
                  void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif
