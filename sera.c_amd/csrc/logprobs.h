/*
 * logprobs.h - what the kernels of sera_logprobs take, and their launcher (internal).
 */
#ifndef LOGPROBS_H
#define LOGPROBS_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

struct logprobs_args {
    const void *logits;
    int64_t stride;
    int rows, vocab;
    const int32_t *tokens;
    int per_row;
    float *token_logprobs, *entropy;
    int top;
    int32_t *top_ids;
    float *top_logprobs;
    int splits;              /* workgroups of a row */
    size_t sums;             /* floats of the workspace in front of the lists */
    float *workspace;
};

int sera_logprobs_splits(int rows, int vocab, int cus);
size_t sera_logprobs_sums(int rows, int splits);
hipError_t sera_launch_logprobs(uint32_t type, const logprobs_args &p, hipStream_t s);

#endif
