// What the host side of qwen_b200_op_sample hands to its kernel.
#pragma once
#include "common.cuh"

namespace qb {

constexpr uint32_t SM_MAX_VOCAB = 524216;

struct SampleArgs {
    const uint16_t *logits;
    uint64_t stride;
    uint32_t rows, vocab;
    const float *temperature, *top_p, *min_p, *u;
    const uint32_t *top_k;
    uint32_t *tokens;
    float *probs;
    uint32_t part;  // 16-byte groups that each CTA of a row counts
    int unit;       // weights are whole multiples of 2^-unit
};
int launch_sample(SampleArgs a, cudaStream_t st);

}  // namespace qb
