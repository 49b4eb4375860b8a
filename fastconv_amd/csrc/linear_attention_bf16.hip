// Linear attention in chunks: the kernels for bf16.
#include "linear_attention_chunk.h"

int fc_la_answer_bf16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    return la_launch<FC_BF16, true>(ctx, r, heads, segments, segment, parts);
}

int fc_la_state_bf16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    return la_launch<FC_BF16, false>(ctx, r, heads, segments, segment, parts);
}
