// Linear attention in chunks: the kernels for fp32.
#include "linear_attention_chunk.h"

int fc_la_answer_f32(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    return la_launch<FC_F32, true>(ctx, r, heads, segments, segment, parts);
}

int fc_la_state_f32(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    return la_launch<FC_F32, false>(ctx, r, heads, segments, segment, parts);
}
