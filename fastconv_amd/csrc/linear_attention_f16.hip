// Linear attention in chunks: the kernels for IEEE half.
#include "linear_attention_chunk.h"

int fc_la_answer_f16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    return la_launch<FC_F16, true>(ctx, r, heads, segments, segment, parts);
}

int fc_la_state_f16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    return la_launch<FC_F16, false>(ctx, r, heads, segments, segment, parts);
}
