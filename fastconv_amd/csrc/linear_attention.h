// Linear attention with a decay for each head: what its kernels share.
//
//   S_t = l S_(t-1) + k_t v_t^T,   o_t = scale * S_t^T q_t,   l = exp(log_decay)
//
// The backward pass is made of the same recurrence.  With the gradient do of o and dS of the last state,
//   dq_t = scale * S_t do_t:                      the forward run over (do, v, k) from S_0^T
//   G_t = l G_(t+1) + scale * q_t do_t^T,  dk_t = G_t v_t,  dv_t = G_t^T k_t:   runs from the last token to the first over
//                                                 (v, do, q) and (k, q, do); the state enters as dS = l G_(T+1), and l G_1
//                                                 is the gradient of S_0
// So one run serves all: a direction, three operands with heads and strides of their own, a state that may be read and
// written transposed.  A forward run decays its state before it takes a token in, a backward one after it has answered.
#pragma once

#include "token_types.h"

struct fc_la_operand {
    const void *p;
    long batch, token, head;
    int share;               // heads that read one of this operand's heads
};

struct fc_la_run {
    fc_la_operand q, k, v;
    void *o;                 // in the tensors' type, or
    bool o_fp32;             // in fp32, where answers are added up afterwards
    long o_batch, o_token, o_head;
    const float *state_in;   // element (row, column) of head bh at bh*state_head + row*state_row + column*state_col
    float *state_out;
    long state_head, state_row, state_col;
    long part_row, part_col; // the same of the states that segments begin from
    bool parts_ready;        // which another run has left, transposed or not
    const float *log_decay;
    const int32_t *lengths;
    long T;
    int H, Dk, Dv;           // of this run: rows and columns of its state
    int reverse;
    float scale_in, scale_out;      // of what enters the state, of what leaves it
    bool wide;               // four channels of every operand lie within one access
};

// Wavefronts of 32 columns in a workgroup of a run with a state of Dk x Dv: two where the state has no more than 64 columns, if they have the registers to
// lay out its rows for each other; else four, half of which idle.  With two and four, 8 x 1225 tokens of 8 heads, each cut for its own: states of 32x32 in fp32
// 37 and 42 us (with the backward pass 131 and 146); 64x64 in fp32 71 and 55 (32 x 515 tokens of 32 heads 250 and 195), in bf16 36 and 39, in half 47 and 44 (212 and 266);
// 63x61, by single elements, in half 86 and 65 (64 x 515 tokens of 32 heads 575 and 454), in bf16 55 and 53; 128x64 in fp32 290 and 131, in half 150 and 69, in
// bf16 108 and 52.
static inline int fc_la_wavefronts(int dtype, int Dk, int Dv, bool wide) {
    return Dv <= 64 && (Dk <= 32 || (Dk <= 64 && (dtype == FC_BF16 || (dtype == FC_F16 && wide)))) ? 2 : 4;
}

// linear_attention_<type>.hip: `segments` parts of `segment` tokens of each of `heads` heads.  _state: the state that each but the
// last adds to none, to parts [heads][segments][Dk][Dv].  _answer: the answers; each segment begins from its state in parts, or, if it is the only
// one, from state_in.
int fc_la_state_bf16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts);
int fc_la_state_f16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts);
int fc_la_state_f32(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts);
int fc_la_answer_bf16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts);
int fc_la_answer_f16(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts);
int fc_la_answer_f32(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts);

__device__ __forceinline__ long fc_la_length(const fc_la_run &r, long b) {
    if (!r.lengths) return r.T;
    const long n = r.lengths[b];
    return n < 0 ? 0 : n > r.T ? r.T : n;
}

// exp(n * log_decay) in two parts, n >= 0: a decay's own rounding, the same at every step, would grow with their number
struct fc_la_power {
    float hi, lo;
    __device__ __forceinline__ fc_la_power(float log_decay, long n) {
        const double l = n ? exp((double)log_decay * (double)n) : 1.0;
        hi = (float)l;
        lo = (float)(l - hi);
    }
    __device__ __forceinline__ float times(float s) const { return __builtin_fmaf(hi, s, lo * s); }
};
