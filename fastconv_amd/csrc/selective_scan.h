// Selective scan: what its kernels share.
//
//   dt = softplus(delta + delta_bias) or delta + delta_bias
//   h_t[n] = exp(dt A[n]) h_(t-1)[n] + dt x_t B_t[n],   y_t = (sum over n of C_t[n] h_t[n] + D x_t) * silu(z_t)        for each channel
//
// and backwards, with g = dy silu(z), G_t = dL/dh_t:
//   G_t[n] = C_t[n] g_t + exp(dt_(t+1) A[n]) G_(t+1)[n],   K_t[n] = G_t[n] exp(dt A[n]) h_(t-1)[n]
//   dx = dt sum of G B + D g,   d(dt) = x sum of G B + sum of K A,   dA = sum of dt K,   dB[n] = sum over channels of G dt x,   dC[n] = of g h,
//   dD = sum of g x,   dz = dy (C h + D x) silu'(z)
//
// A workgroup takes 64 channels (32 or 16 where there are more than 16 states) and walks over their tokens in tiles of 32.  Each channel has L lanes of
// S states: what all its states need of a token (dt, dt x, the gate) is formed once, by threads that lie along the channels, and reaches the lanes through LDS, as
// B and C do; so the inner loop is S states' exponentials and multiply-adds.
#pragma once

#include "selective_scan_forms.h"
#include "token_math.h"

struct fc_scan_run {
    const void *x, *delta, *b, *c, *z, *dy;
    const float *A, *D, *delta_bias;
    void *y, *dx, *ddelta, *dz;
    const float *state_in, *dstate_out;
    float *state_out, *dstate_in;
    const int32_t *lengths;
    float *parts;            // [B][segments][D][N]: what a segment adds to no state; then what enters it
    float *grads;            // the same of G: what a segment adds to none; then what comes from the tokens after it
    float *steps;            // [B][segments][D]: the sum of dt over a segment
    float *shared;           // [blocks][B][T][2][N]: what a workgroup's channels add to dB and dC
    float *sums;             // [B][walks][D][N + 2]: what a walk's tokens add to dA, dD and the gradient of delta_bias
    long T, segment;         // tokens
    int segments, per_walk, walks;      // segments that a workgroup takes one after another
    int B, channels, N, G;   // channels: D of the interface
    int per_group, blocks;   // channels of a group; workgroups side by side for all channels
    int softplus;
    long x_batch, x_token, delta_batch, delta_token, z_batch, z_token, y_batch, y_token;
    long b_batch, b_token, b_group, c_batch, c_token, c_group;
};

// selective_scan_<type>.hip.  ends: parts, steps and, if dy is there, grads of each segment.  answers: y and the last state, each segment from what
// enters it.  step: the same for a few tokens.  gradients: of each segment, from what enters it on both sides.
int fc_scan_ends_bf16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_ends_f16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_ends_f32(fc_context *ctx, const fc_scan_run &r);
int fc_scan_answers_bf16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_answers_f16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_answers_f32(fc_context *ctx, const fc_scan_run &r);
int fc_scan_step_bf16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_step_f16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_step_f32(fc_context *ctx, const fc_scan_run &r);
int fc_scan_gradients_bf16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_gradients_f16(fc_context *ctx, const fc_scan_run &r);
int fc_scan_gradients_f32(fc_context *ctx, const fc_scan_run &r);

__device__ __forceinline__ long fc_scan_length(const fc_scan_run &r, long b) {
    if (!r.lengths) return r.T;
    const long n = r.lengths[b];
    return n < 0 ? 0 : n > r.T ? r.T : n;
}

// A rate for powers of two.  Infinite ones become the largest number, so that a step of 0 leaves a state as it is.
__device__ __forceinline__ float fc_scan_rate(float a) {
    const float r = a * 1.44269504f;
    return r < -3.4028235e38f ? -3.4028235e38f : r > 3.4028235e38f ? 3.4028235e38f : r;
}
