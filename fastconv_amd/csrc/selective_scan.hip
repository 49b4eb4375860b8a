// Selective scan: entry points, plan, and the kernels that join segments and sums.  See selective_scan.h for the formulas.
#include "selective_scan.h"

namespace {

constexpr int kThreads = 256;
constexpr long kMostThreads = 1l << 32;      // of a launch, not reached
constexpr int kMostStates = 64;
constexpr long kMostShared = 16384;      // workgroups of the sums of dB and dC
// Up to so many tokens run without tiles.  16 states, bf16, without and with: 64 sequences of 4096 channels, 1 token 11.8 us and 28.0, 4 tokens 18.4 and 29.1, 8
// tokens 33.1 and 31.7; one of 2048 channels, 4 tokens 5.4 and 5.9, 8 tokens 7.3 and 6.3.
constexpr long kMostSteps = 4;
// A sequence is cut where its channels leave the chip idle, and then into as many segments as fill it: a cut forms every state twice.  2048 tokens of 2048
// channels, 16 states, bf16: 8 sequences (1024 wavefronts) 268 us uncut and 236 in 8 segments, 11 of them 337 and 315 in 5, 12 of them 335 and 336.  One sequence of
// 12544 tokens: 219 us in 56 segments (8192 wavefronts), 229 in 31, 259 in 16; 4 of 3136 tokens 203 in 14, 216 in 8, 246 in 4, 405 uncut.
constexpr long kEnoughWavefronts = 1536, kWavefronts = 8192;
// A tile takes a lone workgroup about 4 us, two launches more about 8: 6 sequences of 288 channels, 16 states, tiles of one segment each and uncut: 4 tiles 17.6 and 20.4
// us, 7 tiles 18.9 and 32.7, 13 tiles 22.4 and 55.9 (32.7 in segments of three).
constexpr long kLeastTiles = 4;
// The join goes through the segments one after another, about 0.05 us each against 4 of a tile twice, so that a segment has about the square root of a 160th of the
// tiles at least.  One sequence of 64 channels, 16 states: 12544 tokens 43.8 us in 196 segments, 58.5 in 392 and 48.8 in 98; 100000 tokens 138, 221 (in 1563) and 127 (391).
constexpr long kTilesSquared = 160;
// Workgroups of the gradients' kernel, each of which leaves sums of dA: 4 sequences of 3136 tokens, 2048 channels, 16 states 733 us with 1024 of them, 682 with 2048
// and 693 with 4096; 8 of 2048 tokens, 1024 channels, 8 states 333, 329 and 336.
constexpr long kWorkgroupsBackward = 2048;

// What enters each segment, from what each adds to none.  Bound by the chain of segments, eight of which are read at once.  GRADS: from the last to the
// first, and what leaves the first is the gradient of the state before it.
template <bool GRADS>
__device__ __forceinline__ void join_segments(const fc_scan_run &r) {
    constexpr int AHEAD = 8;
    const long i = (long)blockIdx.x * kThreads + threadIdx.x, size = (long)r.channels * r.N, b = i / size, dn = i - b * size;
    if (b >= r.B) return;
    const long d = dn / r.N;
    const float rate = fc_scan_rate(r.A[dn]);
    float *p = (GRADS ? r.grads : r.parts) + b * r.segments * size + dn;
    const float *steps = r.steps + b * r.segments * r.channels + d, *given = GRADS ? r.dstate_out : r.state_in;
    float s = given ? given[i] : 0.f;
    // the segment whose own part nothing follows is not asked for it
    const int parts = GRADS ? r.segments : r.segments - 1;
    for (int first = 0; first < r.segments; first += AHEAD) {
        float add[AHEAD], dt[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const bool there = first + a < parts;
            const long at = GRADS ? r.segments - 1 - first - a : first + a;
            add[a] = there ? p[at * size] : 0.f;
            dt[a] = there ? steps[at * r.channels] : 0.f;
        }
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            if (first + a >= r.segments) break;
            const long at = GRADS ? r.segments - 1 - first - a : first + a;
            p[at * size] = s;
            s = __builtin_fmaf(__builtin_amdgcn_exp2f(rate * dt[a]), s, add[a]);
        }
    }
    if (GRADS && r.dstate_in) r.dstate_in[i] = s;
}

// States, and in the second row of workgroups gradients.
__global__ __launch_bounds__(kThreads) void fc_selective_scan_join_kernel(const fc_scan_run r) {
    if (blockIdx.y == 0) join_segments<false>(r);
    else join_segments<true>(r);
}

// Always in the same order: in the first workgroups dA, dD and the gradient of delta_bias from those of each walk, [D][N + 2] each; in the others dB and dC of a group from
// those of its workgroups.
template <int DT>
__global__ __launch_bounds__(kPartThreads) void fc_selective_scan_sums_kernel(const fc_scan_run r, float *dA, float *dD, float *dbias, unsigned first, void *db, void *dc,
                                                                              long values) {
    typedef typename fc_elem<DT>::type E;
    if (blockIdx.x < first) {
        long i;
        float s;
        if (!fc_sum_parts(r.sums, (long)r.B * r.walks, (long)r.channels * (r.N + 2), i, s)) return;
        const long d = i / (r.N + 2);
        const int n = (int)(i - d * (r.N + 2));
        if (n < r.N) {
            if (dA) dA[d * r.N + n] = s;
        } else if (n == r.N) {
            if (dD) dD[d] = s;
        } else if (dbias) {
            dbias[d] = s;
        }
        return;
    }
    const int per = r.blocks / r.G;
    const long block = (long)r.B * r.T * 2 * r.N;
    for (long i = (long)(blockIdx.x - first) * kPartThreads + threadIdx.x; i < values; i += (long)(gridDim.x - first) * kPartThreads) {      // [B][T][G][2][N]
        long rest = i / r.N;
        const int n = (int)(i - rest * r.N), half = (int)(rest & 1);
        rest >>= 1;
        const long bt = rest / r.G, g = rest - bt * r.G, b = bt / r.T, t = bt - b * r.T;
        const float *p = r.shared + g * per * block + (bt * 2 + half) * r.N + n;
        float s = 0.f;
        int k = 0;
        for (; k + 8 <= per; k += 8) {      // eight on their way at once
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = p[(k + u) * block];
#pragma unroll
            for (int u = 0; u < 8; u++) s += v[u];
        }
        for (; k < per; k++) s += p[k * block];
        if (half) ((E *)dc)[b * r.c_batch + t * r.c_token + g * r.c_group + n] = (E)s;
        else ((E *)db)[b * r.b_batch + t * r.b_token + g * r.b_group + n] = (E)s;
    }
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

bool shape_ok(const fc_selective_scan_shape *s) {
    if (!s || s->B < 1 || s->T < 1 || s->D < 1 || s->N < 1 || s->G < 1 || s->D % s->G || !fc_dtype_ok(s->dtype)) return false;
    const long strides[14] = {s->x_batch, s->x_token, s->delta_batch, s->delta_token, s->z_batch, s->z_token, s->b_batch,
                              s->b_token, s->b_group, s->c_batch, s->c_token, s->c_group, s->y_batch, s->y_token};
    for (long v : strides)
        if (v < 0) return false;
    return true;
}

bool same(const fc_selective_scan_plan &a, const fc_selective_scan_plan &b) {
    const fc_selective_scan_shape &s = a.shape, &t = b.shape;
    return s.B == t.B && s.T == t.T && s.D == t.D && s.N == t.N && s.G == t.G && s.dtype == t.dtype && s.softplus == t.softplus && s.x_batch == t.x_batch &&
           s.x_token == t.x_token && s.delta_batch == t.delta_batch && s.delta_token == t.delta_token && s.z_batch == t.z_batch && s.z_token == t.z_token &&
           s.b_batch == t.b_batch && s.b_token == t.b_token && s.b_group == t.b_group && s.c_batch == t.c_batch && s.c_token == t.c_token &&
           s.c_group == t.c_group && s.y_batch == t.y_batch && s.y_token == t.y_token && a.tiles == b.tiles && a.segments == b.segments &&
           a.walks_backward == b.walks_backward && a.ws_bytes == b.ws_bytes && a.ws_backward_bytes == b.ws_backward_bytes;
}

int check_plan(fc_context *ctx, const fc_selective_scan_plan *plan, const char *what) {
    fc_selective_scan_plan own;
    if (!plan || fc_selective_scan_make_plan(&plan->shape, &own) != FC_OK || !same(*plan, own)) return fail(ctx, FC_ERR_INVALID, what);
    return FC_OK;
}

int blocks_of(const fc_selective_scan_shape &s) {
    const int width = fc_scan_channels(s.N), per_group = s.D / s.G;
    return s.G * ((per_group + width - 1) / width);
}

size_t states_of(const fc_selective_scan_shape &s, long segments) { return (size_t)s.B * segments * s.D * s.N; }

fc_scan_run run_of(const fc_selective_scan_shape &s) {
    fc_scan_run r = {};
    r.B = s.B; r.T = s.T; r.channels = s.D; r.N = s.N; r.G = s.G; r.per_group = s.D / s.G; r.blocks = blocks_of(s); r.softplus = s.softplus;
    r.x_batch = s.x_batch; r.x_token = s.x_token; r.delta_batch = s.delta_batch; r.delta_token = s.delta_token;
    r.z_batch = s.z_batch; r.z_token = s.z_token; r.y_batch = s.y_batch; r.y_token = s.y_token;
    r.b_batch = s.b_batch; r.b_token = s.b_token; r.b_group = s.b_group; r.c_batch = s.c_batch; r.c_token = s.c_token; r.c_group = s.c_group;
    return r;
}

int join(fc_context *ctx, const fc_scan_run &r, bool grads) {
    const dim3 grid((unsigned)(((long)r.B * r.channels * r.N + kThreads - 1) / kThreads), grads ? 2 : 1);
    fc_selective_scan_join_kernel<<<grid, dim3(kThreads), 0, ctx->stream>>>(r);
    FC_LAUNCH_CHECK(ctx, "fc_selective_scan_join_kernel");
    return FC_OK;
}

}  // namespace

#define FC_SCAN_CALL(what, dtype, ...)                                                              \
    ((dtype) == FC_F32 ? fc_scan_##what##_f32(__VA_ARGS__) : (dtype) == FC_BF16 ? fc_scan_##what##_bf16(__VA_ARGS__) : fc_scan_##what##_f16(__VA_ARGS__))

extern "C" int fc_selective_scan_make_plan(const fc_selective_scan_shape *s, fc_selective_scan_plan *plan) {
    if (!plan || !shape_ok(s)) return FC_ERR_INVALID;
    if (s->N > kMostStates || s->T >= (1l << 31) || fc_count(s->B, s->D, 16 * kMostStates) < 0) return FC_ERR_UNSUPPORTED;
    const long tiles = (s->T + kScanTile - 1) / kScanTile, workgroups = (long)blocks_of(*s) * s->B;
    // threads of the widest launch: every tile of every channel, or every state
    if (fc_count(workgroups, tiles) < 0 || workgroups * tiles >= kMostThreads / kThreads || fc_count(s->B, s->D) >= kMostThreads / kMostStates ||
        fc_count(s->B * tiles, s->D, kScanTile * kMostStates) < 0)
        return FC_ERR_UNSUPPORTED;
    // the sums of the gradients of A, D and delta_bias take 32 threads for each, beside which there are workgroups for dB and dC
    if (fc_count(s->D, s->N + 2) >= kMostThreads / 32 - kMostShared * kPartThreads / 32) return FC_ERR_UNSUPPORTED;
    // a tile's offsets are 31 bits
    const long far = s->x_token | s->delta_token | s->z_token | s->b_token | s->c_token | s->y_token;
    if (s->T > 1 && far >= (1l << 24)) return FC_ERR_UNSUPPORTED;
    *plan = {};
    plan->shape = *s;
    plan->tiles = s->T > kMostSteps ? (int)tiles : 0;
    plan->segments = 1;
    const long wavefronts = workgroups * (kScanThreads / 64);
    if (tiles >= kLeastTiles && wavefronts < kEnoughWavefronts) {
        long least = 1;
        while (least * least * kTilesSquared < tiles) least++;
        const long segments = kWavefronts / wavefronts < tiles ? kWavefronts / wavefronts : tiles, even = (tiles + segments - 1) / segments;
        const long per = even > least ? even : least;
        plan->segments = (int)((tiles + per - 1) / per);
    }
    if (plan->segments > 1) plan->ws_bytes = (states_of(*s, plan->segments) + (size_t)s->B * plan->segments * s->D) * sizeof(float);
    long walks = (kWorkgroupsBackward + workgroups - 1) / workgroups;
    if (walks > tiles) walks = tiles;
    const long per_walk = (tiles + walks - 1) / walks;
    plan->walks_backward = (int)((tiles + per_walk - 1) / per_walk);
    plan->ws_backward_bytes = (2 * states_of(*s, tiles) + (size_t)s->B * tiles * s->D + (size_t)blocks_of(*s) * s->B * s->T * 2 * s->N +
                               (size_t)s->B * plan->walks_backward * s->D * (s->N + 2)) * sizeof(float);
    return FC_OK;
}

extern "C" int fc_selective_scan(fc_context *ctx, const fc_selective_scan_plan *plan, const void *x_dev, const void *delta_dev, const float *A_dev,
                                 const void *B_dev, const void *C_dev, const float *D_dev, const void *z_dev, const float *delta_bias_dev, void *y_dev,
                                 const float *state_in_dev, float *state_out_dev, const int32_t *lengths_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_selective_scan: not a plan of fc_selective_scan_make_plan")) return FC_ERR_INVALID;
    const fc_selective_scan_shape &s = plan->shape;
    if (!x_dev || !delta_dev || !A_dev || !B_dev || !C_dev || !y_dev || (!ws_dev && plan->ws_bytes))
        return fail(ctx, FC_ERR_INVALID, "fc_selective_scan: null pointer");
    if ((((uint64_t)x_dev | (uint64_t)delta_dev | (uint64_t)B_dev | (uint64_t)C_dev | (uint64_t)z_dev | (uint64_t)y_dev) & (fc_elem_size(s.dtype) - 1)) ||
        (((uint64_t)A_dev | (uint64_t)D_dev | (uint64_t)delta_bias_dev | (uint64_t)state_in_dev | (uint64_t)state_out_dev | (uint64_t)lengths_dev |
          (uint64_t)ws_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_selective_scan: unaligned pointer");
    if (!fc_apart({{s.B, s.y_batch}, {s.T, s.y_token}}, s.D)) return fail(ctx, FC_ERR_INVALID, "fc_selective_scan: tokens of y overlap");
    fc_scan_run r = run_of(s);
    r.x = x_dev; r.delta = delta_dev; r.A = A_dev; r.b = B_dev; r.c = C_dev; r.D = D_dev; r.z = z_dev; r.delta_bias = delta_bias_dev; r.y = y_dev;
    r.state_in = state_in_dev; r.state_out = state_out_dev; r.lengths = lengths_dev;
    const fc_device_scope on(ctx);
    if (!plan->tiles) return FC_SCAN_CALL(step, s.dtype, ctx, r);
    const long tiles = (s.T + kScanTile - 1) / kScanTile, per = (tiles + plan->segments - 1) / plan->segments;
    r.segments = plan->segments;
    r.segment = per * kScanTile;
    r.per_walk = 1;
    if (r.segments > 1) {
        r.parts = (float *)ws_dev;
        r.steps = r.parts + states_of(s, r.segments);
        r.walks = r.segments - 1;      // nothing follows the last
        int rc = FC_SCAN_CALL(ends, s.dtype, ctx, r);
        if (rc || (rc = join(ctx, r, false))) return rc;
    }
    r.walks = r.segments;
    return FC_SCAN_CALL(answers, s.dtype, ctx, r);
}

extern "C" int fc_selective_scan_backward(fc_context *ctx, const fc_selective_scan_plan *plan, const void *dy_dev, const void *x_dev,
                                          const void *delta_dev, const float *A_dev, const void *B_dev, const void *C_dev, const float *D_dev,
                                          const void *z_dev, const float *delta_bias_dev, void *dx_dev, void *ddelta_dev, float *dA_dev, void *dB_dev,
                                          void *dC_dev, float *dD_dev, void *dz_dev, float *ddelta_bias_dev, const float *state_in_dev,
                                          const float *dstate_out_dev, float *dstate_in_dev, const int32_t *lengths_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_selective_scan_backward: not a plan of fc_selective_scan_make_plan")) return FC_ERR_INVALID;
    const fc_selective_scan_shape &s = plan->shape;
    if (!dy_dev || !x_dev || !delta_dev || !A_dev || !B_dev || !C_dev || !dx_dev || !ddelta_dev || !dB_dev || !dC_dev || (z_dev && !dz_dev) || !ws_dev)
        return fail(ctx, FC_ERR_INVALID, "fc_selective_scan_backward: null pointer");
    const uint64_t addr = (uint64_t)dy_dev | (uint64_t)x_dev | (uint64_t)delta_dev | (uint64_t)B_dev | (uint64_t)C_dev | (uint64_t)z_dev |
                          (uint64_t)dx_dev | (uint64_t)ddelta_dev | (uint64_t)dB_dev | (uint64_t)dC_dev | (uint64_t)dz_dev;
    const uint64_t floats = (uint64_t)A_dev | (uint64_t)D_dev | (uint64_t)delta_bias_dev | (uint64_t)dA_dev | (uint64_t)dD_dev | (uint64_t)ddelta_bias_dev |
                            (uint64_t)state_in_dev | (uint64_t)dstate_out_dev | (uint64_t)dstate_in_dev | (uint64_t)lengths_dev | (uint64_t)ws_dev;
    if ((addr & (fc_elem_size(s.dtype) - 1)) || (floats & 3)) return fail(ctx, FC_ERR_INVALID, "fc_selective_scan_backward: unaligned pointer");
    if (!fc_apart({{s.B, s.x_batch}, {s.T, s.x_token}}, s.D) || !fc_apart({{s.B, s.delta_batch}, {s.T, s.delta_token}}, s.D) ||
        (z_dev && !fc_apart({{s.B, s.z_batch}, {s.T, s.z_token}}, s.D)) || !fc_apart({{s.B, s.b_batch}, {s.T, s.b_token}, {s.G, s.b_group}}, s.N) ||
        !fc_apart({{s.B, s.c_batch}, {s.T, s.c_token}, {s.G, s.c_group}}, s.N))
        return fail(ctx, FC_ERR_INVALID, "fc_selective_scan_backward: tokens of a gradient overlap");
    fc_scan_run r = run_of(s);
    r.dy = dy_dev; r.x = x_dev; r.delta = delta_dev; r.A = A_dev; r.b = B_dev; r.c = C_dev; r.D = D_dev; r.z = z_dev; r.delta_bias = delta_bias_dev;
    r.dx = dx_dev; r.ddelta = ddelta_dev; r.dz = dz_dev;
    r.state_in = state_in_dev; r.dstate_out = dstate_out_dev; r.dstate_in = dstate_in_dev; r.lengths = lengths_dev;
    const long tiles = (s.T + kScanTile - 1) / kScanTile;
    r.segments = (int)tiles;
    r.segment = kScanTile;
    r.walks = plan->walks_backward;
    r.per_walk = (int)((tiles + r.walks - 1) / r.walks);
    r.parts = (float *)ws_dev;
    r.grads = r.parts + states_of(s, tiles);
    r.steps = r.grads + states_of(s, tiles);
    r.shared = r.steps + (size_t)s.B * tiles * s.D;
    r.sums = r.shared + (size_t)r.blocks * s.B * s.T * 2 * s.N;
    const fc_device_scope on(ctx);
    int rc = FC_SCAN_CALL(ends, s.dtype, ctx, r);
    if (rc || (rc = join(ctx, r, true))) return rc;
    rc = FC_SCAN_CALL(gradients, s.dtype, ctx, r);
    if (rc) return rc;
    const long values = (long)s.B * s.T * s.G * 2 * s.N, want = (values + kPartThreads - 1) / kPartThreads;
    const unsigned first = dA_dev || dD_dev || ddelta_bias_dev ? (unsigned)(((long)s.D * (s.N + 2) + kPartValues - 1) / kPartValues) : 0;
    const auto sums = s.dtype == FC_F32    ? fc_selective_scan_sums_kernel<FC_F32>
                      : s.dtype == FC_BF16 ? fc_selective_scan_sums_kernel<FC_BF16>
                                           : fc_selective_scan_sums_kernel<FC_F16>;
    sums<<<dim3(first + (unsigned)(want < kMostShared ? want : kMostShared)), dim3(kPartThreads), 0, ctx->stream>>>(r, dA_dev, dD_dev, ddelta_bias_dev, first, dB_dev, dC_dev, values);
    FC_LAUNCH_CHECK(ctx, "fc_selective_scan_sums_kernel");
    return FC_OK;
}
