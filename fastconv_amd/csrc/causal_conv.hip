// Short causal convolution of each channel over the tokens of a sequence, channels last, with its activation:
//
//   z_t = bias + sum over j of w[j] x_(t - taps + 1 + j),   y_t = act(z_t);   rows before the first are the state
//   dz = dy act'(z),   dx_t = sum over j of w[j] dz_(t + taps - 1 - j),   dw[j] = sum over t of dz_t x_(t - taps + 1 + j),   dbias = sum of dz
//
// Bound by memory: 2 * taps operations a value against 4 bytes read and written in 16-bit types.  A thread walks down the tokens of a few
// neighbouring channels with the last rows in registers, so that every row is read once; sequences are cut into walks to fill the chip, each of
// which reads the taps - 1 rows before its own (backward: and after) once more.  4 x 3136 tokens of 2048 channels, four taps, bf16: 24 to 28 us (103 MB, about
// 4 TB/s), gradients 37 to 41 us (154 MB) and 4.2 for the sums of the walks' parts.
#include <type_traits>

#include "token_math.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMostTaps = 8;
// Channels of a thread, one access wherever they begin; one where there are fewer.  4 x 3136 tokens of 2048 channels, bf16: 24.2 us with two, 24.8 with one, 24.4
// with four, 32 sequences 183, 215 and 204, gradients of 4 40.9, 41.8 and 59.0.
constexpr int kChannels = 2;
// Tokens read before the first is used.  Of eight: 24.7 us for 24.2, gradients 53.5 for 40.9.
constexpr int kAhead = 4, kAheadBackward = 4;
// Threads that fill the chip: a sequence is cut until there are as many, into walks of some tokens at least.  With half and with twice as many: 31.2 and 25.1 us,
// gradients 50.1 and 48.0.
constexpr long kFill = 4096 * 64;

struct conv_params {
    const void *x, *dy, *state_in, *dstate_out;
    void *y, *state_out, *dstate_in;      // y: or dx
    const float *w, *bias;
    float *part;             // backward: [B * walks][taps + 1][C], the sums of dw and, last, dbias
    const int32_t *lengths;
    long T, walk;            // tokens of a sequence and of a walk
    int B, C, walks, act;
    fc_fastdiv by_columns, by_walks;
    long x_batch, x_token, y_batch, y_token;

    __device__ __forceinline__ int length(long b) const {
        const int n = lengths ? lengths[b] : (int)T;
        return n < 0 ? 0 : n > T ? (int)T : n;
    }
};

// What a thread walks over: channels c.. of sequence b, tokens t0 to t1.
struct conv_place {
    int c, skip, walk;       // the last thread of a row begins where its access ends with the row, and leaves out what its neighbour has
    long b;
    int t0, t1, len;
    bool none;
    __device__ __forceinline__ conv_place(const conv_params &p, int columns, int vec) {
        const uint32_t i = blockIdx.x * kThreads + threadIdx.x, row = fc_div(i, p.by_columns);
        none = row >= (uint32_t)(p.B * p.walks);
        const int from = (int)(i - row * columns) * vec;
        c = from + vec <= p.C ? from : p.C - vec;
        skip = from - c;
        b = fc_div(row, p.by_walks);
        walk = (int)(row - b * p.walks);
        t0 = (int)(walk * p.walk);
        t1 = (int)(t0 + p.walk < p.T ? t0 + p.walk : p.T);
        len = none ? 0 : p.length(b);
    }
};

// Some rows from token t on: N of them, or as many as there are tokens.  A row that is not there reads the first, without a branch of its own, which would keep
// all loads before it waiting.
template <int N, class V, class E>
__device__ __forceinline__ void read_rows(V (&to)[N], const E *first, const E *row, long token, int t, int len) {
    if (t + N <= len) {
#pragma unroll
        for (int u = 0; u < N; u++) __builtin_memcpy(&to[u], row + u * token, sizeof(V));
    } else {
#pragma unroll
        for (int u = 0; u < N; u++) __builtin_memcpy(&to[u], t + u < len ? row + u * token : first, sizeof(V));
    }
}

// The rows before token t of a window: those of the state, or zeros, before the first token.
template <int N, class V, class E>
__device__ __forceinline__ void read_before(V (&to)[N], const E *first, const E *state, long token, int C, int taps, int t, int len) {
    const V zeros = {};
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int row = t - N + i;
        const bool early = row < 0 && state && row >= 1 - taps, there = early || (row >= 0 && row < len);
        __builtin_memcpy(&to[i], early ? state + (long)(row + taps - 1) * C : first + (there ? row * token : 0), sizeof(V));
        if (!there) to[i] = zeros;
    }
}

// The window moves on by the N rows of `now`.
template <int N, int W, class V>
__device__ __forceinline__ void move_on(V (&window)[W], const V (&now)[N]) {
#pragma unroll
    for (int i = 0; i < W; i++) window[i] = i + N < W ? window[i + N < W ? i + N : 0] : now[i + N < W ? 0 : i + N - W];
}

template <class V, class E>
__device__ __forceinline__ void store(E *to, const V &v, int skip, bool whole) {      // whole: no thread of the launch leaves anything out
    if (whole || !skip) {
        __builtin_memcpy(to, &v, sizeof v);
        return;
    }
#pragma unroll
    for (int i = 1; i < (int)(sizeof(V) / sizeof(E)); i++)
        if (i >= skip) to[i] = v.v[i];
}

// Weights by distance: back[m] belongs to the row m tokens back.
template <int DT, int VEC, int TAPS>
__global__ __launch_bounds__(kThreads) void fc_causal_conv_kernel(const conv_params p, int columns) {
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    const conv_place at(p, columns, VEC);
    if (at.none) return;
    const E *x = (const E *)p.x + at.b * p.x_batch + at.c, *before = (const E *)p.state_in + at.b * (TAPS - 1) * p.C + at.c;
    E *y = (E *)p.y + at.b * p.y_batch + at.c;
    float back[VEC][TAPS], bias[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        bias[v] = p.bias ? p.bias[at.c + v] : 0.f;
#pragma unroll
        for (int m = 0; m < TAPS; m++) back[v][m] = p.w[(long)(at.c + v) * TAPS + TAPS - 1 - m];
    }
    V window[TAPS - 1], now[kAhead], next[kAhead];
    const bool whole = p.C % VEC == 0;
    read_before(window, x, p.state_in ? before : nullptr, p.x_token, p.C, TAPS, at.t0, at.len);
    const E *row = x + at.t0 * p.x_token;
    E *to = y + at.t0 * p.y_token;
    read_rows(next, x, row, p.x_token, at.t0, at.len);
    for (int t = at.t0; t < at.t1; t += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) now[u] = next[u];
        row += kAhead * p.x_token;
        if (t + kAhead < at.t1) read_rows(next, x, row, p.x_token, t + kAhead, at.len);
        auto results = [&](auto edge) __attribute__((always_inline)) {      // edge: some of the tokens are not there, or another walk's
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                V out;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    float z = bias[v];
#pragma unroll
                    for (int m = TAPS - 1; m >= 0; m--)
                        z = __builtin_fmaf(back[v][m], u >= m ? now[u >= m ? u - m : 0].get(v) : window[u >= m ? 0 : TAPS - 1 + u - m].get(v), z);
                    if (p.act == FC_ACT_SILU) z = fc_silu(z);
                    out.set(v, edge && t + u >= at.len ? 0.f : z);
                }
                if (!edge || t + u < at.t1) store(to + u * p.y_token, out, at.skip, whole);
            }
        };
        if (t + kAhead <= (at.len < at.t1 ? at.len : at.t1)) results(std::false_type());
        else results(std::true_type());
        to += kAhead * p.y_token;
        move_on(window, now);
    }
    // The last rows, by whoever read the first: the state may be written over the one before.  Row i lies at or before what it is read from.
    if (at.walk == 0 && p.state_out) {
        E *after = (E *)p.state_out + at.b * (TAPS - 1) * p.C + at.c;
        for (int i = 0; i < TAPS - 1; i++) {
            V last[1];
            read_before(last, x, p.state_in ? before : nullptr, p.x_token, p.C, TAPS, at.len - (TAPS - 1) + i + 1, at.len);
            store(after + (long)i * p.C, last[0], at.skip, whole);
        }
    }
}

// Four wavefronts a SIMD: three, which 133 registers at four taps would leave, take 50 us for 41.  More taps spill there: seven 60 us with the registers that they need, 244 with 128.
template <int DT, int VEC, int TAPS>
__global__ __launch_bounds__(kThreads, TAPS <= 4 ? 4 : 2) void fc_causal_conv_gradient_kernel(const conv_params p, int columns) {
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    const conv_place at(p, columns, VEC);
    if (at.none) return;
    const E *x = (const E *)p.x + at.b * p.x_batch + at.c, *before = (const E *)p.state_in + at.b * (TAPS - 1) * p.C + at.c;
    const E *dy = (const E *)p.dy + at.b * p.y_batch + at.c, *dlast = (const E *)p.dstate_out + at.b * (TAPS - 1) * p.C + at.c;
    E *dx = (E *)p.y + at.b * p.x_batch + at.c, *dfirst = (E *)p.dstate_in + at.b * (TAPS - 1) * p.C + at.c;
    float back[VEC][TAPS], bias[VEC], dback[VEC][TAPS], dbias[VEC], dz[VEC][TAPS];      // dz: of the last tokens, the newest last
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        bias[v] = p.bias ? p.bias[at.c + v] : 0.f;
        dbias[v] = 0.f;
#pragma unroll
        for (int m = 0; m < TAPS; m++) {
            back[v][m] = p.w[(long)(at.c + v) * TAPS + TAPS - 1 - m];
            dback[v][m] = dz[v][m] = 0.f;
        }
    }
    constexpr int AHEAD = kAheadBackward;
    V window[TAPS - 1], now[AHEAD], grads[AHEAD], next[AHEAD], more_grads[AHEAD];
    const bool whole = p.C % VEC == 0;
    const V zeros = {};
    read_before(window, x, p.state_in ? before : nullptr, p.x_token, p.C, TAPS, at.t0, at.len);
    const E *row = x + at.t0 * p.x_token, *from = dy + at.t0 * p.y_token;
    E *to = dx + ((long)at.t0 - (TAPS - 1)) * p.x_token;      // of row t - (TAPS - 1), whose gradient is whole once dz_t is there:
    const int end = at.t1 + TAPS - 1;                         // TAPS - 1 tokens past the walk's own
    read_rows(next, x, row, p.x_token, at.t0, at.len);
    read_rows(more_grads, dy, from, p.y_token, at.t0, at.len);
    for (int t = at.t0; t < end; t += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            now[u] = next[u];
            grads[u] = more_grads[u];
        }
        row += AHEAD * p.x_token;
        from += AHEAD * p.y_token;
        if (t + AHEAD < end) {
            read_rows(next, x, row, p.x_token, t + AHEAD, at.len);
            read_rows(more_grads, dy, from, p.y_token, t + AHEAD, at.len);
        }
        auto results = [&](auto edge) __attribute__((always_inline)) {      // edge: some of the tokens or rows are not there, or another walk's, or in the state
            auto x_back = [&](int u, int m, int v) __attribute__((always_inline)) { return u >= m ? now[u >= m ? u - m : 0].get(v) : window[u >= m ? 0 : TAPS - 1 + u - m].get(v); };
            float gs[AHEAD][VEC];
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
#pragma unroll
                for (int v = 0; v < VEC; v++) gs[u][v] = grads[u].get(v);
            if (p.act == FC_ACT_SILU)      // one branch for all of them
#pragma unroll
                for (int u = 0; u < AHEAD; u++)
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        float z = bias[v];
#pragma unroll
                        for (int m = TAPS - 1; m >= 0; m--) z = __builtin_fmaf(back[v][m], x_back(u, m, v), z);
                        gs[u][v] *= fc_silu_slope(z);
                    }
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const bool there = !edge || t + u < at.len, mine = !edge || (there && t + u < at.t1);
                const int r = t + u - (TAPS - 1), last = r - (at.len - (TAPS - 1));      // last: row of the state after the last token
                V more = zeros, out;
                const bool wanted = !edge || r >= at.t0 || (at.walk == 0 && r >= 1 - TAPS && p.dstate_in);
                if (edge && p.dstate_out && wanted && last >= 0 && last < TAPS - 1) __builtin_memcpy(&more, dlast + (long)last * p.C, sizeof more);
#pragma unroll
                for (int v = 0; v < VEC; v++) {
#pragma unroll
                    for (int j = 0; j < TAPS - 1; j++) dz[v][j] = dz[v][j + 1];
                    float g = gs[u][v];
                    if (!there) g = 0.f;      // what was read in place of rows that are not there may be anything
                    dz[v][TAPS - 1] = g;
                    if (mine) {
                        dbias[v] += g;
#pragma unroll
                        for (int m = 0; m < TAPS; m++)
                            dback[v][m] = __builtin_fmaf(g, x_back(u, m, v), dback[v][m]);
                    }
                    float s = edge ? more.get(v) : 0.f;
#pragma unroll
                    for (int m = 0; m < TAPS; m++)
                        s = __builtin_fmaf(back[v][m], dz[v][m], s);      // dz of row r + m
                    out.set(v, edge && r >= at.len ? 0.f : s);
                }
                if (!edge || (t + u < end && r >= at.t0)) store(to + u * p.x_token, out, at.skip, whole);
                else if (t + u < end && r < 0 && wanted) store(dfirst + (long)(r + TAPS - 1) * p.C, out, at.skip, whole);
            }
        };
        const int inside = at.len < at.t1 ? at.len : at.t1;      // rows of the state after the last token come later
        if (t + AHEAD <= inside && t - (TAPS - 1) >= at.t0) results(std::false_type());
        else results(std::true_type());
        to += AHEAD * p.x_token;
        move_on(window, now);
    }
    if (!p.part) return;
    float *part = p.part + (at.b * p.walks + at.walk) * (TAPS + 1) * p.C + at.c;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        if (v < at.skip) continue;
#pragma unroll
        for (int m = 0; m < TAPS; m++)
            part[(long)(TAPS - 1 - m) * p.C + v] = dback[v][m];
        part[(long)TAPS * p.C + v] = dbias[v];
    }
}

// dw and dbias from the walks' sums, [taps + 1][C] each.
__global__ __launch_bounds__(kPartThreads) void fc_causal_conv_sum_kernel(const float *part, float *dw, float *dbias, int parts, int C, int taps) {
    long i;
    float s;
    if (!fc_sum_parts(part, parts, (long)(taps + 1) * C, i, s)) return;
    const int j = (int)(i / C), c = (int)(i - (long)j * C);
    if (j == taps) {
        if (dbias) dbias[c] = s;
    } else if (dw) {
        dw[(long)c * taps + j] = s;
    }
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

bool same(const fc_causal_conv_plan &a, const fc_causal_conv_plan &b) {
    const fc_causal_conv_shape &s = a.shape, &t = b.shape;
    return s.B == t.B && s.T == t.T && s.C == t.C && s.taps == t.taps && s.dtype == t.dtype && s.act == t.act && s.x_batch == t.x_batch &&
           s.x_token == t.x_token && s.y_batch == t.y_batch && s.y_token == t.y_token && a.walks == b.walks &&
           a.walks_backward == b.walks_backward && a.ws_backward_bytes == b.ws_backward_bytes;
}

int check_plan(fc_context *ctx, const fc_causal_conv_plan *plan, const char *what) {
    fc_causal_conv_plan own;
    if (!plan || fc_causal_conv_make_plan(&plan->shape, &own) != FC_OK || !same(*plan, own)) return fail(ctx, FC_ERR_INVALID, what);
    return FC_OK;
}

int channels_of(const fc_causal_conv_shape &s) { return s.C < kChannels ? 1 : kChannels; }
int columns_of(const fc_causal_conv_shape &s) { return (s.C + channels_of(s) - 1) / channels_of(s); }

// Walks of `least` tokens or more.  They hold a window at least: only the first reads the state, which it may write over.
long walks_of(const fc_causal_conv_shape *s, int least) {
    const long rows = (long)columns_of(*s) * s->B, most = s->T > least ? s->T / least : 1;
    long walks = (kFill + rows - 1) / rows;
    if (walks > most) walks = most;
    const long walk = (s->T + walks - 1) / walks;
    return (s->T + walk - 1) / walk;
}

template <int DT, int VEC, class F>
void with_taps(int taps, F launch) {
    using std::integral_constant;
    typedef integral_constant<int, DT> dt;
    typedef integral_constant<int, VEC> vec;
    if (taps == 2) launch(dt(), vec(), integral_constant<int, 2>());
    else if (taps == 3) launch(dt(), vec(), integral_constant<int, 3>());
    else if (taps == 4) launch(dt(), vec(), integral_constant<int, 4>());
    else if (taps == 5) launch(dt(), vec(), integral_constant<int, 5>());
    else if (taps == 6) launch(dt(), vec(), integral_constant<int, 6>());
    else if (taps == 7) launch(dt(), vec(), integral_constant<int, 7>());
    else launch(dt(), vec(), integral_constant<int, 8>());
}

template <class F>
void with_kernel(const fc_causal_conv_shape &s, F launch) {
    const bool one = channels_of(s) == 1;
    if (s.dtype == FC_F32) return one ? with_taps<FC_F32, 1>(s.taps, launch) : with_taps<FC_F32, kChannels>(s.taps, launch);
    if (s.dtype == FC_BF16) return one ? with_taps<FC_BF16, 1>(s.taps, launch) : with_taps<FC_BF16, kChannels>(s.taps, launch);
    return one ? with_taps<FC_F16, 1>(s.taps, launch) : with_taps<FC_F16, kChannels>(s.taps, launch);
}

conv_params params_of(const fc_causal_conv_shape &s, int walks) {
    conv_params p = {};
    p.B = s.B; p.T = s.T; p.C = s.C; p.act = s.act;
    p.walks = walks;
    p.walk = (s.T + walks - 1) / walks;
    p.by_columns = fc_make_fastdiv((uint32_t)columns_of(s));
    p.by_walks = fc_make_fastdiv((uint32_t)walks);
    p.x_batch = s.x_batch; p.x_token = s.x_token; p.y_batch = s.y_batch; p.y_token = s.y_token;
    return p;
}

}  // namespace

extern "C" int fc_causal_conv_make_plan(const fc_causal_conv_shape *s, fc_causal_conv_plan *plan) {
    if (!plan || !s || s->B < 1 || s->T < 1 || s->C < 1 || s->taps < 2 || !fc_dtype_ok(s->dtype)) return FC_ERR_INVALID;
    if (s->act != FC_ACT_NONE && s->act != FC_ACT_SILU) return s->act < FC_ACT_NONE || s->act > FC_ACT_GELU ? FC_ERR_INVALID : FC_ERR_UNSUPPORTED;
    if (s->x_batch < 0 || s->x_token < 0 || s->y_batch < 0 || s->y_token < 0) return FC_ERR_INVALID;
    // tokens are counted in 32 bits, past the last; the sums of dw and dbias take 32 threads for each of (taps + 1) * C
    if (s->taps > kMostTaps || s->T > (1l << 30) || s->C > (1 << 23) || fc_count(s->B, s->C) < 0 || fc_count(s->B, s->C) >= (1l << 30)) return FC_ERR_UNSUPPORTED;
    *plan = {};
    plan->shape = *s;
    plan->walks = (int)walks_of(s, s->taps - 1 > kAhead ? s->taps - 1 : kAhead);
    plan->walks_backward = (int)walks_of(s, 4 * s->taps);
    plan->ws_backward_bytes = (size_t)s->B * plan->walks_backward * (s->taps + 1) * s->C * sizeof(float);
    return FC_OK;
}

extern "C" int fc_causal_conv(fc_context *ctx, const fc_causal_conv_plan *plan, const void *x_dev, const float *w_dev, const float *bias_dev,
                              void *y_dev, const void *state_in_dev, void *state_out_dev, const int32_t *lengths_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_causal_conv: not a plan of fc_causal_conv_make_plan")) return FC_ERR_INVALID;
    const fc_causal_conv_shape &s = plan->shape;
    if (!x_dev || !w_dev || !y_dev) return fail(ctx, FC_ERR_INVALID, "fc_causal_conv: null pointer");
    const uint64_t addr = (uint64_t)x_dev | (uint64_t)y_dev | (uint64_t)state_in_dev | (uint64_t)state_out_dev;
    if ((addr & (fc_elem_size(s.dtype) - 1)) || (((uint64_t)w_dev | (uint64_t)bias_dev | (uint64_t)lengths_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_causal_conv: unaligned pointer");
    if (!fc_apart({{s.B, s.y_batch}, {s.T, s.y_token}}, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_causal_conv: tokens of y overlap");
    const int columns = columns_of(s);
    conv_params p = params_of(s, plan->walks);
    p.x = x_dev; p.w = w_dev; p.bias = bias_dev; p.y = y_dev; p.state_in = state_in_dev; p.state_out = state_out_dev; p.lengths = lengths_dev;
    const unsigned blocks = (unsigned)(((long)s.B * p.walks * columns + kThreads - 1) / kThreads);
    const fc_device_scope on(ctx);
    with_kernel(s, [&](auto dt, auto v, auto taps) {
        fc_causal_conv_kernel<decltype(dt)::value, decltype(v)::value, decltype(taps)::value><<<dim3(blocks), dim3(kThreads), 0, ctx->stream>>>(p, columns);
    });
    FC_LAUNCH_CHECK(ctx, "fc_causal_conv_kernel");
    return FC_OK;
}

extern "C" int fc_causal_conv_backward(fc_context *ctx, const fc_causal_conv_plan *plan, const void *dy_dev, const void *x_dev, const float *w_dev,
                                       const float *bias_dev, void *dx_dev, float *dw_dev, float *dbias_dev, const void *state_in_dev,
                                       const void *dstate_out_dev, void *dstate_in_dev, const int32_t *lengths_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_causal_conv_backward: not a plan of fc_causal_conv_make_plan")) return FC_ERR_INVALID;
    const fc_causal_conv_shape &s = plan->shape;
    const bool sums = dw_dev || dbias_dev;
    if (!dy_dev || !x_dev || !w_dev || !dx_dev || (sums && !ws_dev)) return fail(ctx, FC_ERR_INVALID, "fc_causal_conv_backward: null pointer");
    const uint64_t addr = (uint64_t)dy_dev | (uint64_t)x_dev | (uint64_t)dx_dev | (uint64_t)state_in_dev | (uint64_t)dstate_out_dev | (uint64_t)dstate_in_dev;
    if ((addr & (fc_elem_size(s.dtype) - 1)) ||
        (((uint64_t)w_dev | (uint64_t)bias_dev | (uint64_t)dw_dev | (uint64_t)dbias_dev | (uint64_t)lengths_dev | (uint64_t)ws_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_causal_conv_backward: unaligned pointer");
    if (!fc_apart({{s.B, s.x_batch}, {s.T, s.x_token}}, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_causal_conv_backward: tokens of dx overlap");
    const int columns = columns_of(s);
    conv_params p = params_of(s, plan->walks_backward);
    p.dy = dy_dev; p.x = x_dev; p.w = w_dev; p.bias = bias_dev; p.y = dx_dev; p.state_in = state_in_dev; p.dstate_out = dstate_out_dev;
    p.dstate_in = dstate_in_dev; p.lengths = lengths_dev;
    p.part = sums ? (float *)ws_dev : nullptr;
    const unsigned blocks = (unsigned)(((long)s.B * p.walks * columns + kThreads - 1) / kThreads);
    const fc_device_scope on(ctx);
    with_kernel(s, [&](auto dt, auto v, auto taps) {
        fc_causal_conv_gradient_kernel<decltype(dt)::value, decltype(v)::value, decltype(taps)::value>
            <<<dim3(blocks), dim3(kThreads), 0, ctx->stream>>>(p, columns);
    });
    FC_LAUNCH_CHECK(ctx, "fc_causal_conv_gradient_kernel");
    if (!sums) return FC_OK;
    const long size = (long)(s.taps + 1) * s.C;
    fc_causal_conv_sum_kernel<<<dim3((unsigned)((size + kPartValues - 1) / kPartValues)), dim3(kPartThreads), 0, ctx->stream>>>(p.part, dw_dev, dbias_dev,
                                                                                                                                s.B * p.walks, s.C, s.taps);
    FC_LAUNCH_CHECK(ctx, "fc_causal_conv_sum_kernel");
    return FC_OK;
}
