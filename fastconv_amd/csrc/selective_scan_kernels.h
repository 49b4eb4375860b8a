// Kernels of the selective scan, for one element type each (selective_scan_<type>.hip).
#pragma once

#include <type_traits>

#include "selective_scan.h"

namespace {

// v of the lane that a cross-lane pattern of DPP names
template <int CONTROL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CONTROL, 0xf, 0xf, true));
}

// The sum over the L neighbouring lanes of a channel, in all of them.
template <int L>
__device__ __forceinline__ float sum_states(float v) {
    if (L > 1) v += dpp<0xB1>(v);       // lanes 1, 0, 3, 2
    if (L > 2) v += dpp<0x4E>(v);       // lanes 2, 3, 0, 1
    if (L > 4) v += dpp<0x141>(v);      // eight lanes in reverse
    if (L > 8) v += dpp<0x140>(v);      // sixteen
    return v;
}

// Where a workgroup is, and its threads in both of their arrangements.
template <int L, int S>
struct scan_place {
    typedef scan_form<L, S> F;
    long b, len;
    int walk, group, block;
    long first;              // channel of the tensors that the workgroup begins with
    int c, row;              // channel and first token of a tile, along the channels
    int d, ds;               // channel along the channels and along the states; -1 past the last
    int chan, sg;            // along the states: channel of the workgroup, which S states of it
    __device__ __forceinline__ scan_place(const fc_scan_run &r) {
        unsigned i = blockIdx.x;
        block = i % r.blocks;
        i /= r.blocks;
        walk = i % r.walks;
        b = i / r.walks;
        len = fc_scan_length(r, b);
        const int per = r.blocks / r.G;
        group = block / per;
        const int from = (block - group * per) * F::CH, tid = threadIdx.x;
        first = group * (long)r.per_group + from;
        c = F::channel(tid);
        row = F::row(tid);
        chan = tid / L;
        sg = tid % L;
        d = from + c < r.per_group ? group * r.per_group + from + c : -1;
        ds = from + chan < r.per_group ? group * r.per_group + from + chan : -1;
    }
};

// A thread's offsets in bytes into tiles of the tensors, and the tokens' distances.
struct scan_offsets {
    uint32_t x, delta, z, y, b, c;
    uint32_t x_token, delta_token, z_token, y_token, b_token, c_token;
    template <int L, int S>
    __device__ __forceinline__ scan_offsets(const fc_scan_run &r, const scan_place<L, S> &at, uint32_t es) {
        typedef scan_form<L, S> F;
        x_token = (uint32_t)r.x_token * es;
        delta_token = (uint32_t)r.delta_token * es;
        z_token = (uint32_t)r.z_token * es;
        y_token = (uint32_t)r.y_token * es;
        b_token = (uint32_t)r.b_token * es;
        c_token = (uint32_t)r.c_token * es;
        const bool there = at.d >= 0;
        x = F::channel_offset(threadIdx.x, there, es, x_token);
        delta = F::channel_offset(threadIdx.x, there, es, delta_token);
        z = F::channel_offset(threadIdx.x, there, es, z_token);
        y = F::channel_offset(threadIdx.x, there, es, y_token);
        b = F::shared_offset(threadIdx.x, r.N, es, b_token);
        c = F::shared_offset(threadIdx.x, r.N, es, c_token);
    }
};

// One branch for all steps of a thread: their chains of dependent operations run side by side.
template <int N>
__device__ __forceinline__ void to_steps(const fc_scan_run &r, float (&v)[N]) {
    if (!r.softplus) return;
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = fc_softplus(v[k]);
}

// A tensor's tokens from t0 of a tile on, through a buffer resource: a thread has one 32-bit offset for all its tokens, whose distances are scalars, and an
// offset past 2^31 reads zeros and writes nothing.
template <int DT>
struct scan_window {
    typedef typename fc_elem<DT>::type E;
    static constexpr int ES = (int)sizeof(E);
    __amdgpu_buffer_rsrc_t res;
    __device__ __forceinline__ scan_window(const void *base, long offset)
        : res(__builtin_amdgcn_make_buffer_rsrc(uniform_ptr((E *)base + offset), 0, 0x7fffffff, 0x00020000)) {}
    __device__ __forceinline__ E get(uint32_t at, uint32_t further) const {
        if constexpr (ES == 4) return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b32(res, at, further, 0));
        else return __builtin_bit_cast(E, __builtin_amdgcn_raw_buffer_load_b16(res, at, further, 0));
    }
    __device__ __forceinline__ void put(float v, uint32_t at, uint32_t further) const {
        const E e = (E)v;
        if constexpr (ES == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, e), res, at, further, 0);
        else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, e), res, at, further, 0);
    }
};

// What a thread has of a tile before it is laid out for the states: values of its channel, one every ROWS tokens.  `n` tokens are there, the others zeros.
template <int DT, int L, int S, bool GATE, bool DY>
struct scan_tile {
    typedef scan_form<L, S> F;
    typedef typename fc_elem<DT>::type E;
    typedef scan_window<DT> W;
    E x[F::EACH], delta[F::EACH], z[GATE ? F::EACH : 1], dy[DY ? F::EACH : 1], b[F::SHARED], c[F::SHARED];

    // channels: x, delta, z, dy; states: B, and C if asked for
    __device__ __forceinline__ void read(const fc_scan_run &r, const scan_place<L, S> &at, const scan_offsets &off, long t0, long end, bool channels, bool states,
                                         bool with_c) {
        const int n = (int)(end - t0 < kScanTile ? end - t0 : kScanTile);
        const W wx(r.x, at.b * r.x_batch + t0 * r.x_token + at.first), wd(r.delta, at.b * r.delta_batch + t0 * r.delta_token + at.first);
        const W wz(r.z, at.b * r.z_batch + t0 * r.z_token + at.first), wy(r.dy, at.b * r.y_batch + t0 * r.y_token + at.first);
        const W wb(r.b, at.b * r.b_batch + t0 * r.b_token + at.group * r.b_group), wc(r.c, at.b * r.c_batch + t0 * r.c_token + at.group * r.c_group);
        auto all = [&](auto each, auto several) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < F::EACH && channels; k++) {
                x[k] = each(wx, off.x, off.x_token, k);
                delta[k] = each(wd, off.delta, off.delta_token, k);
                if (GATE) z[k] = each(wz, off.z, off.z_token, k);
                if (DY) dy[k] = each(wy, off.y, off.y_token, k);
            }
#pragma unroll
            for (int k = 0; k < F::SHARED && states; k++) {
                b[k] = several(wb, off.b, off.b_token, k);
                if (with_c) c[k] = several(wc, off.c, off.c_token, k);
            }
        };
        if (n == kScanTile) {
            all([&](const W &w, uint32_t lane, uint32_t token, int k) __attribute__((always_inline)) { return w.get(lane, k * F::ROWS * token); },
                [&](const W &w, uint32_t lane, uint32_t token, int k) __attribute__((always_inline)) { return w.get(lane, k * F::BC * token); });
        } else {
            const int row = F::shared_token(threadIdx.x);
            all([&](const W &w, uint32_t lane, uint32_t token, int k) __attribute__((always_inline)) {
                    return w.get(at.row + k * F::ROWS < n ? lane + k * F::ROWS * token : kNowhere, 0);
                },
                [&](const W &w, uint32_t lane, uint32_t token, int k) __attribute__((always_inline)) {
                    return w.get(row + k * F::BC < n ? lane + k * F::BC * token : kNowhere, 0);
                });
        }
    }
};

// The same laid out for the states.
template <int L, int S>
struct alignas(16) scan_shared {
    typedef scan_form<L, S> F;
    float2 du[kScanTile][F::CH];      // dt and dt x
    float b[kScanTile][F::NP], c[kScanTile][F::NP];
};

template <class F, class E>
__device__ __forceinline__ void lay_out(float (*to)[F::NP], const E (&v)[F::SHARED]) {
#pragma unroll
    for (int k = 0; k < F::SHARED; k++) {
        const int i = threadIdx.x + k * F::THREADS;
        if (i < kScanTile * F::NP) to[i / F::NP][i % F::NP] = (float)v[k];
    }
}

// A lane's S values of a row in LDS, in one access.
template <int S>
__device__ __forceinline__ void take(float (&to)[S], const float *from) {
    __builtin_memcpy(to, __builtin_assume_aligned(from, S * sizeof(float)), sizeof to);
}

template <int L, int S>
__device__ __forceinline__ void read_rates(const fc_scan_run &r, const scan_place<L, S> &at, float (&rate)[S]) {
#pragma unroll
    for (int j = 0; j < S; j++) {
        const int n = at.sg * S + j;
        rate[j] = at.ds >= 0 && n < r.N ? fc_scan_rate(r.A[(long)at.ds * r.N + n]) : 0.f;
    }
}

template <int L, int S>
__device__ __forceinline__ void read_states(const fc_scan_run &r, const scan_place<L, S> &at, const float *from, long row, float (&h)[S]) {
#pragma unroll
    for (int j = 0; j < S; j++) {
        const int n = at.sg * S + j;
        h[j] = from && at.ds >= 0 && n < r.N ? from[(row * r.channels + at.ds) * r.N + n] : 0.f;
    }
}

template <int L, int S>
__device__ __forceinline__ void write_states(const fc_scan_run &r, const scan_place<L, S> &at, float *to, long row, const float (&h)[S]) {
#pragma unroll
    for (int j = 0; j < S; j++) {
        const int n = at.sg * S + j;
        if (at.ds >= 0 && n < r.N) to[(row * r.channels + at.ds) * r.N + n] = h[j];
    }
}

// Answers.  Bound by the vector ALUs, which are busy 99 % of the time: an exponential (two instructions' time) and four instructions a state, and for each token of a
// lane about 15 more, 4 of which sum the lanes' parts, 5 form the step and 3 the gate.  12544 tokens of 2048 channels, 16 states, bf16: 114 to 124 us, of
// which 62 are the states' own.  u B through 4x4x1 matrix instructions takes 12 cycles of 157 off the vector ALUs and leaves the time as it is (118 to 122 us).
template <int DT, int L, int S, bool GATE>
__global__ __launch_bounds__(kScanThreads, 4) void fc_selective_scan_kernel(const fc_scan_run r) {
    typedef scan_form<L, S> F;
    typedef typename fc_elem<DT>::type E;
    __shared__ scan_shared<L, S> lds;
    __shared__ float ys[kScanTile][F::CH];
    const scan_place<L, S> at(r);
    const long t0 = at.walk * r.segment, t1 = t0 + r.segment < r.T ? t0 + r.segment : r.T, end = t1 < at.len ? t1 : at.len;
    float rate[S], h[S];
    read_rates<L, S>(r, at, rate);
    if (r.segments > 1) read_states<L, S>(r, at, r.parts, at.b * r.segments + at.walk, h);
    else read_states<L, S>(r, at, r.state_in, at.b, h);
    const float bias = r.delta_bias && at.d >= 0 ? r.delta_bias[at.d] : 0.f, skip = r.D && at.d >= 0 ? r.D[at.d] : 0.f;
    const scan_offsets off(r, at, sizeof(E));
    scan_tile<DT, L, S, GATE, false> now;
    if (t0 < end) now.read(r, at, off, t0, end, true, true, true);
    for (long t = t0; t < end; t += kScanTile) {
        const int n = (int)(end - t < kScanTile ? end - t : kScanTile);
        float x[F::EACH], z[GATE ? F::EACH : 1], dt[F::EACH];
#pragma unroll
        for (int k = 0; k < F::EACH; k++) {
            x[k] = (float)now.x[k];
            if (GATE) z[k] = (float)now.z[k];
            dt[k] = (float)now.delta[k] + bias;
        }
        to_steps(r, dt);
#pragma unroll
        for (int k = 0; k < F::EACH; k++) lds.du[at.row + k * F::ROWS][at.c] = make_float2(dt[k], dt[k] * x[k]);
        lay_out<F>(lds.b, now.b);
        lay_out<F>(lds.c, now.c);
        __syncthreads();
        if (t + kScanTile < end) now.read(r, at, off, t + kScanTile, end, true, true, true);
        float mine = 0.f;
        auto token = [&](int i) __attribute__((always_inline)) {
            const float2 du = lds.du[i][at.chan];
            float bs[S], cs[S];
            take(bs, &lds.b[i][at.sg * S]);
            take(cs, &lds.c[i][at.sg * S]);
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < S; j++) {
                h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(du.x * rate[j]), h[j], du.y * bs[j]);
                s = __builtin_fmaf(cs[j], h[j], s);
            }
            return sum_states<L>(s);
        };
        if (n == kScanTile) {
#pragma unroll 8
            for (int i = 0; i < kScanTile; i++) {
                const float s = token(i);
                mine = i % L == at.sg ? s : mine;      // each lane keeps one of L tokens
                if (i % L == L - 1) ys[i - L + 1 + at.sg][at.chan] = mine;
            }
        } else {
            for (int i = 0; i < n; i++) {
                const float s = token(i);
                if (at.sg == 0) ys[i][at.chan] = s;
            }
        }
        __syncthreads();
        const scan_window<DT> y(r.y, at.b * r.y_batch + t * r.y_token + at.first);
        float out[F::EACH];
#pragma unroll
        for (int k = 0; k < F::EACH; k++) {
            out[k] = __builtin_fmaf(skip, x[k], ys[at.row + k * F::ROWS][at.c]);
            if (GATE) out[k] *= fc_silu(z[k]);
        }
        if (n == kScanTile) {
#pragma unroll
            for (int k = 0; k < F::EACH; k++) y.put(out[k], off.y, k * F::ROWS * off.y_token);
        } else {
#pragma unroll
            for (int k = 0; k < F::EACH; k++) y.put(out[k], at.row + k * F::ROWS < n ? off.y + k * F::ROWS * off.y_token : kNowhere, 0);
        }
    }
    // tokens past the end of a shorter sequence
    if (at.d >= 0)
        for (long t = (end > t0 ? end : t0) + at.row; t < t1; t += F::ROWS) ((E *)r.y)[at.b * r.y_batch + t * r.y_token + at.d] = (E)0.f;
    if (r.state_out && at.walk == r.segments - 1) write_states<L, S>(r, at, r.state_out, at.b, h);
}

// What each segment adds to no state, the sum of its steps and, with GRADS, what it adds to no gradient: the gradient of a state is the sum of what each later token
// adds, decayed on its way, and the product of the decays from the segment's begin on is at hand.  Bound as the answers are: 87 to 93 us there, with GRADS 147 to 159 (4 x 3136
// tokens).
template <int DT, int L, int S, bool GRADS, bool GATE>
__global__ __launch_bounds__(kScanThreads, GRADS ? 3 : 4) void fc_selective_scan_ends_kernel(const fc_scan_run r) {
    typedef scan_form<L, S> F;
    __shared__ scan_shared<L, S> lds;
    __shared__ float gs[GRADS ? kScanTile : 1][GRADS ? F::CH : 1];
    const scan_place<L, S> at(r);
    const long first = (long)at.walk * r.per_walk * r.segment, last = first + r.per_walk * r.segment < r.T ? first + r.per_walk * r.segment : r.T;
    const long end = last < at.len ? last : at.len;
    float rate[S], h[S], decay[S], grad[S], steps = 0.f;
    read_rates<L, S>(r, at, rate);
    const float bias = r.delta_bias && at.d >= 0 ? r.delta_bias[at.d] : 0.f;
    const scan_offsets off(r, at, sizeof(typename fc_elem<DT>::type));
    scan_tile<DT, L, S, GATE && GRADS, GRADS> now;
    if (first < end) now.read(r, at, off, first, end, true, true, GRADS);
    long segment = at.b * r.segments + (long)at.walk * r.per_walk;
    for (long t = first; t < last; t += kScanTile) {
        const int n = (int)(end - t < 0 ? 0 : end - t < kScanTile ? end - t : kScanTile);
        if ((t - first) % r.segment == 0) {
            steps = 0.f;
#pragma unroll
            for (int j = 0; j < S; j++) {
                h[j] = grad[j] = 0.f;
                decay[j] = 1.f;
            }
        }
        if (n > 0) {
            float dt[F::EACH];
#pragma unroll
            for (int k = 0; k < F::EACH; k++) dt[k] = (float)now.delta[k] + bias;
            to_steps(r, dt);
#pragma unroll
            for (int k = 0; k < F::EACH; k++) {
                lds.du[at.row + k * F::ROWS][at.c] = make_float2(dt[k], dt[k] * (float)now.x[k]);
                if constexpr (GRADS) {
                    float g = (float)now.dy[k];
                    if (GATE) g *= fc_silu((float)now.z[k]);
                    gs[at.row + k * F::ROWS][at.c] = g;
                }
            }
            lay_out<F>(lds.b, now.b);
            if (GRADS) lay_out<F>(lds.c, now.c);
            __syncthreads();
            if (t + kScanTile < end) now.read(r, at, off, t + kScanTile, end, true, true, GRADS);
            auto token = [&](int i) __attribute__((always_inline)) {
                const float2 du = lds.du[i][at.chan];
                float bs[S];
                take(bs, &lds.b[i][at.sg * S]);
                float cs[S] = {}, g = 0.f;
                if constexpr (GRADS) {
                    take(cs, &lds.c[i][at.sg * S]);
                    g = gs[i][at.chan];
                }
                steps += du.x;
#pragma unroll
                for (int j = 0; j < S; j++) {
                    const float a = __builtin_amdgcn_exp2f(du.x * rate[j]);
                    h[j] = __builtin_fmaf(a, h[j], du.y * bs[j]);
                    if (GRADS) {
                        decay[j] *= a;
                        grad[j] = __builtin_fmaf(decay[j], cs[j] * g, grad[j]);
                    }
                }
            };
            if (n == kScanTile) {
#pragma unroll 8
                for (int i = 0; i < kScanTile; i++) token(i);
            } else {
                for (int i = 0; i < n; i++) token(i);
            }
            __syncthreads();
        }
        const long next = t + kScanTile;
        if ((next - first) % r.segment == 0 || next >= last) {
            write_states<L, S>(r, at, r.parts, segment, h);
            if (GRADS) write_states<L, S>(r, at, r.grads, segment, grad);
            if (at.sg == 0 && at.ds >= 0) r.steps[segment * r.channels + at.ds] = steps;
            segment++;
        }
    }
}

// A few tokens, L lanes a channel without LDS.  Bound by the states, read and written once a call (64 sequences of 4096 channels and 16 states: 33.5 MB in 11 us);
// what belongs to a channel is read once for SEQUENCES of them, whose loads are on their way together.
template <int DT, int L, int S, bool GATE, int SEQUENCES>
__global__ __launch_bounds__(256) void fc_selective_scan_step_kernel(const fc_scan_run r, unsigned across) {      // workgroups for all channels
    typedef typename fc_elem<DT>::type E;
    typedef fc_vec<DT, S> V;
    const long at = (long)(blockIdx.x % across) * 256 + threadIdx.x;
    const int d = (int)(at / L), sg = threadIdx.x % L, n0 = sg * S;
    if (d >= r.channels) return;
    const int group = d / r.per_group;
    // a lane's four states, or those that there are
    const bool whole = n0 + S <= r.N;
    float rate[S];
    if (whole) __builtin_memcpy(rate, r.A + (long)d * r.N + n0, sizeof rate);
    else
#pragma unroll
        for (int j = 0; j < S; j++) rate[j] = n0 + j < r.N ? r.A[(long)d * r.N + n0 + j] : 0.f;
#pragma unroll
    for (int j = 0; j < S; j++) rate[j] = fc_scan_rate(rate[j]);
    const float bias = r.delta_bias ? r.delta_bias[d] : 0.f, skip = r.D ? r.D[d] : 0.f;
    const int first = (int)(blockIdx.x / across) * SEQUENCES;
    float h[SEQUENCES][S];
    long len[SEQUENCES];
#pragma unroll
    for (int s = 0; s < SEQUENCES; s++) {
        const long b = first + s < r.B ? first + s : r.B - 1;
        len[s] = first + s < r.B ? fc_scan_length(r, b) : 0;
        const float *from = r.state_in + (b * r.channels + d) * r.N + n0;
#pragma unroll
        for (int j = 0; j < S; j++) h[s][j] = 0.f;
        if (r.state_in && whole) {
            __builtin_memcpy(h[s], from, sizeof h[s]);
        } else if (r.state_in) {
#pragma unroll
            for (int j = 0; j < S; j++)
                if (n0 + j < r.N) h[s][j] = from[j];
        }
    }
    for (long t = 0; t < r.T; t++) {
        E x[SEQUENCES], delta[SEQUENCES], z[SEQUENCES];
        V B[SEQUENCES], C[SEQUENCES];
#pragma unroll
        for (int s = 0; s < SEQUENCES; s++) {      // a token past the end is read where the first lies, and moves nothing
            const long b = first + s < r.B ? first + s : r.B - 1, u = t < len[s] ? t : 0;
            x[s] = ((const E *)r.x)[b * r.x_batch + u * r.x_token + d];
            delta[s] = ((const E *)r.delta)[b * r.delta_batch + u * r.delta_token + d];
            if (GATE) z[s] = ((const E *)r.z)[b * r.z_batch + u * r.z_token + d];
            const E *pb = (const E *)r.b + b * r.b_batch + u * r.b_token + group * r.b_group, *pc = (const E *)r.c + b * r.c_batch + u * r.c_token + group * r.c_group;
            if (whole) {
                __builtin_memcpy(&B[s], pb + n0, sizeof(V));
                __builtin_memcpy(&C[s], pc + n0, sizeof(V));
            } else {
#pragma unroll
                for (int j = 0; j < S; j++) {
                    B[s].v[j] = n0 + j < r.N ? pb[n0 + j] : (E)0.f;
                    C[s].v[j] = n0 + j < r.N ? pc[n0 + j] : (E)0.f;
                }
            }
        }
        float steps[SEQUENCES];
#pragma unroll
        for (int s = 0; s < SEQUENCES; s++) steps[s] = (float)delta[s] + bias;
        to_steps(r, steps);
#pragma unroll
        for (int s = 0; s < SEQUENCES; s++) {
            const bool there = t < len[s];
            const float v = (float)x[s], dt = steps[s], u = dt * v;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < S; j++) {
                const float now = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * rate[j]), h[s][j], u * B[s].get(j));
                h[s][j] = there ? now : h[s][j];
                sum = __builtin_fmaf(C[s].get(j), now, sum);
            }
            sum = __builtin_fmaf(skip, v, sum_states<L>(sum));
            if (GATE) sum *= fc_silu((float)z[s]);
            if (sg == 0 && first + s < r.B) ((E *)r.y)[(first + s) * r.y_batch + t * r.y_token + d] = (E)(there ? sum : 0.f);
        }
    }
    if (!r.state_out) return;
#pragma unroll
    for (int s = 0; s < SEQUENCES; s++) {
        if (first + s >= r.B) break;
        float *to = r.state_out + ((long)(first + s) * r.channels + d) * r.N + n0;
        if (whole) {
            __builtin_memcpy(to, h[s], sizeof h[s]);
        } else {
#pragma unroll
            for (int j = 0; j < S; j++)
                if (n0 + j < r.N) to[j] = h[s][j];
        }
    }
}

// The sum of two values over lanes that lie 32 (ROWS: 16) apart: the first where the lane's bit is 0, the second where it is 1.
template <bool ROWS>
__device__ __forceinline__ float sum_two(float a, float b) {
    const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
    const auto s = ROWS ? __builtin_amdgcn_permlane16_swap(x, y, false, false) : __builtin_amdgcn_permlane32_swap(x, y, false, false);
    const unsigned u = s[0], v = s[1];
    return __builtin_bit_cast(float, u) + __builtin_bit_cast(float, v);
}

// Sums over the channels of a wavefront (lanes with the same lane % L) of 2 S values a lane, spread over its four rows of 16 lanes: rows 0 and 1 get the first S values'
// sums, half of them each (S = 1: both the same), rows 2 and 3 the others'.
template <int L, int S2, int O>
__device__ __forceinline__ void sum_channels(float (&o)[O], float (&v)[S2]) {
    constexpr int S = S2 / 2;
    float w[S];
#pragma unroll
    for (int i = 0; i < S; i++) w[i] = sum_two<false>(v[i], v[i + S]);
#pragma unroll
    for (int i = 0; i < O; i++) {
        o[i] = sum_two<true>(w[i], w[S > 1 ? i + O : i]);
        if (L <= 8) o[i] += dpp<0x128>(o[i]);      // lanes turned by 8 of 16
        if (L <= 4) o[i] += dpp<0x124>(o[i]);
    }
}

// Gradients of each segment, which is a tile: forwards through it from the state that enters, states in registers, then backwards.  Bound by the vector ALUs, busy
// 77 % of the time with two wavefronts a SIMD (256 registers): 121 instructions for each token of a lane, 64 of them the states' own.  dB and dC are sums over
// channels, of a wavefront's by lane swaps, of a workgroup's through LDS, of all by a launch of their own, so that their order is always the same.  4 x 3136 tokens of
// 2048 channels, 16 states, bf16: 462 to 495 us.
template <int DT, int L, int S, bool GATE>
__global__ __launch_bounds__(kScanThreads, 2) void fc_selective_scan_gradient_kernel(const fc_scan_run r) {
    typedef scan_form<L, S> F;
    typedef typename fc_elem<DT>::type E;
    // Tokens whose states and decays are in registers at a time.  2048 channels of 4 x 3136 tokens and 16 states: 709 us with 8, 903 with 16, and 732 with 16 whose
    // decays are formed again.
    constexpr int PART = L < 16 ? 8 : 16;
    __shared__ scan_shared<L, S> lds;
    __shared__ float gs[kScanTile][F::CH], ys[GATE ? kScanTile : 1][GATE ? F::CH : 1];
    constexpr int HELD = L < 16 ? kScanTile : PART;      // tokens: with 16 lanes a whole tile of them would leave room for one workgroup a unit
    __shared__ alignas(16) float waves[F::WAVES][HELD][2 * F::NP];      // dB and dC of each wavefront's channels
    __shared__ float2 rows[F::ROWS][F::CH];
    const scan_place<L, S> at(r);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float rate[S], dA[S] = {}, dD = 0.f, dbias = 0.f;
    read_rates<L, S>(r, at, rate);
    const float bias = r.delta_bias && at.d >= 0 ? r.delta_bias[at.d] : 0.f, skip = r.D && at.d >= 0 ? r.D[at.d] : 0.f;
    const long first = (long)at.walk * r.per_walk, last = first + r.per_walk < r.segments ? first + r.per_walk : r.segments;
    const scan_offsets off(r, at, sizeof(E));
    scan_tile<DT, L, S, GATE, true> now;
    if (first * kScanTile < at.len) now.read(r, at, off, first * kScanTile, at.len, true, true, true);
    for (long seg = first; seg < last; seg++) {
        const long t = seg * kScanTile, end = t + kScanTile < r.T ? t + kScanTile : r.T;
        const int n = (int)(at.len - t < 0 ? 0 : at.len - t < kScanTile ? at.len - t : kScanTile);
        float *shared = r.shared + ((at.block * (long)r.B + at.b) * r.T + t) * 2 * r.N;
        if (n > 0) {
            float start[S], G[S];
            read_states<L, S>(r, at, r.parts, at.b * r.segments + seg, start);
            read_states<L, S>(r, at, r.grads, at.b * r.segments + seg, G);
            float steps[F::EACH];
#pragma unroll
            for (int k = 0; k < F::EACH; k++) steps[k] = (float)now.delta[k] + bias;
            to_steps(r, steps);
#pragma unroll
            for (int k = 0; k < F::EACH; k++) {
                const int i = at.row + k * F::ROWS;
                const bool in = i < n && at.d >= 0;      // a token past the last moves nothing
                const float x = in ? (float)now.x[k] : 0.f;
                steps[k] = in ? steps[k] : 0.f;
                float g = in ? (float)now.dy[k] : 0.f;
                if (GATE && in) g *= fc_silu((float)now.z[k]);
                lds.du[i][at.c] = make_float2(steps[k], steps[k] * x);
                gs[i][at.c] = g;
            }
            lay_out<F>(lds.b, now.b);
            lay_out<F>(lds.c, now.c);
            __syncthreads();
            // Some tokens' states and decays are kept at a time: with all of them there are no registers left for what comes next.  First the states that enter each
            // part but the first; they wait where the sums of the part before theirs will lie.
            static_assert(PART == kScanTile || sizeof(waves[0][0]) * PART >= 64 * S * sizeof(float));
            auto mid = [&](int part) __attribute__((always_inline)) { return &waves[wave][HELD == PART ? 0 : part - PART][0] + lane * S; };
            float h[S];
#pragma unroll
            for (int j = 0; j < S; j++) h[j] = start[j];
#pragma unroll 1
            for (int part = PART; part < kScanTile; part += PART) {
#pragma unroll
                for (int i = 0; i < PART; i++) {
                    const float2 du = lds.du[part - PART + i][at.chan];
                    float bs[S];
                    take(bs, &lds.b[part - PART + i][at.sg * S]);
#pragma unroll
                    for (int j = 0; j < S; j++) h[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(du.x * rate[j]), h[j], du.y * bs[j]);
                }
                __builtin_memcpy(__builtin_assume_aligned(mid(part), S * sizeof(float)), h, sizeof h);
            }
            // the workgroup's sums of dB and dC of `count` tokens from `from` on
            auto add_up = [&](int from, int count) __attribute__((always_inline)) {
                for (int i = threadIdx.x; i < count * 2 * F::NP; i += F::THREADS) {
                    const int token = i / (2 * F::NP), k = i % (2 * F::NP), half = k / F::NP, state = k % F::NP;
                    if (state >= r.N) continue;
                    float s = waves[0][token][k];
#pragma unroll
                    for (int w = 1; w < F::WAVES; w++) s += waves[w][token][k];
                    shared[((long)(from + token) * 2 + half) * r.N + state] = s;
                }
            };
#pragma unroll 1
            for (int part = kScanTile - PART; part >= 0; part -= PART) {
                float hs[PART][S], as[PART][S], enters[S];
#pragma unroll
                for (int j = 0; j < S; j++) enters[j] = start[j];
                if (part) take(enters, mid(part));
#pragma unroll
                for (int i = 0; i < PART; i++) {
                    if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);      // else all reads move to the front, and registers spill
                    const float2 du = lds.du[part + i][at.chan];
                    float bs[S];
                    take(bs, &lds.b[part + i][at.sg * S]);
#pragma unroll
                    for (int j = 0; j < S; j++) {
                        as[i][j] = __builtin_amdgcn_exp2f(du.x * rate[j]);
                        hs[i][j] = __builtin_fmaf(as[i][j], i ? hs[i ? i - 1 : 0][j] : enters[j], du.y * bs[j]);
                    }
                }
                fc_wave_sync();
                float2 kept = make_float2(0.f, 0.f);
                float mine = 0.f;
#pragma unroll
                for (int i = PART - 1; i >= 0; i--) {
                    if (i % 2) __builtin_amdgcn_sched_barrier(0);
                    const float2 du = lds.du[part + i][at.chan];
                    const float g = gs[part + i][at.chan];
                    float bs[S], cs[S];
                    take(bs, &lds.b[part + i][at.sg * S]);
                    take(cs, &lds.c[part + i][at.sg * S]);
                    float v[2 * S], du_sum = 0.f, dt_sum = 0.f, y = 0.f;
#pragma unroll
                    for (int j = 0; j < S; j++) {
                        G[j] = __builtin_fmaf(cs[j], g, G[j]);
                        v[j] = G[j] * du.y;
                        v[S + j] = g * hs[i][j];
                        if (GATE) y = __builtin_fmaf(cs[j], hs[i][j], y);
                        du_sum = __builtin_fmaf(G[j], bs[j], du_sum);
                        G[j] *= as[i][j];
                        const float k = G[j] * (i ? hs[i ? i - 1 : 0][j] : enters[j]);
                        dt_sum = __builtin_fmaf(k, rate[j], dt_sum);
                        dA[j] = __builtin_fmaf(k, du.x, dA[j]);
                    }
                    du_sum = sum_states<L>(du_sum);
                    dt_sum = sum_states<L>(dt_sum);
                    float s[S < 4 ? 1 : 2];
                    sum_channels<L>(s, v);
                    if ((L == 16 || (lane & 15) < L) && (S > 1 || (lane & 16) == 0))
                        __builtin_memcpy(__builtin_assume_aligned(&waves[wave][HELD == PART ? i : part + i][(lane >> 5) * F::NP + (lane & 15) * S + (lane >> 4 & 1) * (S / 2)], sizeof s), s, sizeof s);
                    // each lane keeps one of L tokens
                    if (i % L == at.sg) kept = make_float2(du_sum, dt_sum);
                    if (i % L == 0) lds.du[part + i + at.sg][at.chan] = kept;      // these tokens' steps are not needed any more
                    if constexpr (GATE) {
                        y = sum_states<L>(y);
                        mine = i % L == at.sg ? y : mine;
                        if (i % L == 0) ys[part + i + at.sg][at.chan] = mine;
                    }
                }
                if (HELD < kScanTile) {
                    __syncthreads();
                    add_up(part, n - part < 0 ? 0 : n - part < PART ? n - part : PART);
                    if (part) __syncthreads();
                }
            }
            scan_tile<DT, L, S, GATE, true> here;
            // this tile's values once more: kept, they would leave the states no registers
            here.read(r, at, off, t, at.len, true, false, false);
            __syncthreads();
            if (HELD == kScanTile) add_up(0, n);
            if (seg + 1 < last && t + kScanTile < at.len) now.read(r, at, off, t + kScanTile, at.len, true, true, true);
            const scan_window<DT> dx(r.dx, at.b * r.x_batch + t * r.x_token + at.first), dd(r.ddelta, at.b * r.delta_batch + t * r.delta_token + at.first);
            const scan_window<DT> dz(r.dz, at.b * r.z_batch + t * r.z_token + at.first);
            float slope[F::EACH];      // of the step
#pragma unroll
            for (int k = 0; k < F::EACH; k++) slope[k] = 1.f;
            if (r.softplus)
#pragma unroll
                for (int k = 0; k < F::EACH; k++) slope[k] = fc_sigmoid((float)here.delta[k] + bias);
#pragma unroll
            for (int k = 0; k < F::EACH; k++) {
                const int i = at.row + k * F::ROWS;
                const bool in = i < n;      // channels past the last are zeros and nowhere
                const float2 s = lds.du[i][at.c];
                const float x = (float)here.x[k], g = gs[i][at.c];
                const float dstep = __builtin_fmaf(x, s.x, 0.693147181f * s.y) * slope[k];
                auto put = [&](const scan_window<DT> &w, float v, uint32_t lane, uint32_t token) __attribute__((always_inline)) {
                    if (n == kScanTile) w.put(v, lane, k * F::ROWS * token);
                    else w.put(v, in ? lane + k * F::ROWS * token : kNowhere, 0);
                };
                put(dx, __builtin_fmaf(steps[k], s.x, skip * g), off.x, off.x_token);
                put(dd, dstep, off.delta, off.delta_token);
                if constexpr (GATE) put(dz, (float)here.dy[k] * __builtin_fmaf(skip, x, ys[i][at.c]) * fc_silu_slope((float)here.z[k]), off.z, off.z_token);
                dD = in ? __builtin_fmaf(g, x, dD) : dD;
                dbias = in ? dbias + dstep : dbias;
            }
            __syncthreads();
        }
        // tokens past the end of a shorter sequence
        if (at.d >= 0)
            for (long i = t + n + at.row; i < end; i += F::ROWS) {
                ((E *)r.dx)[at.b * r.x_batch + i * r.x_token + at.d] = (E)0.f;
                ((E *)r.ddelta)[at.b * r.delta_batch + i * r.delta_token + at.d] = (E)0.f;
                if (GATE) ((E *)r.dz)[at.b * r.z_batch + i * r.z_token + at.d] = (E)0.f;
            }
        for (long i = (long)n * 2 * r.N + threadIdx.x; i < (end - t) * 2 * r.N; i += F::THREADS) shared[i] = 0.f;
    }
    // what this walk adds to the gradients of its channels
    float *sums = r.sums + ((at.b * r.walks + at.walk) * r.channels) * (r.N + 2);
#pragma unroll
    for (int j = 0; j < S; j++) {
        const int s = at.sg * S + j;
        if (at.ds >= 0 && s < r.N) sums[(long)at.ds * (r.N + 2) + s] = dA[j];
    }
    rows[at.row][at.c] = make_float2(dD, dbias);
    __syncthreads();
    if (at.row == 0 && at.d >= 0) {
        float2 s = rows[0][at.c];
#pragma unroll
        for (int k = 1; k < F::ROWS; k++) {
            s.x += rows[k][at.c].x;
            s.y += rows[k][at.c].y;
        }
        sums[(long)at.d * (r.N + 2) + r.N] = s.x;
        sums[(long)at.d * (r.N + 2) + r.N + 1] = s.y;
    }
}

template <int DT>
int scan_answers(fc_context *ctx, const fc_scan_run &r) {
    with_lanes(r.N, [&](auto lanes, auto states) {
        constexpr int L = decltype(lanes)::value, S = decltype(states)::value;
        const auto kernel = r.z ? fc_selective_scan_kernel<DT, L, S, true> : fc_selective_scan_kernel<DT, L, S, false>;
        kernel<<<dim3((unsigned)((long)r.blocks * r.walks * r.B)), dim3(kScanThreads), 0, ctx->stream>>>(r);
    });
    FC_LAUNCH_CHECK(ctx, "fc_selective_scan_kernel");
    return FC_OK;
}

template <int DT>
int scan_ends(fc_context *ctx, const fc_scan_run &r) {
    with_lanes(r.N, [&](auto lanes, auto states) {
        constexpr int L = decltype(lanes)::value, S = decltype(states)::value;
        const auto kernel = !r.dy  ? fc_selective_scan_ends_kernel<DT, L, S, false, false>
                            : r.z ? fc_selective_scan_ends_kernel<DT, L, S, true, true>
                                  : fc_selective_scan_ends_kernel<DT, L, S, true, false>;
        kernel<<<dim3((unsigned)((long)r.blocks * r.walks * r.B)), dim3(kScanThreads), 0, ctx->stream>>>(r);
    });
    FC_LAUNCH_CHECK(ctx, "fc_selective_scan_ends_kernel");
    return FC_OK;
}

// Lanes from which on two sequences share a channel's values, where a token is all there is: 64 sequences of 4096 channels, 16 states, bf16 11.8 us and 12.1, 16
// sequences 5.8 and 5.8; four tokens of 64 sequences 19.6 and 18.4.
constexpr long kManyLanes = 1l << 18;

template <int DT>
int scan_step(fc_context *ctx, const fc_scan_run &r) {
    with_step_lanes(r.N, [&](auto lanes, auto states) {
        constexpr int L = decltype(lanes)::value, S = decltype(states)::value;
        const unsigned across = (unsigned)(((long)r.channels * L + 255) / 256);
        if (r.T == 1 && (long)r.channels * L * r.B >= kManyLanes) {
            constexpr int Q = 2;
            const auto kernel = r.z ? fc_selective_scan_step_kernel<DT, L, S, true, Q> : fc_selective_scan_step_kernel<DT, L, S, false, Q>;
            kernel<<<dim3(across * (unsigned)((r.B + Q - 1) / Q)), dim3(256), 0, ctx->stream>>>(r, across);
        } else {
            const auto kernel = r.z ? fc_selective_scan_step_kernel<DT, L, S, true, 1> : fc_selective_scan_step_kernel<DT, L, S, false, 1>;
            kernel<<<dim3(across * (unsigned)r.B), dim3(256), 0, ctx->stream>>>(r, across);
        }
    });
    FC_LAUNCH_CHECK(ctx, "fc_selective_scan_step_kernel");
    return FC_OK;
}

template <int DT>
int scan_gradients(fc_context *ctx, const fc_scan_run &r) {
    with_lanes(r.N, [&](auto lanes, auto states) {
        constexpr int L = decltype(lanes)::value, S = decltype(states)::value;
        const auto kernel = r.z ? fc_selective_scan_gradient_kernel<DT, L, S, true> : fc_selective_scan_gradient_kernel<DT, L, S, false>;
        kernel<<<dim3((unsigned)((long)r.blocks * r.walks * r.B)), dim3(kScanThreads), 0, ctx->stream>>>(r);
    });
    FC_LAUNCH_CHECK(ctx, "fc_selective_scan_gradient_kernel");
    return FC_OK;
}

}  // namespace
