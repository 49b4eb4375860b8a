// RMS norm over rows of channels, after the addition of a residual, with a result in the rows' type or in 8 bits with a scale for each row:
//
//   h = x + residual, rounded to the rows' type,   rstd = 1/sqrt(mean of h^2 + eps),   y = h * rstd * gamma
//   8 bits: scale = max |y| / 127,  q = y / scale rounded to nearest, ties to even
//   dh = rstd * (gamma dy - xhat * mean of (gamma dy xhat)) + dsum,   dgamma = sum over rows of dy xhat,   xhat = h * rstd
//
// Bound by memory: about 10 operations a value against 8 bytes in 16-bit types.  A row stays in the registers of its wavefronts between its
// two uses, gamma from row to row.  rstd is no part of q: y / scale is 127 h gamma / max |h gamma|, so that the sum of squares and the largest
// value are found together, with one wait.
#include <type_traits>

#include "token_types.h"

namespace {

constexpr long kMostRows = 1l << 40;
constexpr int kMostChannels = 1 << 20;
// Rows whose largest value is smaller are zeros in 8 bits, with a scale of 0: their scale would leave the normal numbers.
constexpr float kLeastTop = 7.7037197775489434e-34f;      // 2^-110

enum { TO_TYPE = 0, TO_INT8 = 1, ONLY_INT8 = 2 };      // ONLY_INT8: no norm

struct rms_params {
    const void *x, *residual, *dy, *h, *dsum;
    void *sum, *y;           // y: the result, 8 bits or the rows' type; or dx
    const float *gamma;
    float *rstd, *scale, *part;
    long rows;
    int C;
    float eps;
    long x_row, residual_row, sum_row, y_row, dy_row;
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

// Sums and largest values over the WAVES wavefronts that share a row.  `turn` tells calls apart: the next one's values may lie beside this
// one's, so that one barrier is enough.
template <int WAVES>
__device__ __forceinline__ float2 join(float2 v, float2 (*slots)[16], int turn) {
    v.x = fc_wave_sum(v.x);
    v.y = wave_max(v.y);
    if constexpr (WAVES > 1) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane == 0) slots[turn & 1][wave] = v;
        __syncthreads();
        v = slots[turn & 1][0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) {
            const float2 o = slots[turn & 1][w];
            v.x += o.x;
            v.y = fmaxf(v.y, o.y);
        }
    }
    return v;
}

// 1/sqrt(mean of squares + eps) in two factors: values are multiplied by `unit`, a power of two, first and by `rstd` afterwards.
struct row_scale {
    float unit, rstd;
    __device__ __forceinline__ float whole() const { return rstd * unit; }
};

// WAVES wavefronts a row; R accesses of VEC values a thread, or any number, read twice, if R is 0.
template <int DT, int VEC, int WAVES, int R, int TO>
__global__ __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) void fc_rms_norm_kernel(const rms_params p) {
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    struct alignas(VEC) bytes {
        int8_t v[VEC];
    };
    constexpr int PER = 64 * WAVES, ROWS = WAVES > 1 ? 1 : 4, KEEP = R ? R : 1;
    __shared__ float2 slots[2][16];
    const int me = WAVES > 1 ? threadIdx.x : threadIdx.x & 63, accesses = p.C / VEC;
    const int loops = R ? R : (accesses + PER - 1) / PER;
    float g[KEEP][VEC];
    auto read_gamma = [&](int k, float (&to)[VEC]) __attribute__((always_inline)) {
        const int a = me + k * PER;
#pragma unroll
        for (int v = 0; v < VEC; v++) to[v] = p.gamma && a < accesses ? p.gamma[a * VEC + v] : 1.f;
    };
    if constexpr (R > 0 && TO != ONLY_INT8) {
#pragma unroll
        for (int k = 0; k < R; k++) read_gamma(k, g[k]);
    }
    int turn = 0;
    for (long row = (long)blockIdx.x * ROWS + (WAVES > 1 ? 0 : threadIdx.x >> 6); row < p.rows; row += (long)gridDim.x * ROWS) {
        const E *x = (const E *)p.x + row * p.x_row, *res = (const E *)p.residual + row * p.residual_row;
        E *sum = (E *)p.sum + row * p.sum_row;
        V h[KEEP];
        // x + residual; again: where it is stored, from there
        auto read = [&](int k, V &to, bool again) __attribute__((always_inline)) {
            const int a = me + k * PER;
            if (a >= accesses) return;
            if (again && p.sum) {
                to = *(const V *)(sum + a * VEC);
                return;
            }
            to = *(const V *)(x + a * VEC);
            if (p.residual) {
                const V r = *(const V *)(res + a * VEC);
#pragma unroll
                for (int v = 0; v < VEC; v++) to.set(v, to.get(v) + r.get(v));
            }
            if (p.sum && !again) *(V *)(sum + a * VEC) = to;
        };
        // the sum of squares and the largest |h gamma|, of h times unit
        auto measure = [&](bool again, float unit) __attribute__((always_inline)) {
            float2 m = make_float2(0.f, 0.f);
            bool bad = false;
#pragma unroll
            for (int k = 0; k < loops; k++) {
                V &t = h[R ? k : 0];
                if (!R || !again) read(k, t, again);
                if constexpr (R == 0 && TO == TO_INT8) read_gamma(k, g[0]);
                if (me + k * PER >= accesses) continue;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const float s = t.get(v) * unit;
                    if (TO != ONLY_INT8) m.x = __builtin_fmaf(s, s, m.x);
                    if (TO != TO_TYPE) {
                        const float w = TO == ONLY_INT8 ? s : s * g[R ? k : 0][v];
                        m.y = fmaxf(m.y, __builtin_fabsf(w));
                        bad |= !(__builtin_fabsf(w) < __builtin_inff());
                    }
                }
            }
            if (TO != TO_TYPE && bad) m.y = __builtin_inff();      // also where it is NaN, which fmaxf drops
            return join<WAVES>(m, slots, turn++);
        };
        float2 m = measure(false, 1.f);
        row_scale s = {1.f, 1.f};
        if constexpr (TO != ONLY_INT8) {
            float eps = p.eps;
            // Squares that overflow, or vanish beside no eps to speak of: again, of values near 1.
            if (!(m.x < 1e36f) || !(m.y < 1e36f) || (m.x < 1e-20f && eps < 1e-20f)) {
                float2 top = make_float2(0.f, 0.f);
#pragma unroll
                for (int k = 0; k < loops; k++) {
                    V &t = h[R ? k : 0];
                    if (!R) read(k, t, true);
                    if (me + k * PER >= accesses) continue;
#pragma unroll
                    for (int v = 0; v < VEC; v++) top.y = fmaxf(top.y, __builtin_fabsf(t.get(v)));
                }
                top = join<WAVES>(top, slots, turn++);
                if (top.y > 0.f && top.y < __builtin_inff()) {
                    int e = ilogbf(top.y);
                    if (eps > 0.f && ilogbf(eps) / 2 > e) e = ilogbf(eps) / 2;
                    e = e < -120 ? -120 : e > 120 ? 120 : e;
                    s.unit = ldexpf(1.f, -e);
                    eps = ldexpf(eps, -2 * e);
                    m = measure(true, s.unit);
                }
            }
            s.rstd = 1.f / sqrtf(m.x / (float)p.C + eps);
            if (p.rstd && me == 0) p.rstd[row] = s.whole();
        }
        float inv = 0.f;
        if constexpr (TO != TO_TYPE) {
            // y = h unit gamma rstd; q is the same of max |h unit gamma|
            const float top = m.y * s.rstd;
            const bool number = top < __builtin_inff();
            if (top >= kLeastTop && number) inv = 127.f / m.y;
            if (me == 0) p.scale[row] = !number ? __builtin_nanf("") : top >= kLeastTop ? top / 127.f : 0.f;
        }
#pragma unroll
        for (int k = 0; k < loops; k++) {
            V &t = h[R ? k : 0];
            if (!R) read(k, t, true);
            if constexpr (R == 0 && TO != ONLY_INT8) read_gamma(k, g[0]);
            const int a = me + k * PER;
            if (a >= accesses) continue;
            if constexpr (TO == TO_TYPE) {
#pragma unroll
                for (int v = 0; v < VEC; v++) t.set(v, t.get(v) * s.unit * s.rstd * g[R ? k : 0][v]);
                *(V *)((E *)p.y + row * p.y_row + a * VEC) = t;
            } else {
                bytes q;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const float w = TO == ONLY_INT8 ? t.get(v) : t.get(v) * s.unit * g[R ? k : 0][v];
                    q.v[v] = inv > 0.f ? (int8_t)(int)rintf(w * inv) : (int8_t)0;
                }
                *(bytes *)((int8_t *)p.y + row * p.y_row + a * VEC) = q;
            }
        }
    }
}

// dx, and what each workgroup's rows add to dgamma: part[workgroup][C] (WAVES == 1: [wavefront][C]).
template <int DT, int VEC, int WAVES, int R>
__global__ __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) void fc_rms_norm_gradient_kernel(const rms_params p) {
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    constexpr int PER = 64 * WAVES, ROWS = WAVES > 1 ? 1 : 4, KEEP = R ? R : 1;
    __shared__ float2 slots[2][16];
    const int me = WAVES > 1 ? threadIdx.x : threadIdx.x & 63, accesses = p.C / VEC;
    const int loops = R ? R : (accesses + PER - 1) / PER;
    const long first = (long)blockIdx.x * ROWS + (WAVES > 1 ? 0 : threadIdx.x >> 6);
    float *part = p.part ? p.part + first * p.C : nullptr;
    float g[KEEP][VEC], dg[KEEP][VEC];
    auto read_gamma = [&](int k, float (&to)[VEC]) __attribute__((always_inline)) {
        const int a = me + k * PER;
#pragma unroll
        for (int v = 0; v < VEC; v++) to[v] = p.gamma && a < accesses ? p.gamma[a * VEC + v] : 1.f;
    };
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        if constexpr (R > 0) read_gamma(k, g[k]);
#pragma unroll
        for (int v = 0; v < VEC; v++) dg[k][v] = 0.f;
    }
    int turn = 0;
    for (long row = first; row < p.rows; row += (long)gridDim.x * ROWS) {
        const E *hr = (const E *)p.h + row * p.sum_row, *dr = (const E *)p.dy + row * p.dy_row;
        const float rstd = p.rstd[row];
        V h[KEEP], d[KEEP];
        float2 along = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < loops; k++) {
            const int a = me + k * PER, i = R ? k : 0;
            if (a >= accesses) continue;
            h[i] = *(const V *)(hr + a * VEC);
            d[i] = *(const V *)(dr + a * VEC);
            if constexpr (R == 0) read_gamma(k, g[0]);
#pragma unroll
            for (int v = 0; v < VEC; v++) along.x = __builtin_fmaf(g[i][v] * d[i].get(v), h[i].get(v) * rstd, along.x);
        }
        along = join<WAVES>(along, slots, turn++);
        const float mean = along.x / (float)p.C;
#pragma unroll
        for (int k = 0; k < loops; k++) {
            const int a = me + k * PER, i = R ? k : 0;
            if (a >= accesses) continue;
            if constexpr (R == 0) {
                h[0] = *(const V *)(hr + a * VEC);
                d[0] = *(const V *)(dr + a * VEC);
                read_gamma(k, g[0]);
            }
            V more;
            if (p.dsum) more = *(const V *)((const E *)p.dsum + row * p.sum_row + a * VEC);
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                const float xhat = h[i].get(v) * rstd, dy = d[i].get(v);
                if constexpr (R > 0) dg[i][v] = __builtin_fmaf(dy, xhat, dg[i][v]);
                else if (part) {      // a thread's own place, from row to row
                    float *to = part + a * VEC + v;
                    *to = row == first ? dy * xhat : __builtin_fmaf(dy, xhat, *to);
                }
                const float dh = rstd * __builtin_fmaf(-xhat, mean, g[i][v] * dy);
                h[i].set(v, p.dsum ? dh + more.get(v) : dh);
            }
            *(V *)((E *)p.y + row * p.x_row + a * VEC) = h[i];
        }
    }
    if constexpr (R > 0) {
        if (!part) return;
#pragma unroll
        for (int k = 0; k < R; k++) {
            const int a = me + k * PER;
            if (a >= accesses) continue;
#pragma unroll
            for (int v = 0; v < VEC; v++) part[a * VEC + v] = dg[k][v];
        }
    }
}

// dgamma from its parts, always in the same order: 64 channels a workgroup, four wavefronts that share the parts.
__global__ __launch_bounds__(256) void fc_rms_norm_dgamma_kernel(const float *part, float *dgamma, int parts, int C) {
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (c < C) {
        for (int i = wave; i < parts; i += 4) s += part[(long)i * C + c];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < C) dgamma[c] = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

// Accesses are 16 bytes wide, two 16-bit values, or single values.
int width_of(int dtype, uint64_t bits, uint64_t addr) {
    const int w = fc_widest(dtype, bits, addr), most = 16 / (int)fc_elem_size(dtype);
    return w == most ? w : dtype != FC_F32 && w >= 2 ? 2 : 1;
}

// Wavefronts of a row: one, four or sixteen, and whether the row stays in their registers.
struct row_form {
    int waves;
    bool kept;
    long blocks(long rows) const {
        const long want = waves > 1 ? rows : (rows + 3) / 4, most = waves > 4 ? 512 : 2048;
        return want < most ? want : most;
    }
};

constexpr int kAccesses = 4;      // of a thread
row_form form_of(long rows, int C, int vec) {
    const int accesses = C / vec;
    // few rows: as many wavefronts as there are accesses for, a wait for one access each; many: as few as hold the row
    const int least = rows < 1024 ? 1 : kAccesses;
    if (accesses <= 64 * least) return {1, true};
    if (accesses <= 256 * kAccesses) return {4, true};
    return {16, accesses <= 1024 * kAccesses};
}

template <int DT, int VEC, class F>
void with_rows(const row_form &f, F launch) {
    using std::integral_constant;
    typedef integral_constant<int, DT> dt;
    typedef integral_constant<int, VEC> vec;
    if (f.waves == 1) launch(dt(), vec(), integral_constant<int, 1>(), integral_constant<int, kAccesses>());
    else if (f.waves == 4) launch(dt(), vec(), integral_constant<int, 4>(), integral_constant<int, kAccesses>());
    else if (f.kept) launch(dt(), vec(), integral_constant<int, 16>(), integral_constant<int, kAccesses>());
    else launch(dt(), vec(), integral_constant<int, 16>(), integral_constant<int, 0>());
}

template <class F>
void with_kernel(int dtype, int vec, const row_form &f, F launch) {
    if (dtype == FC_F32) return vec == 4 ? with_rows<FC_F32, 4>(f, launch) : with_rows<FC_F32, 1>(f, launch);
    if (dtype == FC_BF16) return vec == 8 ? with_rows<FC_BF16, 8>(f, launch) : vec == 2 ? with_rows<FC_BF16, 2>(f, launch) : with_rows<FC_BF16, 1>(f, launch);
    return vec == 8 ? with_rows<FC_F16, 8>(f, launch) : vec == 2 ? with_rows<FC_F16, 2>(f, launch) : with_rows<FC_F16, 1>(f, launch);
}

template <int TO>
int run(fc_context *ctx, const rms_params &p, int dtype, uint64_t bits, uint64_t addr, const char *name) {
    const int vec = width_of(dtype, bits | (uint64_t)p.C, addr);
    const row_form f = form_of(p.rows, p.C, vec);
    with_kernel(dtype, vec, f, [&](auto dt, auto v, auto waves, auto r) {
        constexpr int W = decltype(waves)::value;
        fc_rms_norm_kernel<decltype(dt)::value, decltype(v)::value, W, decltype(r)::value, TO>
            <<<dim3((unsigned)f.blocks(p.rows)), dim3(W > 4 ? 64 * W : 256), 0, ctx->stream>>>(p);
    });
    FC_LAUNCH_CHECK(ctx, name);
    return FC_OK;
}

bool same(const fc_rms_norm_plan &a, const fc_rms_norm_plan &b) {
    const fc_rms_norm_shape &s = a.shape, &t = b.shape;
    return s.rows == t.rows && s.C == t.C && s.dtype == t.dtype && s.eps == t.eps && s.x_row == t.x_row && s.residual_row == t.residual_row &&
           s.sum_row == t.sum_row && s.y_row == t.y_row && a.parts == b.parts && a.ws_backward_bytes == b.ws_backward_bytes;
}

int check_plan(fc_context *ctx, const fc_rms_norm_plan *plan, const char *what) {
    fc_rms_norm_plan own;
    if (!plan || fc_rms_norm_make_plan(&plan->shape, &own) != FC_OK || !same(*plan, own)) return fail(ctx, FC_ERR_INVALID, what);
    return FC_OK;
}

// What both forward calls check and set.
int forward_params(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x, const void *residual, const float *gamma, void *sum, rms_params &p,
                   uint64_t &bits, uint64_t &addr) {
    const fc_rms_norm_shape &s = plan->shape;
    if (!x) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: null pointer");
    if (sum && !fc_apart(s.rows, s.sum_row, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: rows of the sum overlap");
    bits = (uint64_t)s.x_row;
    addr = (uint64_t)x;
    if (residual) {
        bits |= (uint64_t)s.residual_row;
        addr |= (uint64_t)residual;
    }
    if (sum) {
        bits |= (uint64_t)s.sum_row;
        addr |= (uint64_t)sum;
    }
    if ((addr & (fc_elem_size(s.dtype) - 1)) || ((uint64_t)gamma & 3)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: unaligned pointer");
    p.x = x; p.residual = residual; p.sum = sum; p.gamma = gamma;
    p.rows = s.rows; p.C = s.C; p.eps = s.eps;
    p.x_row = s.x_row; p.residual_row = s.residual_row; p.sum_row = s.sum_row; p.y_row = s.y_row;
    return FC_OK;
}

}  // namespace

extern "C" int fc_rms_norm_make_plan(const fc_rms_norm_shape *s, fc_rms_norm_plan *plan) {
    if (!plan || !s || s->rows < 1 || s->C < 1 || !fc_dtype_ok(s->dtype) || !(s->eps >= 0.f) || !(s->eps < __builtin_inff())) return FC_ERR_INVALID;
    if (s->x_row < 0 || s->residual_row < 0 || s->sum_row < 0 || s->y_row < 0) return FC_ERR_INVALID;
    if (s->rows > kMostRows || s->C > kMostChannels) return FC_ERR_UNSUPPORTED;
    *plan = {};
    plan->shape = *s;
    // wherever the tensors begin: the most parts that any access width leads to
    const int widths[3] = {16 / (int)fc_elem_size(s->dtype), 2, 1};
    for (int w : widths) {
        const row_form f = form_of(s->rows, s->C, w);
        const long parts = f.blocks(s->rows) * (f.waves == 1 ? 4 : 1);
        if (parts > plan->parts) plan->parts = (int)parts;
    }
    plan->ws_backward_bytes = (size_t)plan->parts * s->C * sizeof(float);
    return FC_OK;
}

extern "C" int fc_rms_norm(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x_dev, const void *residual_dev, const float *gamma_dev,
                           void *sum_dev, void *y_dev, float *rstd_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_rms_norm: not a plan of fc_rms_norm_make_plan")) return FC_ERR_INVALID;
    const fc_rms_norm_shape &s = plan->shape;
    rms_params p = {};
    uint64_t bits, addr;
    const int rc = forward_params(ctx, plan, x_dev, residual_dev, gamma_dev, sum_dev, p, bits, addr);
    if (rc) return rc;
    if (!y_dev) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: null pointer");
    if (((uint64_t)y_dev & (fc_elem_size(s.dtype) - 1)) || ((uint64_t)rstd_dev & 3)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: unaligned pointer");
    if (!fc_apart(s.rows, s.y_row, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: rows of y overlap");
    p.y = y_dev;
    p.rstd = rstd_dev;
    const fc_device_scope on(ctx);
    return run<TO_TYPE>(ctx, p, s.dtype, bits | (uint64_t)s.y_row, addr | (uint64_t)y_dev, "fc_rms_norm");
}

// Rows of bytes: an access of n values writes n of them.
static void add_bytes(int dtype, long row, const void *q, uint64_t &bits, uint64_t &addr) {
    bits |= (uint64_t)row;
    addr |= (uint64_t)q * fc_elem_size(dtype);
}

extern "C" int fc_rms_norm_int8(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x_dev, const void *residual_dev, const float *gamma_dev,
                                void *sum_dev, int8_t *q_dev, float *scale_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_rms_norm_int8: not a plan of fc_rms_norm_make_plan")) return FC_ERR_INVALID;
    const fc_rms_norm_shape &s = plan->shape;
    rms_params p = {};
    uint64_t bits, addr;
    const int rc = forward_params(ctx, plan, x_dev, residual_dev, gamma_dev, sum_dev, p, bits, addr);
    if (rc) return rc;
    if (!q_dev || !scale_dev) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_int8: null pointer");
    if ((uint64_t)scale_dev & 3) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_int8: unaligned pointer");
    if (!fc_apart(s.rows, s.y_row, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_int8: rows of q overlap");
    p.y = q_dev;
    p.scale = scale_dev;
    add_bytes(s.dtype, s.y_row, q_dev, bits, addr);
    const fc_device_scope on(ctx);
    return run<TO_INT8>(ctx, p, s.dtype, bits, addr, "fc_rms_norm_int8");
}

extern "C" int fc_quantize_rows(fc_context *ctx, long rows, int C, int dtype, const void *x_dev, long x_row, int8_t *q_dev, long q_row,
                                float *scale_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (rows < 1 || C < 1 || !fc_dtype_ok(dtype) || x_row < 0 || q_row < 0) return fail(ctx, FC_ERR_INVALID, "fc_quantize_rows: bad shape");
    if (rows > kMostRows || C > kMostChannels) return fail(ctx, FC_ERR_UNSUPPORTED, "fc_quantize_rows: more than 2^40 rows or 2^20 channels");
    if (!x_dev || !q_dev || !scale_dev) return fail(ctx, FC_ERR_INVALID, "fc_quantize_rows: null pointer");
    if (((uint64_t)x_dev & (fc_elem_size(dtype) - 1)) || ((uint64_t)scale_dev & 3)) return fail(ctx, FC_ERR_INVALID, "fc_quantize_rows: unaligned pointer");
    if (!fc_apart(rows, q_row, C)) return fail(ctx, FC_ERR_INVALID, "fc_quantize_rows: rows of q overlap");
    rms_params p = {};
    p.x = x_dev; p.y = q_dev; p.scale = scale_dev;
    p.rows = rows; p.C = C; p.x_row = x_row; p.y_row = q_row;
    uint64_t bits = (uint64_t)x_row, addr = (uint64_t)x_dev;
    add_bytes(dtype, q_row, q_dev, bits, addr);
    const fc_device_scope on(ctx);
    return run<ONLY_INT8>(ctx, p, dtype, bits, addr, "fc_quantize_rows");
}

extern "C" int fc_rms_norm_backward(fc_context *ctx, const fc_rms_norm_plan *plan, const void *dy_dev, const void *sum_dev, const float *gamma_dev,
                                    const float *rstd_dev, const void *dsum_dev, void *dx_dev, float *dgamma_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_rms_norm_backward: not a plan of fc_rms_norm_make_plan")) return FC_ERR_INVALID;
    const fc_rms_norm_shape &s = plan->shape;
    if (!dy_dev || !sum_dev || !rstd_dev || !dx_dev || (dgamma_dev && !ws_dev)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_backward: null pointer");
    const uint64_t addr = (uint64_t)dy_dev | (uint64_t)sum_dev | (uint64_t)dsum_dev | (uint64_t)dx_dev;
    if ((addr & (fc_elem_size(s.dtype) - 1)) || (((uint64_t)gamma_dev | (uint64_t)rstd_dev | (uint64_t)dgamma_dev | (uint64_t)ws_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_backward: unaligned pointer");
    if (!fc_apart(s.rows, s.x_row, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_backward: rows of dx overlap");
    rms_params p = {};
    p.dy = dy_dev; p.h = sum_dev; p.dsum = dsum_dev; p.y = dx_dev; p.gamma = gamma_dev;
    p.rstd = const_cast<float *>(rstd_dev);      // only read
    p.part = dgamma_dev ? (float *)ws_dev : nullptr;
    p.rows = s.rows; p.C = s.C;
    p.x_row = s.x_row; p.sum_row = s.sum_row; p.dy_row = s.y_row;
    const int vec = width_of(s.dtype, (uint64_t)s.C | (uint64_t)s.x_row | (uint64_t)s.sum_row | (uint64_t)s.y_row, addr);
    const row_form f = form_of(s.rows, s.C, vec);
    const long blocks = f.blocks(s.rows);
    const fc_device_scope on(ctx);
    with_kernel(s.dtype, vec, f, [&](auto dt, auto v, auto waves, auto r) {
        constexpr int W = decltype(waves)::value;
        fc_rms_norm_gradient_kernel<decltype(dt)::value, decltype(v)::value, W, decltype(r)::value>
            <<<dim3((unsigned)blocks), dim3(W > 4 ? 64 * W : 256), 0, ctx->stream>>>(p);
    });
    FC_LAUNCH_CHECK(ctx, "fc_rms_norm_gradient_kernel");
    if (!dgamma_dev) return FC_OK;
    // rows past the last have no wavefront: parts of wavefronts that had none are not written
    const long parts = f.waves > 1 ? blocks : blocks * 4 < s.rows ? blocks * 4 : s.rows;
    fc_rms_norm_dgamma_kernel<<<dim3((unsigned)((s.C + 63) / 64)), dim3(256), 0, ctx->stream>>>(p.part, dgamma_dev, (int)parts, s.C);
    FC_LAUNCH_CHECK(ctx, "fc_rms_norm_dgamma_kernel");
    return FC_OK;
}
