// RMS norm over rows of channels, after the addition of a residual, with a result in the rows' type or in 8 bits with a scale for each row:
//
//   h = x + residual, rounded to the rows' type,   rstd = 1/sqrt(mean of h^2 + eps),   y = h * rstd * gamma
//   8 bits: scale = max |y| / 127,  q = y / scale rounded to nearest, ties to even, of y in fp32
//   dh = rstd * (gamma dy - xhat * mean of (gamma dy xhat)) + dsum,   dgamma = sum over rows of dy xhat,   xhat = h * rstd
//
// Bound by memory: about 10 operations a value against 8 bytes in 16-bit types.  A row stays in the registers of its wavefronts between its
// two uses, gamma from row to row.  12544 rows of 2048, bf16, with residual and sum: 32 us in the kernel (206 MB, some of them from the last cache; 41 us where they
// come from memory, 5.0 TB/s); 9800 rows of 771, fp32: 19 to 25 us, gradients 18 to 22 and 4 for the sums of dgamma.  In 8 bits every step is one fp32 operation, as
// it is written: a value on the border between two steps goes where it goes for whoever rounds y to fp32 and divides.  That takes the norm first and the largest y then,
// two waits a row: 36 us at the first size, rows to 8 bits 15.3 (77 MB, some of them from the last cache); one row of 2048 4.4 to 4.6 and 4.1 us, an empty launch's time.
#include <type_traits>

#include "token_types.h"

namespace {

constexpr long kMostRows = 1l << 40;
constexpr int kMostChannels = 1 << 20;
// Rows whose largest value is smaller are zeros in 8 bits, with a scale of 0: their scale would leave the normal numbers.
constexpr float kLeastTop = 0x1p-110f;
constexpr float kLeastDivisor = 0x1p-100f;      // a remainder of half a step by it has its last place at 2^-147

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

// Values of a 16-byte access.
template <int DT>
constexpr int kVec = DT == FC_F32 ? 4 : 8;

// A thread's share of a row: R accesses of 16 bytes in registers (any number, read again for each use, if R is 0), and one value of those that fill no
// access.  Accesses past the row's last read that one again and count as zeros: a load behind a branch would keep the others waiting.
template <int DT, int WAVES, int R>
struct row_share {
    static constexpr int VEC = kVec<DT>, PER = 64 * WAVES, KEEP = R ? R : 1;
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    int me, full, tail;      // full: accesses of the row; tail: values that are left
    __device__ __forceinline__ explicit row_share(int C)
        : me(WAVES > 1 ? threadIdx.x : threadIdx.x & 63), full(C / VEC), tail(C - C / VEC * VEC) {}
    __device__ __forceinline__ bool has(int k) const { return me + k * PER < full; }
    __device__ __forceinline__ int at(int k) const { return (has(k) ? me + k * PER : full - 1) * VEC; }
    __device__ __forceinline__ int last() const { return full * VEC + (me < tail ? me : 0); }      // the single value's place
    __device__ __forceinline__ void read(V (&to)[KEEP], fc_vec<DT, 1> &one, const E *row) const {
        if (full) {
#pragma unroll
            for (int k = 0; k < R; k++) __builtin_memcpy(&to[k], row + at(k), sizeof(V));
        }
        if (tail) one.v[0] = row[last()];
    }
    __device__ __forceinline__ void clear(V (&of)[KEEP], fc_vec<DT, 1> &one) const {
        const V zeros = {};
#pragma unroll
        for (int k = 0; k < R; k++)
            if (!has(k)) of[k] = zeros;
        if (me >= tail) one.v[0] = (E)0.f;
    }
    __device__ __forceinline__ void read_gamma(float (&g)[KEEP][VEC], float &one, const float *gamma) const {
#pragma unroll
        for (int k = 0; k < KEEP; k++)
#pragma unroll
            for (int v = 0; v < VEC; v++) g[k][v] = 1.f;
        one = 1.f;
        if (!gamma) return;
        if (full) {
#pragma unroll
            for (int k = 0; k < R; k++) __builtin_memcpy(g[k], gamma + at(k), sizeof g[k]);
        }
        if (tail) one = gamma[last()];
    }
};

// WAVES wavefronts a row.
template <int DT, int WAVES, int R, int TO>
__global__ __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) void fc_rms_norm_kernel(const rms_params p) {
    typedef row_share<DT, WAVES, R> share;
    typedef typename share::V V;
    typedef typename share::E E;
    typedef fc_vec<DT, 1> one;
    constexpr int VEC = share::VEC, PER = share::PER, ROWS = WAVES > 1 ? 1 : 4, KEEP = share::KEEP;
    __shared__ float2 slots[2][16];
    const share of(p.C);
    float g[KEEP][VEC], g1 = 1.f;
    if constexpr (TO != ONLY_INT8) of.read_gamma(g, g1, p.gamma);
    int turn = 0;
    for (long row = (long)blockIdx.x * ROWS + (WAVES > 1 ? 0 : threadIdx.x >> 6); row < p.rows; row += (long)gridDim.x * ROWS) {
        const E *x = (const E *)p.x + row * p.x_row, *res = (const E *)p.residual + row * p.residual_row;
        E *sum = (E *)p.sum + row * p.sum_row;
        V h[KEEP];
        one h1;
        h1.v[0] = (E)0.f;
        auto add = [](auto &a, const auto &b, int n) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < n; v++) a.set(v, a.get(v) + b.get(v));
        };
        if constexpr (R > 0) {
            of.read(h, h1, x);
            if (p.residual) {
                V r[KEEP];
                one r1 = h1;
                of.read(r, r1, res);
#pragma unroll
                for (int k = 0; k < R; k++) add(h[k], r[k], VEC);
                add(h1, r1, 1);
            }
            of.clear(h, h1);
            if (p.sum) {
#pragma unroll
                for (int k = 0; k < R; k++)
                    if (of.has(k)) __builtin_memcpy(sum + of.at(k), &h[k], sizeof(V));
                if (of.me < of.tail) sum[of.last()] = h1.v[0];
            }
        }
        // f(values of h, of gamma, how many, where): what the thread has of the row.  Where it is not kept it is read, and the sum written the first time.
        auto visit = [&](bool again, auto f) __attribute__((always_inline)) {
            if constexpr (R > 0) {
#pragma unroll
                for (int k = 0; k < R; k++) f(h[k], g[k], std::integral_constant<int, VEC>(), of.at(k), of.has(k));
                f(h1, &g1, std::integral_constant<int, 1>(), of.last(), of.me < of.tail);
            } else {
                auto part = [&](auto &t, auto &r, const float *gamma, auto n, int at) __attribute__((always_inline)) {
                    const bool stored = again && p.sum;
                    __builtin_memcpy(&t, (stored ? sum : x) + at, sizeof t);
                    if (p.residual && !stored) {
                        __builtin_memcpy(&r, res + at, sizeof r);
                        add(t, r, n);
                    }
                    if (p.sum && !again) __builtin_memcpy(sum + at, &t, sizeof t);
                    f(t, gamma, n, at, true);
                };
                for (int a = of.me; a < of.full; a += PER) {
                    V t, r;
                    if (TO != ONLY_INT8 && p.gamma) __builtin_memcpy(g[0], p.gamma + a * VEC, sizeof g[0]);
                    part(t, r, g[0], std::integral_constant<int, VEC>(), a * VEC);
                }
                if (of.me < of.tail) {
                    one t, r;
                    part(t, r, &g1, std::integral_constant<int, 1>(), of.last());
                }
            }
        };
        // the sum of squares of h times unit
        auto squares = [&](bool again, float unit) __attribute__((always_inline)) {
            float sum = 0.f;
            visit(again, [&](const auto &t, const float *, auto n, int, bool) __attribute__((always_inline)) {
#pragma unroll
                for (int v = 0; v < n; v++) {
                    const float s = t.get(v) * unit;
                    sum = __builtin_fmaf(s, s, sum);
                }
            });
            return join<WAVES>(make_float2(sum, 0.f), slots, turn++).x;
        };
        row_scale s = {1.f, 1.f};
        if constexpr (TO != ONLY_INT8) {
            float sum = squares(false, 1.f), eps = p.eps;
            // Squares that overflow, or vanish beside no eps to speak of: again, of values near 1.
            if (!(sum < 1e36f) || (sum < 1e-20f && eps < 1e-20f)) {
                float top = 0.f;
                visit(true, [&](const auto &t, const float *, auto n, int, bool) __attribute__((always_inline)) {
#pragma unroll
                    for (int v = 0; v < n; v++) top = fmaxf(top, __builtin_fabsf(t.get(v)));
                });
                top = join<WAVES>(make_float2(0.f, top), slots, turn++).y;
                if (top > 0.f && top < __builtin_inff()) {
                    int e = ilogbf(top);
                    if (eps > 0.f && ilogbf(eps) / 2 > e) e = ilogbf(eps) / 2;
                    e = e < -120 ? -120 : e > 120 ? 120 : e;
                    s.unit = ldexpf(1.f, -e);
                    eps = ldexpf(eps, -2 * e);
                    sum = squares(true, s.unit);
                }
            }
            s.rstd = 1.f / sqrtf(sum / (float)p.C + eps);
            if (p.rstd && of.me == 0) p.rstd[row] = s.whole();
        }
        auto result = [&](float h, float gamma) __attribute__((always_inline)) { return TO == ONLY_INT8 ? h : h * s.unit * s.rstd * gamma; };
        float scale = 0.f, inv = 0.f;
        if constexpr (TO != TO_TYPE) {
            float top = 0.f;
            bool bad = false;
            visit(TO != ONLY_INT8, [&](const auto &t, const float *gamma, auto n, int, bool) __attribute__((always_inline)) {
#pragma unroll
                for (int v = 0; v < n; v++) {
                    const float y = __builtin_fabsf(result(t.get(v), gamma[v]));
                    top = fmaxf(top, y);
                    bad |= !(y < __builtin_inff());
                }
            });
            if (bad) top = __builtin_inff();      // also where it is NaN, which fmaxf drops
            top = join<WAVES>(make_float2(0.f, top), slots, turn++).y;
            const bool number = top < __builtin_inff();
            if (top >= kLeastTop && number) {
                scale = top / 127.f;
                inv = 1.f / scale;
            }
            if (of.me == 0) p.scale[row] = number ? scale : __builtin_nanf("");
        }
        // y / scale, rounded as a division rounds it: y times 1 / scale, which is off by less than two last places, takes what is left of y twice, the second time from
        // a last place off at most, so that the remainder is exact and what it adds is off by less than any quotient lies from the middle of two floats (Markstein,
        // Computation of elementary functions on the IBM RISC System/6000 processor, 1990).  Rows to 8 bits, 12544 of 2048, bf16: 15.3 us, 21.5 where a division decides
        // next to a border, 13.5 with the first product alone.
        auto quotient = [&](float y) __attribute__((always_inline)) {
            float q = y * inv;
            q = __builtin_fmaf(__builtin_fmaf(-q, scale, y), inv, q);
            return __builtin_fmaf(__builtin_fmaf(-q, scale, y), inv, q);
        };
        auto write = [&](auto smallest) __attribute__((always_inline)) {
            visit(true, [&](const auto &t, const float *gamma, auto n, int at, bool there) __attribute__((always_inline)) {
                if constexpr (TO == TO_TYPE) {
                    auto y = t;
#pragma unroll
                    for (int v = 0; v < n; v++) y.set(v, result(t.get(v), gamma[v]));
                    if (there) __builtin_memcpy((E *)p.y + row * p.y_row + at, &y, sizeof y);
                } else {
                    int8_t q[n];
#pragma unroll
                    for (int v = 0; v < n; v++) {
                        const float y = result(t.get(v), gamma[v]);
                        q[v] = smallest ? scale > 0.f ? (int8_t)(int)rintf(y / scale) : (int8_t)0 : (int8_t)(int)rintf(quotient(y));
                    }
                    if (there) __builtin_memcpy((int8_t *)p.y + row * p.y_row + at, q, n);
                }
            });
        };
        if (TO == TO_TYPE || scale >= kLeastDivisor) write(std::false_type());
        else write(std::true_type());
    }
}

// dx, and what each workgroup's rows add to dgamma: part[workgroup][C].
template <int DT, int WAVES, int R>
__global__ __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) void fc_rms_norm_gradient_kernel(const rms_params p) {
    typedef row_share<DT, WAVES, R> share;
    typedef typename share::V V;
    typedef typename share::E E;
    typedef fc_vec<DT, 1> one;
    constexpr int VEC = share::VEC, PER = share::PER, ROWS = WAVES > 1 ? 1 : 4, KEEP = share::KEEP;
    __shared__ float2 slots[2][16];
    const share of(p.C);
    const int wave = threadIdx.x >> 6;
    const long first = (long)blockIdx.x * ROWS + (WAVES > 1 ? 0 : wave);
    float *part = p.part ? p.part + (long)blockIdx.x * p.C : nullptr;
    float g[KEEP][VEC], dg[KEEP][VEC], g1 = 1.f, dg1 = 0.f;
    of.read_gamma(g, g1, p.gamma);
#pragma unroll
    for (int k = 0; k < KEEP; k++)
#pragma unroll
        for (int v = 0; v < VEC; v++) dg[k][v] = 0.f;
    int turn = 0;
    for (long row = first; row < p.rows; row += (long)gridDim.x * ROWS) {
        const E *hr = (const E *)p.h + row * p.sum_row, *dr = (const E *)p.dy + row * p.dy_row, *more = (const E *)p.dsum + row * p.sum_row;
        E *dx = (E *)p.y + row * p.x_row;
        const float rstd = p.rstd[row];
        V h[KEEP], d[KEEP], m[KEEP];
        one h1, d1, m1;
        h1.v[0] = d1.v[0] = m1.v[0] = (E)0.f;
        if constexpr (R > 0) {
            of.read(h, h1, hr);
            of.read(d, d1, dr);
            if (p.dsum) of.read(m, m1, more);
            of.clear(h, h1);
            of.clear(d, d1);
        }
        // f(h, dy, dsum, gamma, its gradient, how many, where): what the thread has of the row
        auto visit = [&](auto f) __attribute__((always_inline)) {
            if constexpr (R > 0) {
#pragma unroll
                for (int k = 0; k < R; k++) f(h[k], d[k], m[k], g[k], dg[k], std::integral_constant<int, VEC>(), of.at(k), of.has(k));
                f(h1, d1, m1, &g1, &dg1, std::integral_constant<int, 1>(), of.last(), of.me < of.tail);
            } else {
                auto some = [&](auto &a, auto &b, auto &c, float *gamma, auto n, int at) __attribute__((always_inline)) {
                    __builtin_memcpy(&a, hr + at, sizeof a);
                    __builtin_memcpy(&b, dr + at, sizeof b);
                    if (p.dsum) __builtin_memcpy(&c, more + at, sizeof c);
                    if (p.gamma) __builtin_memcpy(gamma, p.gamma + at, n * sizeof(float));
                    f(a, b, c, gamma, part ? part + at : nullptr, n, at, true);
                };
                for (int a = of.me; a < of.full; a += PER) some(h[0], d[0], m[0], g[0], std::integral_constant<int, VEC>(), a * VEC);
                if (of.me < of.tail) some(h1, d1, m1, &g1, std::integral_constant<int, 1>(), of.last());
            }
        };
        float2 along = make_float2(0.f, 0.f);
        visit([&](const auto &a, const auto &b, const auto &, const float *gamma, float *, auto n, int, bool) __attribute__((always_inline)) {
#pragma unroll
            for (int v = 0; v < n; v++) along.x = __builtin_fmaf(gamma[v] * b.get(v), a.get(v) * rstd, along.x);
        });
        along = join<WAVES>(along, slots, turn++);
        const float mean = along.x / (float)p.C;
        visit([&](const auto &a, const auto &b, const auto &c, const float *gamma, float *dgamma, auto n, int at, bool there) __attribute__((always_inline)) {
            auto out = a;
#pragma unroll
            for (int v = 0; v < n; v++) {
                const float xhat = a.get(v) * rstd, dy = b.get(v);
                if constexpr (R > 0) dgamma[v] = __builtin_fmaf(dy, xhat, dgamma[v]);
                else if (dgamma) dgamma[v] = row == first ? dy * xhat : __builtin_fmaf(dy, xhat, dgamma[v]);      // a thread's own place, from row to row
                const float dh = rstd * __builtin_fmaf(-xhat, mean, gamma[v] * dy);
                out.set(v, p.dsum ? dh + c.get(v) : dh);
            }
            if (there) __builtin_memcpy(dx + at, &out, sizeof out);
        });
    }
    if constexpr (R > 0) {
        if (!part) return;
        constexpr int WIDTH = 64 * (R * VEC + 1);
        __shared__ float others[WAVES > 1 ? 1 : 3][WAVES > 1 ? 1 : WIDTH];      // four rows at once: their wavefronts' sums
        if constexpr (WAVES == 1) {
            if (wave) {
#pragma unroll
                for (int k = 0; k < R; k++)
#pragma unroll
                    for (int v = 0; v < VEC; v++) others[wave - 1][(k * VEC + v) * 64 + of.me] = dg[k][v];
                others[wave - 1][R * VEC * 64 + of.me] = dg1;
            }
            __syncthreads();
            if (wave) return;
#pragma unroll
            for (int k = 0; k < R; k++)
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const int i = (k * VEC + v) * 64 + of.me;
                    dg[k][v] = (dg[k][v] + others[0][i]) + (others[1][i] + others[2][i]);
                }
            const int i = R * VEC * 64 + of.me;
            dg1 = (dg1 + others[0][i]) + (others[1][i] + others[2][i]);
        }
#pragma unroll
        for (int k = 0; k < R; k++)
            if (of.has(k)) __builtin_memcpy(part + of.at(k), dg[k], sizeof dg[k]);
        if (of.me < of.tail) part[of.last()] = dg1;
    }
}

__global__ __launch_bounds__(kPartThreads) void fc_rms_norm_dgamma_kernel(const float *part, float *dgamma, int parts, int C) {
    long c;
    float s;
    if (fc_sum_parts(part, parts, C, c, s)) dgamma[c] = s;
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

// Workgroups; each of the gradients' leaves a part of dgamma.  12544 rows of 2048, bf16: 33.8, 32.5 and 33.9 us with 1024, 2048 and 8192, gradients 32.2, 34.2, 36.0
// and 38.2 with 256, 512, 768 and 1024; 4000 rows of 2048, fp32: gradients 28.1, 20.8, 20.7 and 23.0.  Rows of one access a thread need few registers, so that more
// workgroups are on their way at once: 100000 rows of 256, bf16, gradients 48.4, 35.3 and 38.7 with 512, 1024 and 2048, the norm 35.7, 34.6 and 35.0 with 2048,
// 4096 and 8192 (133 and 65 where four accesses are kept).
constexpr long kBlocks = 2048, kBlocksBackward = 512, kNarrow = 2;
// Wavefronts of a row: one, four or sixteen, and the accesses that each of their threads keeps in registers: one, two, four or, where that is too few, none.
// 50000 rows of 600, bf16: gradients 36.7 us with two and 76.6 with four, the norm 39.7 and 43.0.
struct row_form {
    int waves, kept;
    // workgroups, each of which takes rows until there are none
    long blocks(long rows, long most) const {
        const long want = waves > 1 ? rows : (rows + 3) / 4;
        if (waves > 4) most /= 4;
        if (kept == 1) most *= kNarrow;
        return want < most ? want : most;
    }
};

constexpr int kAccesses = 4;      // of a thread
// As few wavefronts as hold the row: nobody waits for another.  12544 rows of 2048, bf16: 32.5 us by one wavefront and 46.4 by four, gradients 35.8 and 78.8.
row_form form_of(int C, int dtype) {
    const int vec = dtype == FC_F32 ? 4 : 8, accesses = (C + vec - 1) / vec;
    if (accesses <= 64) return {1, 1};
    if (accesses <= 128) return {1, 2};
    if (accesses <= 64 * kAccesses) return {1, kAccesses};
    if (accesses <= 256 * kAccesses) return {4, kAccesses};
    return {16, accesses <= 1024 * kAccesses ? kAccesses : 0};
}

template <int DT, class F>
void with_rows(const row_form &f, F launch) {
    using std::integral_constant;
    typedef integral_constant<int, DT> dt;
    if (f.kept == 1) launch(dt(), integral_constant<int, 1>(), integral_constant<int, 1>());
    else if (f.kept == 2) launch(dt(), integral_constant<int, 1>(), integral_constant<int, 2>());
    else if (f.waves == 1) launch(dt(), integral_constant<int, 1>(), integral_constant<int, kAccesses>());
    else if (f.waves == 4) launch(dt(), integral_constant<int, 4>(), integral_constant<int, kAccesses>());
    else if (f.kept) launch(dt(), integral_constant<int, 16>(), integral_constant<int, kAccesses>());
    else launch(dt(), integral_constant<int, 16>(), integral_constant<int, 0>());
}

template <class F>
void with_kernel(int dtype, const row_form &f, F launch) {
    if (dtype == FC_F32) return with_rows<FC_F32>(f, launch);
    if (dtype == FC_BF16) return with_rows<FC_BF16>(f, launch);
    return with_rows<FC_F16>(f, launch);
}

template <int TO>
int run(fc_context *ctx, const rms_params &p, int dtype, const char *name) {
    const row_form f = form_of(p.C, dtype);
    const fc_device_scope on(ctx);
    with_kernel(dtype, f, [&](auto dt, auto waves, auto r) {
        constexpr int W = decltype(waves)::value;
        fc_rms_norm_kernel<decltype(dt)::value, W, decltype(r)::value, TO>
            <<<dim3((unsigned)f.blocks(p.rows, kBlocks)), dim3(W > 4 ? 64 * W : 256), 0, ctx->stream>>>(p);
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
int forward_params(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x, const void *residual, const float *gamma, void *sum, rms_params &p) {
    const fc_rms_norm_shape &s = plan->shape;
    if (!x) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: null pointer");
    if (sum && !fc_apart(s.rows, s.sum_row, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: rows of the sum overlap");
    const uint64_t addr = (uint64_t)x | (uint64_t)residual | (uint64_t)sum;
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
    plan->parts = (int)form_of(s->C, s->dtype).blocks(s->rows, kBlocksBackward);
    plan->ws_backward_bytes = (size_t)plan->parts * s->C * sizeof(float);
    return FC_OK;
}

extern "C" int fc_rms_norm(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x_dev, const void *residual_dev, const float *gamma_dev,
                           void *sum_dev, void *y_dev, float *rstd_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_rms_norm: not a plan of fc_rms_norm_make_plan")) return FC_ERR_INVALID;
    const fc_rms_norm_shape &s = plan->shape;
    rms_params p = {};
    const int rc = forward_params(ctx, plan, x_dev, residual_dev, gamma_dev, sum_dev, p);
    if (rc) return rc;
    if (!y_dev) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: null pointer");
    if (((uint64_t)y_dev & (fc_elem_size(s.dtype) - 1)) || ((uint64_t)rstd_dev & 3)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: unaligned pointer");
    if (!fc_apart(s.rows, s.y_row, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm: rows of y overlap");
    p.y = y_dev;
    p.rstd = rstd_dev;
    return run<TO_TYPE>(ctx, p, s.dtype, "fc_rms_norm");
}

extern "C" int fc_rms_norm_int8(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x_dev, const void *residual_dev, const float *gamma_dev,
                                void *sum_dev, int8_t *q_dev, float *scale_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_rms_norm_int8: not a plan of fc_rms_norm_make_plan")) return FC_ERR_INVALID;
    const fc_rms_norm_shape &s = plan->shape;
    rms_params p = {};
    const int rc = forward_params(ctx, plan, x_dev, residual_dev, gamma_dev, sum_dev, p);
    if (rc) return rc;
    if (!q_dev || !scale_dev) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_int8: null pointer");
    if ((uint64_t)scale_dev & 3) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_int8: unaligned pointer");
    if (!fc_apart(s.rows, s.y_row, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_rms_norm_int8: rows of q overlap");
    p.y = q_dev;
    p.scale = scale_dev;
    return run<TO_INT8>(ctx, p, s.dtype, "fc_rms_norm_int8");
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
    return run<ONLY_INT8>(ctx, p, dtype, "fc_quantize_rows");
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
    const row_form f = form_of(s.C, s.dtype);
    const fc_device_scope on(ctx);
    with_kernel(s.dtype, f, [&](auto dt, auto waves, auto r) {
        constexpr int W = decltype(waves)::value;
        fc_rms_norm_gradient_kernel<decltype(dt)::value, W, decltype(r)::value><<<dim3((unsigned)plan->parts), dim3(W > 4 ? 64 * W : 256), 0, ctx->stream>>>(p);
    });
    FC_LAUNCH_CHECK(ctx, "fc_rms_norm_gradient_kernel");
    if (!dgamma_dev) return FC_OK;
    fc_rms_norm_dgamma_kernel<<<dim3((unsigned)((s.C + kPartValues - 1) / kPartValues)), dim3(kPartThreads), 0, ctx->stream>>>(p.part, dgamma_dev, plan->parts, s.C);
    FC_LAUNCH_CHECK(ctx, "fc_rms_norm_dgamma_kernel");
    return FC_OK;
}
