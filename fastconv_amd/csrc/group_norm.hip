// Group norm with an activation over channels-last pixels, forward and backward.
//
//   xhat = (x - mean) * rstd,  y = act(gamma * xhat + beta),  mean and variance over the P * C/G values of a group
//   dz = dy * act'(z),  dbeta = sum dz,  dgamma = sum dz * xhat
//   dx = rstd * (gamma dz - (s1 + xhat s2) / (P * C/G)),  s1 = sum over the group of gamma dz,  s2 = of gamma dz xhat
//
// Bound by memory: about 10 operations an element against 4 bytes in 16-bit types.  The first y needs the last x of its
// group.  Where a few channels' pixels fit the registers of a workgroup, they wait there: one launch, x read once (1 image of 14x14x512 in bf16
// 6.5 us, the time of a launch with three waits on memory; 32 of 56x56x256 in fp32 51 us, 4.0 TB/s).  Otherwise the pixels of an image are cut into
// chunks: one launch leaves each chunk's statistics, the next joins them and writes the result, reading x a second time, from the 256 MB cache
// where x fits that (32 images of 224x224x64 in bf16, 206 MB: 40 us at 5.1 TB/s and 75 at 5.5).  Backward likewise, with dy beside x (32 of 56x56x256 in
// fp32: sums 44 us, 4.7 TB/s; gradients 52, 5.9 TB/s).
// A thread keeps to one column of 4 to 16 bytes of channels and walks down the pixels, so that whatever belongs to a channel
// stays in registers; a wavefront reads whole lines.
// Statistics are joined, never subtracted: a thread forms the mean of each batch of pixels and the squares of what differs
// from it, and joins batches, threads, channels and chunks by
//   n = na + nb,  mean = ma + d nb/n,  M2 = M2a + M2b + d^2 na nb/n,  d = mb - ma
// (Chan, Golub and LeVeque, "Updating formulae and a pairwise algorithm for computing sample variances", 1979).
#include <type_traits>

#include "token_types.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxGroupChannels = 4096;
constexpr long kMostThreads = 1l << 32;                // of a launch, not reached
constexpr double kCacheBytes = 256.0 * (1 << 20);      // the last cache before HBM

struct norm_params {
    const void *x, *dy;
    void *y;                 // or dx
    const float *gamma, *beta;
    float *mean, *rstd;
    float2 *part;            // forward: (mean, M2) [N][G][chunks]; backward: (s1, s2) likewise
    float2 *channel_part;    // backward: (sum dz, sum dz xhat) [N][chunks][C]
    float *dgamma, *dbeta;
    long P, chunk;           // pixels of an image, and of a chunk
    int N, C, G, Cg;
    int span, spans, chunks;
    bool past_cache;
    int reduce_blocks;       // workgroups of the backward pass's second launch that add up channel_part
    float eps;
    long x_image, x_pixel, y_image, y_pixel;
};

// 1 + erf(z / sqrt(2)) from e = exp(-z^2 / 2), as 1 - erf(|x|) = t Q(t) e with t = 1/(1 + c |x|), x = z / sqrt(2), Q a polynomial.  Where z is
// negative that is the answer itself, as exact in proportion to it far out as near 0; 1 + erf would cancel.
// 16 bits: c = 0.3275911 and five terms, to 1.5e-7 (Hastings' formula, number 7.1.26 in Abramowitz and Stegun's handbook).  fp32: c = 0.375 and nine
// terms, fitted to erfc(x) exp(x^2) / t for x up to 9.6 so that the largest relative error is least, 1.1e-8.  On normal z all of GELU then errs by
// 4e-8 of its size, like the formula with erff, and an element by 7e-8 on average; with five terms it was 9e-8 and 5e-7.
template <int DT>
__device__ __forceinline__ float erf_plus_one(float z, float e) {
    float s;
    if constexpr (DT == FC_F32) {
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.26516504f, __builtin_fabsf(z), 1.f));
        s = __builtin_fmaf(0.061701227f, t, -0.288098425f);
        s = __builtin_fmaf(s, t, 0.433942884f);
        s = __builtin_fmaf(s, t, -0.231134474f);
        s = __builtin_fmaf(s, t, 0.274885684f);
        s = __builtin_fmaf(s, t, 0.121020563f);
        s = __builtin_fmaf(s, t, 0.205435321f);
        s = __builtin_fmaf(s, t, 0.210632786f);
        s = __builtin_fmaf(s, t, 0.21161446f);
        s *= t * e;
        return z < 0.f ? s : 2.f - s;
    } else {
        const float x = z * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, __builtin_fabsf(x), 1.f));
        s = __builtin_fmaf(1.061405429f, t, -1.453152027f);
        s = __builtin_fmaf(s, t, 1.421413741f);
        s = __builtin_fmaf(s, t, -0.284496736f);
        s = __builtin_fmaf(s, t, 0.254829592f);
        s *= t * e;
        return x < 0.f ? s : 2.f - s;
    }
}

template <int DT, int ACT>
__device__ __forceinline__ float activation(float z) {
    if (ACT == FC_ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays
    if (ACT == FC_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
    if (ACT == FC_ACT_GELU) return 0.5f * z * erf_plus_one<DT>(z, __expf(-0.5f * z * z));
    return z;
}

template <int DT, int ACT>
__device__ __forceinline__ float activation_slope(float z) {
    if (ACT == FC_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == FC_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    if (ACT == FC_ACT_GELU) {
        const float e = __expf(-0.5f * z * z);
        return __builtin_fmaf(0.5f, erf_plus_one<DT>(z, e), z * 0.39894228040143268f * e);
    }
    return 1.f;
}

template <bool PAST_CACHE, class V>
__device__ __forceinline__ void store(void *dst, const V &x) {
    if constexpr (PAST_CACHE && sizeof(V) == 16) {
        typedef uint32_t words __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(__builtin_bit_cast(words, x), (words *)dst);
    } else {
        *(V *)dst = x;
    }
}

// What a workgroup works on: a chunk of pixels of one image, a span of its channels.
struct norm_place {
    int chunk, span;
    long n, p0, p1;
    __device__ __forceinline__ norm_place(const norm_params &p, unsigned block) {
        chunk = block % p.chunks;
        const unsigned r = block / p.chunks;
        span = r % p.spans;
        n = r / p.spans;
        p0 = chunk * p.chunk;
        p1 = p0 + p.chunk < p.P ? p0 + p.chunk : p.P;
    }
};

// Threads over a span: `cols` accesses side by side, `rows` pixels at once.
struct norm_threads {
    int cols, rows, tx, ty;
    __device__ __forceinline__ norm_threads(int accesses, int threads = kThreads) {
        cols = accesses < threads ? accesses : threads;
        rows = threads / cols;
        ty = threadIdx.x / cols;
        tx = threadIdx.x - ty * cols;
    }
};

// Sums over a workgroup by butterflies: where the accesses of a span are a power of two of threads side by side, and a group is a power of
// two of accesses or an access holds a power of two of groups, the lanes of a wavefront that belong together differ in bits of their
// number.  `group`: the bits that may differ among the columns of one group (0: sums of each channel).
// Leaves in LDS [units][span] what each wavefront (each part of a wavefront's row) has; returns the number of units.
struct norm_butterfly {
    int cols, group;         // accesses of a span; of a group, 0 if a group is less than an access
    bool fits;
    __device__ __forceinline__ norm_butterfly(const norm_params &p, int vec, int threads) {
        cols = p.span / vec;
        group = p.Cg / vec;
        const int within = p.Cg < vec ? p.Cg : vec;
        fits = cols <= threads && (cols & (cols - 1)) == 0 && (within & (within - 1)) == 0 && (group & (group - 1)) == 0 &&
               p.Cg % within == 0 && (group == 0 || p.Cg == group * vec) && group <= 64;
    }
};

// Sums of `value` over the lanes of each column, by channel.
template <int VEC>
__device__ __forceinline__ void sum_lanes(float (&value)[VEC], int cols) {
#pragma unroll
    for (int m = 32; m; m >>= 1) {
        if (m < cols) break;
#pragma unroll
        for (int v = 0; v < VEC; v++) value[v] += __shfl_xor(value[v], m);
    }
}

// Sums of `value` over a workgroup and each group of the span; every thread gets those of its channels' groups.
template <int VEC, int THREADS>
__device__ __forceinline__ void sum_groups_fast(const norm_params &p, const norm_butterfly &f, const norm_threads &th, float (&value)[VEC], float *lds) {
    // the channels of an access that share a group
#pragma unroll
    for (int m = 1; m < VEC; m <<= 1) {
        if (m >= p.Cg) break;
        float other[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) other[v] = value[v ^ m];
#pragma unroll
        for (int v = 0; v < VEC; v++) value[v] += other[v];
    }
    const int unit = f.cols <= 64 ? threadIdx.x >> 6 : th.ty, units = f.cols <= 64 ? THREADS / 64 : th.rows;
    const int groups = p.span / p.Cg, first = th.tx * VEC / p.Cg;
    if (f.group) {      // one group an access
        float s = value[0];
#pragma unroll
        for (int m = 32; m; m >>= 1)
            if (m >= f.cols || m < f.group) s += __shfl_xor(s, m);
        __syncthreads();      // what was in lds is read
        if (((int)threadIdx.x & 63) < f.cols && (th.tx & (f.group - 1)) == 0) lds[unit * groups + first] = s;
        __syncthreads();
        s = 0.f;
        for (int u = 0; u < units; u++) s += lds[u * groups + first];
#pragma unroll
        for (int v = 0; v < VEC; v++) value[v] = s;
    } else {
        // one value a group of the access: 8 images of 56x56 with 128 channels in 32 groups, bf16: 18.9 -> 13.0 us
        auto join = [&](auto channels) __attribute__((always_inline)) {
            constexpr int STEP = decltype(channels)::value;
#pragma unroll
            for (int m = 32; m; m >>= 1) {
                if (m < f.cols) break;
#pragma unroll
                for (int v = 0; v < VEC; v += STEP) value[v] += __shfl_xor(value[v], m);
            }
            __syncthreads();
            if (((int)threadIdx.x & 63) < f.cols) {
#pragma unroll
                for (int v = 0; v < VEC; v += STEP) lds[(unit * f.cols + th.tx) * VEC + v] = value[v];
            }
            __syncthreads();
#pragma unroll
            for (int v = 0; v < VEC; v++) value[v] = 0.f;
            for (int u = 0; u < units; u++) {
#pragma unroll
                for (int v = 0; v < VEC; v += STEP) value[v] += lds[(u * f.cols + th.tx) * VEC + v];
            }
#pragma unroll
            for (int v = 0; v < VEC; v++) value[v] = value[v / STEP * STEP];
        };
        if (p.Cg == 1) join(std::integral_constant<int, 1>());
        else if (VEC > 2 && p.Cg == 2) join(std::integral_constant<int, (VEC > 2 ? 2 : 1)>());
        else join(std::integral_constant<int, (VEC > 1 ? VEC / 2 : 1)>());
    }
}

// Statistics of each group over a chunk.
template <int DT, int VEC>
__global__ __launch_bounds__(kThreads) void fc_group_norm_stats_kernel(const norm_params p) {
    extern __shared__ float2 entry[];      // (mean, M2) [rows][span]
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    constexpr int U = 8;                   // pixels a batch
    const norm_place at(p, blockIdx.x);
    const norm_threads th(p.span / VEC);
    const norm_butterfly fast(p, VEC, kThreads);
    const int c0 = at.span * p.span;
    const int width = (p.C - c0 < p.span ? p.C - c0 : p.span);
    if (th.ty < th.rows) {
        for (int col = th.tx; col < width / VEC; col += th.cols) {
            const E *src = (const E *)p.x + at.n * p.x_image + c0 + col * VEC;
            float mean[VEC], m2[VEC];
#pragma unroll
            for (int v = 0; v < VEC; v++) mean[v] = m2[v] = 0.f;
            float count = 0.f;
            long q = at.p0 + th.ty;
            const long whole = at.p1 - (long)(U - 1) * th.rows;
            for (; q < whole; q += (long)U * th.rows) {
                V in[U];
#pragma unroll
                for (int u = 0; u < U; u++) in[u] = *(const V *)(src + (q + (long)u * th.rows) * p.x_pixel);
                const float joined = count + U, wb = U / joined, wm = count * wb;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    float s = 0.f, sq = 0.f;
#pragma unroll
                    for (int u = 0; u < U; u++) s += in[u].get(v);
                    s *= 1.f / U;
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const float d = in[u].get(v) - s;
                        sq = __builtin_fmaf(d, d, sq);
                    }
                    const float d = s - mean[v];
                    mean[v] = __builtin_fmaf(d, wb, mean[v]);
                    m2[v] += __builtin_fmaf(d * d, wm, sq);
                }
                count = joined;
            }
            for (; q < at.p1; q += th.rows) {      // what is left, a pixel at a time
                const V in = *(const V *)(src + q * p.x_pixel);
                const float joined = count + 1.f, wb = 1.f / joined, wm = count * wb;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const float d = in.get(v) - mean[v];
                    mean[v] = __builtin_fmaf(d, wb, mean[v]);
                    m2[v] = __builtin_fmaf(d * d, wm, m2[v]);
                }
                count = joined;
            }
            if (fast.fits && width == p.span) {
                const float all = (float)(at.p1 - at.p0) * p.Cg;
                float joined[VEC];
#pragma unroll
                for (int v = 0; v < VEC; v++) joined[v] = count * mean[v];
                sum_groups_fast<VEC, kThreads>(p, fast, th, joined, (float *)entry);
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    joined[v] /= all;
                    const float d = mean[v] - joined[v];
                    mean[v] = joined[v];
                    m2[v] = __builtin_fmaf(count * d, d, m2[v]);
                }
                sum_groups_fast<VEC, kThreads>(p, fast, th, m2, (float *)entry);
                if (th.ty == 0) {
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        const int c = c0 + col * VEC + v;
                        if (c % p.Cg == 0) p.part[(at.n * p.G + c / p.Cg) * p.chunks + at.chunk] = make_float2(mean[v], m2[v]);
                    }
                }
                return;
            }
#pragma unroll
            for (int v = 0; v < VEC; v++) entry[th.ty * p.span + col * VEC + v] = make_float2(mean[v], m2[v]);
        }
    }
    __syncthreads();
    // a wavefront joins the entries of a group: count by count, the means first
    const int lane = threadIdx.x & 63, groups = width / p.Cg, np = (int)(at.p1 - at.p0);
    const float total = (float)np * p.Cg;
    for (int g = threadIdx.x >> 6; g < groups; g += kThreads / 64) {
        float s = 0.f;
        for (int i = lane; i < p.Cg * th.rows; i += 64) {
            const int ty = i / p.Cg, c = i - ty * p.Cg;
            const float cnt = ty < np ? (float)((np - ty + th.rows - 1) / th.rows) : 0.f;
            s += cnt > 0.f ? cnt * entry[ty * p.span + g * p.Cg + c].x : 0.f;
        }
        const float mean = fc_wave_sum(s) / total;
        float m2 = 0.f;
        for (int i = lane; i < p.Cg * th.rows; i += 64) {
            const int ty = i / p.Cg, c = i - ty * p.Cg;
            const float cnt = ty < np ? (float)((np - ty + th.rows - 1) / th.rows) : 0.f;
            if (cnt > 0.f) {
                const float2 e = entry[ty * p.span + g * p.Cg + c];
                m2 += e.y + cnt * (e.x - mean) * (e.x - mean);
            }
        }
        m2 = fc_wave_sum(m2);
        if (lane == 0) p.part[(at.n * p.G + c0 / p.Cg + g) * p.chunks + at.chunk] = make_float2(mean, m2);
    }
}

// Joins the chunks of each group and writes y.
// PAST_CACHE: the result is stored past the caches, which then keep x for this second reading.
template <int DT, int VEC, int ACT, bool PAST_CACHE>
__global__ __launch_bounds__(kThreads) void fc_group_norm_apply_kernel(const norm_params p) {
    extern __shared__ float2 stat[];      // (mean, rstd) of the span's groups
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    constexpr int U = 4;
    const norm_place at(p, blockIdx.x);
    const norm_threads th(p.span / VEC);
    const int c0 = at.span * p.span;
    const int width = (p.C - c0 < p.span ? p.C - c0 : p.span);
    const int groups = width / p.Cg;
    // eight lanes a group where there are many, a wavefront each where there are few
    const int lanes = groups > 4 ? 8 : 64, lane = threadIdx.x & (lanes - 1);
    for (int g = threadIdx.x / lanes; g < groups; g += kThreads / lanes) {
        const long group = at.n * p.G + c0 / p.Cg + g;
        const float2 *part = p.part + group * p.chunks;
        float s = 0.f;
        for (int i = lane; i < p.chunks; i += lanes) {
            const long first = i * p.chunk;
            s += (float)(p.P - first < p.chunk ? p.P - first : p.chunk) * part[i].x;
        }
        for (int m = lanes / 2; m; m >>= 1) s += __shfl_xor(s, m);
        const float mean = s / (float)p.P;
        float m2 = 0.f;
        for (int i = lane; i < p.chunks; i += lanes) {
            const long first = i * p.chunk;
            const float d = part[i].x - mean;
            m2 += part[i].y + (float)(p.P - first < p.chunk ? p.P - first : p.chunk) * p.Cg * d * d;
        }
        for (int m = lanes / 2; m; m >>= 1) m2 += __shfl_xor(m2, m);
        const float rstd = 1.f / sqrtf(m2 / ((float)p.P * p.Cg) + p.eps);
        if (lane == 0) {
            stat[g] = make_float2(mean, rstd);
            if (at.chunk == 0 && p.mean) {
                p.mean[group] = mean;
                p.rstd[group] = rstd;
            }
        }
    }
    __syncthreads();
    if (th.ty >= th.rows) return;
    for (int col = th.tx; col < width / VEC; col += th.cols) {
        float mean[VEC], scale[VEC], shift[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const int c = col * VEC + v;
            const float2 st = stat[c / p.Cg];
            mean[v] = st.x;
            scale[v] = st.y * (p.gamma ? p.gamma[c0 + c] : 1.f);
            shift[v] = p.beta ? p.beta[c0 + c] : 0.f;
        }
        const E *src = (const E *)p.x + at.n * p.x_image + c0 + col * VEC;
        E *dst = (E *)p.y + at.n * p.y_image + c0 + col * VEC;
        for (long q = at.p0 + th.ty; q < at.p1; q += (long)U * th.rows) {
            V in[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long r = q + (long)u * th.rows;
                if (r < at.p1) in[u] = *(const V *)(src + r * p.x_pixel);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long r = q + (long)u * th.rows;
                if (r >= at.p1) break;
#pragma unroll
                for (int v = 0; v < VEC; v++) in[u].set(v, activation<DT, ACT>((in[u].get(v) - mean[v]) * scale[v] + shift[v]));
                store<PAST_CACHE>(dst + r * p.y_pixel, in[u]);
            }
        }
    }
}

// What both launches of the backward pass keep of a column.
template <int VEC>
struct norm_column {
    float mean[VEC], rstd[VEC], gamma[VEC], beta[VEC];
    __device__ __forceinline__ norm_column(const norm_params &p, long n, int c0) {
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const int c = c0 + v;
            const long group = n * p.G + c / p.Cg;
            mean[v] = p.mean[group];
            rstd[v] = p.rstd[group];
            gamma[v] = p.gamma ? p.gamma[c] : 1.f;
            beta[v] = p.beta ? p.beta[c] : 0.f;
        }
    }
};

// Sums of dz and dz xhat of each channel over a chunk, and of both times gamma of each group.
template <int DT, int VEC, int ACT>
__global__ __launch_bounds__(kThreads) void fc_group_norm_sums_kernel(const norm_params p) {
    extern __shared__ float2 entry[];      // (sum dz, sum dz xhat) [rows][span]
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    constexpr int U = 4;
    const norm_place at(p, blockIdx.x);
    const norm_threads th(p.span / VEC);
    const int c0 = at.span * p.span;
    const int width = (p.C - c0 < p.span ? p.C - c0 : p.span);
    if (th.ty < th.rows) {
        for (int col = th.tx; col < width / VEC; col += th.cols) {
            const norm_column<VEC> k(p, at.n, c0 + col * VEC);
            const E *x = (const E *)p.x + at.n * p.x_image + c0 + col * VEC;
            const E *dy = (const E *)p.dy + at.n * p.y_image + c0 + col * VEC;
            float a[VEC], b[VEC];
#pragma unroll
            for (int v = 0; v < VEC; v++) a[v] = b[v] = 0.f;
            for (long q = at.p0 + th.ty; q < at.p1; q += (long)U * th.rows) {
                V xs[U], ds[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const long r = q + (long)u * th.rows;
                    if (r < at.p1) {
                        xs[u] = *(const V *)(x + r * p.x_pixel);
                        ds[u] = *(const V *)(dy + r * p.y_pixel);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (q + (long)u * th.rows >= at.p1) break;
#pragma unroll
                    for (int v = 0; v < VEC; v++) {
                        const float xhat = (xs[u].get(v) - k.mean[v]) * k.rstd[v];
                        const float dz = ds[u].get(v) * activation_slope<DT, ACT>(xhat * k.gamma[v] + k.beta[v]);
                        a[v] += dz;
                        b[v] += dz * xhat;
                    }
                }
            }
#pragma unroll
            for (int v = 0; v < VEC; v++) entry[th.ty * p.span + col * VEC + v] = make_float2(a[v], b[v]);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += kThreads) {
        float2 s = entry[c];
        for (int ty = 1; ty < th.rows; ty++) {
            s.x += entry[ty * p.span + c].x;
            s.y += entry[ty * p.span + c].y;
        }
        p.channel_part[(at.n * p.chunks + at.chunk) * p.C + c0 + c] = s;
        entry[c] = s;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63;
    for (int g = threadIdx.x >> 6; g < width / p.Cg; g += kThreads / 64) {
        float s1 = 0.f, s2 = 0.f;
        for (int i = lane; i < p.Cg; i += 64) {
            const float2 e = entry[g * p.Cg + i];
            const float gamma = p.gamma ? p.gamma[c0 + g * p.Cg + i] : 1.f;
            s1 += gamma * e.x;
            s2 += gamma * e.y;
        }
        s1 = fc_wave_sum(s1);
        s2 = fc_wave_sum(s2);
        if (lane == 0) p.part[(at.n * p.G + c0 / p.Cg + g) * p.chunks + at.chunk] = make_float2(s1, s2);
    }
}

// dgamma and dbeta of 8 channels: 32 threads each over the images' chunks, in a fixed order, eight loads at a time.
__device__ __forceinline__ void reduce_channels(const norm_params &p, unsigned block, float2 *sums) {
    const int lc = threadIdx.x & 7, row = threadIdx.x >> 3, c = block * 8 + lc;
    float2 s = make_float2(0.f, 0.f);
    if (c < p.C) {
        const long rows = (long)p.N * p.chunks;
        long r = row;
        for (; r + 7 * 32 < rows; r += 8 * 32) {
            float2 e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = p.channel_part[(r + 32 * i) * p.C + c];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                s.x += e[i].x;
                s.y += e[i].y;
            }
        }
        for (; r < rows; r += 32) {
            const float2 e = p.channel_part[r * p.C + c];
            s.x += e.x;
            s.y += e.y;
        }
    }
    sums[row * 8 + lc] = s;
    __syncthreads();
    if (row == 0 && c < p.C) {
        for (int r = 1; r < 32; r++) {
            s.x += sums[r * 8 + lc].x;
            s.y += sums[r * 8 + lc].y;
        }
        if (p.dbeta) p.dbeta[c] = s.x;
        if (p.dgamma) p.dgamma[c] = s.y;
    }
}

__global__ __launch_bounds__(kThreads) void fc_group_norm_channels_kernel(const norm_params p) {
    __shared__ float2 sums[kThreads];
    reduce_channels(p, blockIdx.x, sums);
}

// dx; the first workgroups add up dgamma and dbeta meanwhile.
template <int DT, int VEC, int ACT, bool PAST_CACHE>
__global__ __launch_bounds__(kThreads) void fc_group_norm_gradient_kernel(const norm_params p) {
    extern __shared__ float2 stat[];      // (s1, s2) of the span's groups over their values, or the sums of channels
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    constexpr int U = 4;
    if ((int)blockIdx.x < p.reduce_blocks) {
        reduce_channels(p, blockIdx.x, stat);
        return;
    }
    const norm_place at(p, blockIdx.x - p.reduce_blocks);
    const norm_threads th(p.span / VEC);
    const int c0 = at.span * p.span;
    const int width = (p.C - c0 < p.span ? p.C - c0 : p.span);
    const int groups = width / p.Cg, lanes = groups > 4 ? 8 : 64, lane = threadIdx.x & (lanes - 1);
    for (int g = threadIdx.x / lanes; g < groups; g += kThreads / lanes) {
        const float2 *part = p.part + (at.n * p.G + c0 / p.Cg + g) * p.chunks;
        float s1 = 0.f, s2 = 0.f;
        for (int i = lane; i < p.chunks; i += lanes) {
            s1 += part[i].x;
            s2 += part[i].y;
        }
        for (int m = lanes / 2; m; m >>= 1) {
            s1 += __shfl_xor(s1, m);
            s2 += __shfl_xor(s2, m);
        }
        const float inv = 1.f / ((float)p.P * p.Cg);
        if (lane == 0) stat[g] = make_float2(s1 * inv, s2 * inv);
    }
    __syncthreads();
    if (th.ty >= th.rows) return;
    for (int col = th.tx; col < width / VEC; col += th.cols) {
        const norm_column<VEC> k(p, at.n, c0 + col * VEC);
        float2 st[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) st[v] = stat[(col * VEC + v) / p.Cg];
        const E *x = (const E *)p.x + at.n * p.x_image + c0 + col * VEC;
        const E *dy = (const E *)p.dy + at.n * p.y_image + c0 + col * VEC;
        E *dx = (E *)p.y + at.n * p.x_image + c0 + col * VEC;
        for (long q = at.p0 + th.ty; q < at.p1; q += (long)U * th.rows) {
            V xs[U], ds[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long r = q + (long)u * th.rows;
                if (r < at.p1) {
                    xs[u] = *(const V *)(x + r * p.x_pixel);
                    ds[u] = *(const V *)(dy + r * p.y_pixel);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long r = q + (long)u * th.rows;
                if (r >= at.p1) break;
#pragma unroll
                for (int v = 0; v < VEC; v++) {
                    const float xhat = (xs[u].get(v) - k.mean[v]) * k.rstd[v];
                    const float dz = ds[u].get(v) * activation_slope<DT, ACT>(xhat * k.gamma[v] + k.beta[v]);
                    xs[u].set(v, k.rstd[v] * (k.gamma[v] * dz - st[v].x - xhat * st[v].y));
                }
                store<PAST_CACHE>(dx + r * p.x_pixel, xs[u]);
            }
        }
    }
}

// ---- groups that fit a workgroup's registers: x is read once, one launch

// Consecutive spans of an image share cache lines, so they go to one of the eight dies, which take workgroups in turn.
__device__ __forceinline__ unsigned same_die(unsigned block, unsigned blocks) {
    return blocks % 8 ? block : block % 8 * (blocks / 8) + block / 8;
}

// Sums over the pixels of each of a span's channels, from one value a thread and channel of its column.  Leaves in LDS the sums of `parts`
// threads a channel, [parts][span].  Ends with those in LDS for all.
template <int VEC, int THREADS>
__device__ __forceinline__ int sum_pixels(const norm_params &p, const norm_threads &th, const float (&value)[VEC], float *entry) {
    constexpr int PITCH = THREADS + 8;      // [VEC][THREADS], eight banks further on for each channel of an access
    __syncthreads();      // what was in entry is read
#pragma unroll
    for (int v = 0; v < VEC; v++) entry[v * PITCH + threadIdx.x] = value[v];
    __syncthreads();
    const int parts = THREADS / p.span < th.rows ? THREADS / p.span : th.rows;
    const int part = (int)threadIdx.x / p.span, c = (int)threadIdx.x - part * p.span;
    float s = 0.f;
    if (part < parts)
        for (int ty = part; ty < th.rows; ty += parts) s += entry[c % VEC * PITCH + ty * th.cols + c / VEC];
    __syncthreads();
    if (part < parts) entry[threadIdx.x] = s;
    __syncthreads();
    return parts;
}

// Sums over the workgroup and each group of the span; every thread with pixels gets those of its channels' groups.
template <int VEC, int THREADS>
__device__ __forceinline__ void sum_groups(const norm_params &p, const norm_butterfly &fast, const norm_threads &th, float (&value)[VEC], float *entry) {
    if (fast.fits) {
        sum_groups_fast<VEC, THREADS>(p, fast, th, value, entry);
        return;
    }
    const int parts = sum_pixels<VEC, THREADS>(p, th, value, entry);
    float *const stat = entry + VEC * (THREADS + 8);
    const int lane = threadIdx.x & 63;
    for (int g = threadIdx.x >> 6; g < p.span / p.Cg; g += THREADS / 64) {
        float s = 0.f;
        if (parts >= p.Cg) {
            for (int part = lane; part < parts; part += 64)
                for (int i = 0; i < p.Cg; i++) s += entry[part * p.span + g * p.Cg + i];
        } else {
            for (int part = 0; part < parts; part++)
                for (int i = lane; i < p.Cg; i += 64) s += entry[part * p.span + g * p.Cg + i];
        }
        s = fc_wave_sum(s);
        if (lane == 0) stat[g] = s;
    }
    __syncthreads();
    if (th.ty < th.rows) {
#pragma unroll
        for (int v = 0; v < VEC; v++) value[v] = stat[(th.tx * VEC + v) / p.Cg];
    }
}

// Sums over the workgroup of each channel, left in channel[].x or .y by the first threads.
template <int VEC, int THREADS>
__device__ __forceinline__ void sum_channels(const norm_params &p, const norm_butterfly &fast, const norm_threads &th, float (&value)[VEC], float *entry,
                                             float *channel) {
    int parts;
    if (fast.fits) {
        sum_lanes<VEC>(value, fast.cols);
        const int unit = fast.cols <= 64 ? threadIdx.x >> 6 : th.ty;
        parts = fast.cols <= 64 ? THREADS / 64 : th.rows;
        __syncthreads();
        if (((int)threadIdx.x & 63) < fast.cols) {
#pragma unroll
            for (int v = 0; v < VEC; v++) entry[unit * p.span + th.tx * VEC + v] = value[v];
        }
        __syncthreads();
    } else {
        parts = sum_pixels<VEC, THREADS>(p, th, value, entry);
    }
    if ((int)threadIdx.x < p.span) {
        float s = 0.f;
        for (int i = 0; i < parts; i++) s += entry[i * p.span + threadIdx.x];
        channel[2 * threadIdx.x] = s;
    }
}

// Values of 16 bits stay packed between two passes over them: the compiler would keep the unpacked ones, twice the registers (16 accesses
// forward and 8 backward spilled 112 and 67; 32 images of 56x56x256 in bf16: forward 62 -> 36 us, backward alone 124 -> 74; backward with GELU 16 to 20 still spill).
template <class V, int R>
__device__ __forceinline__ void keep_packed(V (&x)[R]) {
    typedef unsigned __attribute__((ext_vector_type(4))) words;
    if constexpr (sizeof(x[0].v[0]) == 2) {
#pragma unroll
        for (int k = 0; k < R; k++) {
            words w = __builtin_bit_cast(words, x[k]);
            asm("" : "+v"(w));
            x[k] = __builtin_bit_cast(V, w);
        }
    }
}

// R pixels of its column a thread.
template <int DT, int VEC, int ACT, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void fc_group_norm_resident_kernel(const norm_params p) {
    extern __shared__ float resident_sums[];      // [VEC][THREADS], then the groups' sums
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    const unsigned block = same_die(blockIdx.x, gridDim.x);
    const long n = block / p.spans;
    const int c0 = (int)(block - n * p.spans) * p.span;
    const norm_threads th(p.span / VEC, THREADS);
    const E *src = (const E *)p.x + n * p.x_image + c0 + th.tx * VEC;
    const int P = th.ty < th.rows ? (int)p.P : 0;      // threads past the last row have no pixels
    V in[R];
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int q = th.ty + k * th.rows;
        if (q < P) in[k] = *(const V *)(src + q * p.x_pixel);
    }
    float sum[VEC], mean[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        sum[v] = 0.f;
#pragma unroll
        for (int k = 0; k < R; k++) sum[v] += th.ty + k * th.rows < P ? in[k].get(v) : 0.f;
    }
    const float values = (float)p.P * p.Cg;
    const norm_butterfly fast(p, VEC, THREADS);
    if (R > 4) keep_packed(in);      // four fit unpacked: 8 images of 35x35x192 in half 15.9 us, 17.7 packed
    sum_groups<VEC, THREADS>(p, fast, th, sum, resident_sums);
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        mean[v] = sum[v] / values;
        sum[v] = 0.f;
#pragma unroll
        for (int k = 0; k < R; k++) {
            const float d = th.ty + k * th.rows < P ? in[k].get(v) - mean[v] : 0.f;
            sum[v] = __builtin_fmaf(d, d, sum[v]);
        }
    }
    if (R > 4) keep_packed(in);
    sum_groups<VEC, THREADS>(p, fast, th, sum, resident_sums);
    if (th.ty >= th.rows) return;
    float scale[VEC], shift[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        const int c = c0 + th.tx * VEC + v;
        const float rstd = 1.f / sqrtf(sum[v] / values + p.eps);
        scale[v] = rstd * (p.gamma ? p.gamma[c] : 1.f);
        shift[v] = p.beta ? p.beta[c] : 0.f;
        if (p.mean && th.ty == 0 && c % p.Cg == 0) {
            p.mean[n * p.G + c / p.Cg] = mean[v];
            p.rstd[n * p.G + c / p.Cg] = rstd;
        }
    }
    E *dst = (E *)p.y + n * p.y_image + c0 + th.tx * VEC;
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int q = th.ty + k * th.rows;
        if (q >= P) break;
#pragma unroll
        for (int v = 0; v < VEC; v++) in[k].set(v, activation<DT, ACT>((in[k].get(v) - mean[v]) * scale[v] + shift[v]));
        *(V *)(dst + q * p.y_pixel) = in[k];
    }
}

template <int DT, int VEC, int ACT, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void fc_group_norm_resident_gradient_kernel(const norm_params p) {
    extern __shared__ float resident_sums[];      // [VEC][THREADS], then dbeta and dgamma of the span's channels, then s1 and s2 of its groups
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    const unsigned block = same_die(blockIdx.x, gridDim.x);
    const long n = block / p.spans;
    const int c0 = (int)(block - n * p.spans) * p.span;
    const norm_threads th(p.span / VEC, THREADS);
    float2 *const channel = (float2 *)(resident_sums + VEC * (THREADS + 8)), *const stat = channel + p.span;
    const E *x = (const E *)p.x + n * p.x_image + c0 + th.tx * VEC;
    const E *dy = (const E *)p.dy + n * p.y_image + c0 + th.tx * VEC;
    const int P = th.ty < th.rows ? (int)p.P : 0;
    V xs[R], ds[R];
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int q = th.ty + k * th.rows;
        if (q < P) {
            xs[k] = *(const V *)(x + q * p.x_pixel);
            ds[k] = *(const V *)(dy + q * p.y_pixel);
        }
    }
    const norm_column<VEC> c(p, n, c0 + th.tx * VEC);
    float a[VEC], b[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) a[v] = b[v] = 0.f;
#pragma unroll
    for (int k = 0; k < R; k++) {
        if (th.ty + k * th.rows >= P) break;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const float xhat = (xs[k].get(v) - c.mean[v]) * c.rstd[v];
            const float dz = ds[k].get(v) * activation_slope<DT, ACT>(xhat * c.gamma[v] + c.beta[v]);
            if (DT == FC_F32) ds[k].set(v, dz);
            a[v] += dz;
            b[v] = __builtin_fmaf(dz, xhat, b[v]);
        }
    }
    const norm_butterfly fast(p, VEC, THREADS);
    keep_packed(xs);
    keep_packed(ds);
    sum_channels<VEC, THREADS>(p, fast, th, a, resident_sums, &channel->x);
    sum_channels<VEC, THREADS>(p, fast, th, b, resident_sums, &channel->y);
    if (p.channel_part && (int)threadIdx.x < p.span) p.channel_part[n * p.C + c0 + threadIdx.x] = channel[threadIdx.x];
    __syncthreads();
    const int lane = threadIdx.x & 63;
    for (int g = threadIdx.x >> 6; g < p.span / p.Cg; g += THREADS / 64) {
        float s1 = 0.f, s2 = 0.f;
        for (int i = lane; i < p.Cg; i += 64) {
            const float2 e = channel[g * p.Cg + i];
            const float gamma = p.gamma ? p.gamma[c0 + g * p.Cg + i] : 1.f;
            s1 += gamma * e.x;
            s2 += gamma * e.y;
        }
        const float inv = 1.f / ((float)p.P * p.Cg);
        s1 = fc_wave_sum(s1) * inv;
        s2 = fc_wave_sum(s2) * inv;
        if (lane == 0) stat[g] = make_float2(s1, s2);
    }
    __syncthreads();
    if (th.ty >= th.rows) return;
    float2 st[VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) st[v] = stat[(th.tx * VEC + v) / p.Cg];
    E *dx = (E *)p.y + n * p.x_image + c0 + th.tx * VEC;
#pragma unroll
    for (int k = 0; k < R; k++) {
        const int q = th.ty + k * th.rows;
        if (q >= P) break;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const float xhat = (xs[k].get(v) - c.mean[v]) * c.rstd[v];
            const float dz = DT == FC_F32 ? ds[k].get(v) : ds[k].get(v) * activation_slope<DT, ACT>(xhat * c.gamma[v] + c.beta[v]);
            xs[k].set(v, c.rstd[v] * (c.gamma[v] * dz - st[v].x - xhat * st[v].y));
        }
        *(V *)(dx + q * p.x_pixel) = xs[k];
    }
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

long gcd(long a, long b) { return b ? gcd(b, a % b) : a; }

bool shape_ok(const fc_group_norm_shape *s) {
    if (!s || s->N < 1 || s->P < 1 || s->C < 1 || s->G < 1 || s->C % s->G || !fc_dtype_ok(s->dtype)) return false;
    if (s->act < FC_ACT_NONE || s->act > FC_ACT_GELU || !(s->eps >= 0.f)) return false;
    return s->x_image >= 0 && s->x_pixel >= 0 && s->y_image >= 0 && s->y_pixel >= 0;
}

bool same(const fc_group_norm_plan &a, const fc_group_norm_plan &b) {
    const fc_group_norm_shape &s = a.shape, &t = b.shape;
    return s.N == t.N && s.P == t.P && s.C == t.C && s.G == t.G && s.dtype == t.dtype && s.act == t.act && s.eps == t.eps &&
           s.x_image == t.x_image && s.x_pixel == t.x_pixel && s.y_image == t.y_image && s.y_pixel == t.y_pixel && a.span == b.span &&
           a.chunks == b.chunks && a.resident == b.resident && a.resident_backward == b.resident_backward &&
           a.ws_bytes == b.ws_bytes && a.ws_backward_bytes == b.ws_backward_bytes;
}

// The widest access of a plan whose tensors begin at `addr`: a column lies within a span.
int width_of(const fc_group_norm_shape &s, int span, uint64_t addr) {
    return fc_widest(s.dtype, (uint64_t)(s.C | span | s.x_image | s.x_pixel | s.y_image | s.y_pixel), addr);
}

template <int ACT, class F>
bool with_width(int dtype, int vec, F f) {
    if (dtype == FC_F32) {
        if (vec == 4) return f.template run<FC_F32, 4, ACT>();
        if (vec == 2) return f.template run<FC_F32, 2, ACT>();
        return f.template run<FC_F32, 1, ACT>();
    }
    if (dtype == FC_BF16) {
        if (vec == 8) return f.template run<FC_BF16, 8, ACT>();
        if (vec == 4) return f.template run<FC_BF16, 4, ACT>();
        if (vec == 2) return f.template run<FC_BF16, 2, ACT>();
        return f.template run<FC_BF16, 1, ACT>();
    }
    if (vec == 8) return f.template run<FC_F16, 8, ACT>();
    if (vec == 4) return f.template run<FC_F16, 4, ACT>();
    if (vec == 2) return f.template run<FC_F16, 2, ACT>();
    return f.template run<FC_F16, 1, ACT>();
}

template <class F>
bool with_kernel(const fc_group_norm_shape &s, int vec, F f) {
    switch (s.act) {
        case FC_ACT_RELU: return with_width<FC_ACT_RELU>(s.dtype, vec, f);
        case FC_ACT_SILU: return with_width<FC_ACT_SILU>(s.dtype, vec, f);
        case FC_ACT_GELU: return with_width<FC_ACT_GELU>(s.dtype, vec, f);
        default: return with_width<FC_ACT_NONE>(s.dtype, vec, f);
    }
}

struct forward_launch {
    hipStream_t stream;
    const norm_params &p;
    unsigned blocks;
    template <int DT, int VEC, int ACT>
    bool run() {
        const int accesses = p.span / VEC, rows = kThreads / (accesses < kThreads ? accesses : kThreads);
        fc_group_norm_stats_kernel<DT, VEC><<<dim3(blocks), dim3(kThreads), (size_t)rows * p.span * sizeof(float2), stream>>>(p);
        constexpr bool whole = VEC * sizeof(typename fc_elem<DT>::type) == 16;
        const auto apply = whole && p.past_cache ? fc_group_norm_apply_kernel<DT, VEC, ACT, whole> : fc_group_norm_apply_kernel<DT, VEC, ACT, false>;
        apply<<<dim3(blocks), dim3(kThreads), (size_t)(p.span / p.Cg) * sizeof(float2), stream>>>(p);
        return true;
    }
};

// Pixels a thread, of 256 threads or of 1024, that a resident kernel of accesses of VEC elements needs; 0 if no kernel has as many.
int resident_pixels(long P, int span, int vec, int threads, int most) {
    const int cols = span / vec;
    if (cols > threads / 2 || span > threads) return 0;
    const long need = (P + threads / cols - 1) / (threads / cols);
    int r = 1;
    while (r < need && r < most) r *= 2;
    return need <= r ? r : 0;
}

// 16 accesses of 16 bytes in registers forward, 8 each of x and dy backward.  Resident against not, 32 images of 56x56x256: forward in bf16 36 and 40 us, in
// fp32 56 and 67; 1 of 14x14x512 in bf16 forward 6.4 and 12.8, backward 9.4 and 20.4; 128 of 28x28x512 in fp32 backward 171 and 205.
constexpr int kResident = 16, kResidentBackward = 8;
// With fewer, a wider workgroup leaves compute units idle: 1 image of 14x14x512 in bf16 6.5 us in 32 workgroups and 9.1 in 16, 8 of 35x35x192 in half
// 13.9 and 17.4 in 32.
constexpr long kResidentWorkgroups = 256;

// Less than 64 bytes of a pixel (half a cache line) are read well by few workgroups with a short wait before their sums.  Forward, resident against
// not, in bf16: 8 images of 8000x256 as 256 workgroups of 16 bytes 32 and 37 us; but 32 of 6272x256 as 512 of 32 bytes 77 and 74, as 1024 of 16
// bytes 112; 4 of 12544x128 as 64 workgroups with 16 accesses a thread 36 and 24.  Backward twice as much would be read again, from the last cache
// if it holds that, best right after a forward pass.  Both passes, resident backward against not, 32 bytes of 3136x256: 32 images in bf16 (51 MB a tensor) 104 and 117,
// 64 in bf16 (103 MB) 205 and 203, 20 in fp32 (64 MB) 121 and 111, 32 in fp32 (103 MB) 153 and 146, 48 in fp32 230 and 229; the backward pass alone 74 and 84,
// 138 and 141, 79 and 72, 101 and 107, 147 and 150.
constexpr long kWhole = 64;
constexpr int kResidentNarrow = 8;
constexpr double kNarrowBackwardBytes = 64e6;

// Channels of a resident workgroup: whole groups and whole accesses of 16 bytes, and with them kWhole bytes of a pixel if they fit; 0 if not even
// those fit, or are read badly.
int resident_span(const fc_group_norm_shape *s, bool backward) {
    const int Cg = s->C / s->G, es = (int)fc_elem_size(s->dtype), vec = 16 / es, most = backward ? kResidentBackward : kResident;
    if (fc_widest(s->dtype, (uint64_t)(s->C | s->x_image | s->x_pixel | s->y_image | s->y_pixel), 0) != vec) return 0;
    const long step = Cg / gcd(Cg, vec) * vec;
    if (step > 256) return 0;
    int found = 0;
    for (long span = step; span <= s->C && span <= 256; span *= 2) {
        if (s->C % span || !resident_pixels(s->P, (int)span, vec, 1024, most)) break;
        if (found && (long)s->N * (s->C / span) < kResidentWorkgroups) break;
        found = (int)span;
        if (span * es >= kWhole) break;
    }
    if (!found) return 0;
    const long blocks = (long)s->N * (s->C / found);
    if (found * es < kWhole) {
        if (backward && (double)s->N * s->P * s->C * es > kNarrowBackwardBytes) return 0;
        if (!backward && (blocks > kResidentWorkgroups || !resident_pixels(s->P, found, vec, 1024, kResidentNarrow))) return 0;
    }
    return blocks * 1024 < kMostThreads ? found : 0;
}

template <int DT, int VEC, int ACT, bool BACKWARD, int THREADS>
void launch_resident(hipStream_t stream, const norm_params &p, int r) {
    const size_t lds = VEC * (THREADS + 8) * sizeof(float) + (size_t)p.span * 2 * sizeof(float2);
    const dim3 grid((unsigned)((long)p.N * p.spans)), threads(THREADS);
    auto launch = [&](auto pixels) {
        if constexpr (BACKWARD) fc_group_norm_resident_gradient_kernel<DT, VEC, ACT, THREADS, decltype(pixels)::value><<<grid, threads, lds, stream>>>(p);
        else fc_group_norm_resident_kernel<DT, VEC, ACT, THREADS, decltype(pixels)::value><<<grid, threads, lds, stream>>>(p);
    };
    if (r == 1) launch(std::integral_constant<int, 1>());
    else if (r == 2) launch(std::integral_constant<int, 2>());
    else if constexpr (THREADS > kThreads) {
        if (r == 4) launch(std::integral_constant<int, 4>());
        else if (r == 8) launch(std::integral_constant<int, 8>());
        else if constexpr (!BACKWARD) launch(std::integral_constant<int, 16>());
    }
}

template <bool BACKWARD>
struct resident_launch {
    hipStream_t stream;
    const norm_params &p;
    template <int DT, int VEC, int ACT>
    bool run() {
        constexpr bool whole = VEC * sizeof(typename fc_elem<DT>::type) == 16;      // the plans' widest access
        if constexpr (whole) {
            const int most = BACKWARD ? kResidentBackward : kResident, few = resident_pixels(p.P, p.span, VEC, kThreads, 2);
            if (few) launch_resident<DT, VEC, ACT, BACKWARD, kThreads>(stream, p, few);
            else launch_resident<DT, VEC, ACT, BACKWARD, 1024>(stream, p, resident_pixels(p.P, p.span, VEC, 1024, most));
        }
        return whole;
    }
};

struct backward_launch {
    hipStream_t stream;
    const norm_params &p;
    unsigned blocks;
    template <int DT, int VEC, int ACT>
    bool run() {
        const int accesses = p.span / VEC, rows = kThreads / (accesses < kThreads ? accesses : kThreads);
        fc_group_norm_sums_kernel<DT, VEC, ACT><<<dim3(blocks), dim3(kThreads), (size_t)rows * p.span * sizeof(float2), stream>>>(p);
        const size_t groups = (size_t)(p.span / p.Cg), need = groups > 256 ? groups : 256;
        constexpr bool whole = VEC * sizeof(typename fc_elem<DT>::type) == 16;
        const auto gradient = whole && p.past_cache ? fc_group_norm_gradient_kernel<DT, VEC, ACT, whole> : fc_group_norm_gradient_kernel<DT, VEC, ACT, false>;
        gradient<<<dim3(blocks + p.reduce_blocks), dim3(kThreads), need * sizeof(float2), stream>>>(p);
        return true;
    }
};

norm_params params_of(const fc_group_norm_plan *plan) {
    const fc_group_norm_shape &s = plan->shape;
    norm_params p = {};
    p.N = s.N; p.P = s.P; p.C = s.C; p.G = s.G; p.Cg = s.C / s.G; p.eps = s.eps;
    p.span = plan->span;
    p.spans = (s.C + plan->span - 1) / plan->span;
    p.chunks = plan->chunks;
    p.chunk = (s.P + plan->chunks - 1) / plan->chunks;
    // 32 images of 224x224x64 in bf16: 147 -> 117 us.  A result that fits beside its input is left in the caches, for whoever reads it next.
    p.past_cache = (double)s.N * s.P * s.C * fc_elem_size(s.dtype) * 2 > kCacheBytes;
    p.x_image = s.x_image; p.x_pixel = s.x_pixel; p.y_image = s.y_image; p.y_pixel = s.y_pixel;
    return p;
}

}  // namespace

extern "C" int fc_group_norm_make_plan(const fc_group_norm_shape *s, fc_group_norm_plan *plan) {
    if (!plan || !shape_ok(s)) return FC_ERR_INVALID;
    const int Cg = s->C / s->G;
    if (Cg > kMaxGroupChannels || fc_count(s->N, s->P, s->C) < 0 || fc_count(s->N, s->C) >= (1l << 31)) return FC_ERR_UNSUPPORTED;
    *plan = {};
    plan->shape = *s;
    // whole groups and whole accesses, up to 4096 channels: the widest access that leaves such a span
    long step = Cg;
    for (int vec = fc_widest(s->dtype, (uint64_t)(s->C | s->x_image | s->x_pixel | s->y_image | s->y_pixel), 0); vec >= 1; vec >>= 1) {
        step = Cg / gcd(Cg, vec) * vec;
        if (step <= kMaxGroupChannels) break;
    }
    long span = step;
    while (span + step <= kMaxGroupChannels && span < s->C) span += step;
    if (span > s->C) span = s->C;
    plan->span = (int)span;
    const long spans = (s->C + span - 1) / span, pixels = s->P;
    // about four workgroups a compute unit, of 32 KB and more each: 32 images of 56x56x256 in fp32 with a backward pass 145 us with 512 or 1024 of them,
    // 151 with 2048; 4 of 112x112x128 in bf16 with a backward pass 58 in parts of 32 KB, 80 in parts of 16
    long chunks = 1024 / (s->N * spans);
    const long least = 32768 / (span * (long)fc_elem_size(s->dtype)) + 1;
    if (chunks > (pixels + least - 1) / least) chunks = (pixels + least - 1) / least;
    if (chunks < 1) chunks = 1;
    if (chunks > 256) chunks = 256;
    const long chunk = (pixels + chunks - 1) / chunks;
    chunks = (pixels + chunk - 1) / chunk;
    if (chunk >= (1l << 30) || (s->N * spans * chunks + s->C / 8 + 1) * kThreads >= kMostThreads) return FC_ERR_UNSUPPORTED;
    plan->chunks = (int)chunks;
    plan->resident = resident_span(s, false);
    plan->resident_backward = resident_span(s, true);
    plan->ws_bytes = (size_t)s->N * s->G * chunks * sizeof(float2);
    plan->ws_backward_bytes = plan->ws_bytes + (size_t)s->N * chunks * s->C * sizeof(float2);
    return FC_OK;
}

static int check_plan(fc_context *ctx, const fc_group_norm_plan *plan, const char *what) {
    fc_group_norm_plan own;
    if (!plan || fc_group_norm_make_plan(&plan->shape, &own) != FC_OK || !same(*plan, own)) return fail(ctx, FC_ERR_INVALID, what);
    return FC_OK;
}

extern "C" int fc_group_norm(fc_context *ctx, const fc_group_norm_plan *plan, const void *x_dev, const float *gamma_dev,
                             const float *beta_dev, void *y_dev, float *mean_dev, float *rstd_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_group_norm: not a plan of fc_group_norm_make_plan")) return FC_ERR_INVALID;
    if (!x_dev || !y_dev || (!ws_dev && plan->ws_bytes) || !mean_dev != !rstd_dev) return fail(ctx, FC_ERR_INVALID, "fc_group_norm: null pointer");
    const uint64_t addr = (uint64_t)x_dev | (uint64_t)y_dev;
    if ((addr & (fc_elem_size(plan->shape.dtype) - 1)) || ((uint64_t)ws_dev & 7) ||
        (((uint64_t)gamma_dev | (uint64_t)beta_dev | (uint64_t)mean_dev | (uint64_t)rstd_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_group_norm: unaligned pointer");
    const fc_group_norm_shape &s = plan->shape;
    if (!fc_apart({{s.N, s.y_image}, {s.P, s.y_pixel}}, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_group_norm: pixels of y overlap");
    norm_params p = params_of(plan);
    p.x = x_dev; p.y = y_dev; p.gamma = gamma_dev; p.beta = beta_dev; p.mean = mean_dev; p.rstd = rstd_dev;
    p.part = (float2 *)ws_dev;
    if (plan->resident && (addr & 15) == 0) {
        p.span = plan->resident;
        p.spans = p.C / p.span;
        with_kernel(plan->shape, 16 / (int)fc_elem_size(plan->shape.dtype), resident_launch<false>{ctx->stream, p});
        FC_LAUNCH_CHECK(ctx, "fc_group_norm");
        return FC_OK;
    }
    forward_launch f = {ctx->stream, p, (unsigned)((long)p.N * p.spans * p.chunks)};
    with_kernel(plan->shape, width_of(plan->shape, plan->span, addr), f);
    FC_LAUNCH_CHECK(ctx, "fc_group_norm");
    return FC_OK;
}

extern "C" int fc_group_norm_backward(fc_context *ctx, const fc_group_norm_plan *plan, const void *dy_dev, const void *x_dev,
                                      const float *gamma_dev, const float *beta_dev, const float *mean_dev, const float *rstd_dev,
                                      void *dx_dev, float *dgamma_dev, float *dbeta_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_group_norm_backward: not a plan of fc_group_norm_make_plan")) return FC_ERR_INVALID;
    if (!dy_dev || !x_dev || !mean_dev || !rstd_dev || !dx_dev || (!ws_dev && plan->ws_backward_bytes))
        return fail(ctx, FC_ERR_INVALID, "fc_group_norm_backward: null pointer");
    const uint64_t addr = (uint64_t)x_dev | (uint64_t)dy_dev | (uint64_t)dx_dev;
    if ((addr & (fc_elem_size(plan->shape.dtype) - 1)) || ((uint64_t)ws_dev & 7) ||
        (((uint64_t)gamma_dev | (uint64_t)beta_dev | (uint64_t)mean_dev | (uint64_t)rstd_dev | (uint64_t)dgamma_dev | (uint64_t)dbeta_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_group_norm_backward: unaligned pointer");
    const fc_group_norm_shape &s = plan->shape;
    if (!fc_apart({{s.N, s.x_image}, {s.P, s.x_pixel}}, s.C)) return fail(ctx, FC_ERR_INVALID, "fc_group_norm_backward: pixels of dx overlap");
    norm_params p = params_of(plan);
    p.x = x_dev; p.dy = dy_dev; p.y = dx_dev; p.gamma = gamma_dev; p.beta = beta_dev;
    p.mean = const_cast<float *>(mean_dev); p.rstd = const_cast<float *>(rstd_dev);      // only read
    p.part = (float2 *)ws_dev;
    p.channel_part = p.part + (size_t)p.N * p.G * p.chunks;
    p.dgamma = dgamma_dev; p.dbeta = dbeta_dev;
    p.reduce_blocks = dgamma_dev || dbeta_dev ? (p.C + 7) / 8 : 0;
    if (plan->resident_backward && (addr & 15) == 0) {
        p.span = plan->resident_backward;
        p.spans = p.C / p.span;
        p.chunks = 1;      // sums of channels, an image each
        p.channel_part = p.reduce_blocks ? (float2 *)ws_dev : nullptr;
        with_kernel(plan->shape, 16 / (int)fc_elem_size(plan->shape.dtype), resident_launch<true>{ctx->stream, p});
        if (p.reduce_blocks) fc_group_norm_channels_kernel<<<dim3((unsigned)p.reduce_blocks), dim3(kThreads), 0, ctx->stream>>>(p);
        FC_LAUNCH_CHECK(ctx, "fc_group_norm_backward");
        return FC_OK;
    }
    backward_launch f = {ctx->stream, p, (unsigned)((long)p.N * p.spans * p.chunks)};
    with_kernel(plan->shape, width_of(plan->shape, plan->span, addr), f);
    FC_LAUNCH_CHECK(ctx, "fc_group_norm_backward");
    return FC_OK;
}
