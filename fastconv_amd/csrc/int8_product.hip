// Products of 8-bit rows with scales for each row (token) and each column (channel):
//
//   y[m][n] = (sum over k of x[m][k] w[n][k]) * x_scale[m] * w_scale[n] + bias[n]
//
// Sums are 32-bit integers, exact up to 131071 terms whatever their order, so every kernel here gives the same bits.  x and w are rows of k: 16 bytes of a
// row are a lane's operand of v_mfma_i32_16x16x64_i8 and v_mfma_i32_32x32x32_i8 as they lie.  w is the first operand: a lane then holds four
// neighbouring channels of one token.
#include <type_traits>

#include "token_types.h"

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

constexpr int kMostTerms = 131071;      // of 128 * 128 each: 2^31 - 2^14
constexpr int kStage = 128;             // bytes of a row that a tile takes at once: 8 words of 16

__device__ const intx4 kZeroWord = {0, 0, 0, 0};

struct product_params {
    const int8_t *x, *w;
    const float *x_scale, *w_scale, *bias;
    void *y;
    long M;
    int N, K;
    long x_row, w_row, y_row;
    int tiles_m, tiles_n;
    bool wide;               // four neighbouring channels of y lie within one access
};

// 16 bytes of a row from k on, wherever they begin; zeros past its end.
__device__ __forceinline__ intx4 row_word(const int8_t *row, int k, int K) {
    intx4 v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else if (k < K) {
        unsigned u[4] = {0, 0, 0, 0};
        for (int i = 0; i < K - k; i++) u[i >> 2] |= (unsigned)(uint8_t)row[k + i] << (8 * (i & 3));
        v = {(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
    }
    return v;
}

// Four neighbouring channels, from n on, of token m.
template <int DT>
__device__ __forceinline__ void put(const product_params &p, long m, int n, const int (&sum)[4], float xs) {
    typedef typename fc_elem<DT>::type E;
    E *y = (E *)p.y + m * p.y_row + n;
    if (p.wide && n + 4 <= p.N) {
        fc_vec<DT, 4> out;
#pragma unroll
        for (int i = 0; i < 4; i++) out.set(i, __builtin_fmaf((float)sum[i] * xs, p.w_scale[n + i], p.bias ? p.bias[n + i] : 0.f));
        *(fc_vec<DT, 4> *)y = out;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < p.N) y[i] = (E)__builtin_fmaf((float)sum[i] * xs, p.w_scale[n + i], p.bias ? p.bias[n + i] : 0.f);
}

// Few tokens.  Bound by w, read once: a workgroup takes 16 * NF channels and up to 16 * MF tokens, its wavefronts take 128 bytes of the rows
// in turn, operands from memory straight into registers, and add up through LDS.
template <int DT, int MF, int NF, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void fc_int8_product_few_kernel(const product_params p) {
    __shared__ intx4 part[WAVES][MF * NF][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16 * NF;
    const long m0 = (long)blockIdx.y * 16 * MF;
    const int8_t *w[NF], *x[MF];
#pragma unroll
    for (int f = 0; f < NF; f++) w[f] = p.w + (n0 + 16 * f + r < p.N ? n0 + 16 * f + r : p.N - 1) * p.w_row;
#pragma unroll
    for (int f = 0; f < MF; f++) x[f] = p.x + (m0 + 16 * f + r < p.M ? m0 + 16 * f + r : p.M - 1) * p.x_row;
    intx4 sum[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) sum[i][j] = intx4{0, 0, 0, 0};
    int k = wave * kStage;
    for (; k + kStage <= p.K; k += WAVES * kStage) {
        intx4 a[2][NF], b[2][MF];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int f = 0; f < NF; f++) __builtin_memcpy(&a[h][f], w[f] + k + 64 * h + 16 * q, 16);
#pragma unroll
            for (int f = 0; f < MF; f++) __builtin_memcpy(&b[h][f], x[f] + k + 64 * h + 16 * q, 16);
        }
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < MF; i++)
#pragma unroll
                for (int j = 0; j < NF; j++) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[h][j], b[h][i], sum[i][j], 0, 0, 0);
    }
    if (k < p.K) {      // the last bytes
#pragma unroll
        for (int h = 0; h < 2; h++) {
            intx4 a[NF], b[MF];
#pragma unroll
            for (int f = 0; f < NF; f++) a[f] = row_word(w[f], k + 64 * h + 16 * q, p.K);
#pragma unroll
            for (int f = 0; f < MF; f++) b[f] = row_word(x[f], k + 64 * h + 16 * q, p.K);
#pragma unroll
            for (int i = 0; i < MF; i++)
#pragma unroll
                for (int j = 0; j < NF; j++) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[j], b[i], sum[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) part[wave][i * NF + j][lane] = sum[i][j];
    __syncthreads();
    for (int f = wave; f < MF * NF; f += WAVES) {
        intx4 s = part[0][f][lane];
#pragma unroll
        for (int v = 1; v < WAVES; v++) s += part[v][f][lane];
        // column of the product: token; four rows: channels
        const long m = m0 + 16 * (f / NF) + r;
        const int n = n0 + 16 * (f % NF) + 4 * q, four[4] = {s[0], s[1], s[2], s[3]};
        if (m < p.M && n < p.N) put<DT>(p, m, n, four, p.x_scale[m]);
    }
}

// Many tokens: tiles of BM tokens x BN channels, WM x WN wavefronts, stages of 128 bytes of the rows in LDS, two of them in turn.  Word c of a
// stage's row lies at place c ^ (row / 2 % 8), so that 16 neighbouring rows' words of one k cover all banks.  DIRECT: rows begin on and are multiples of 16
// bytes, which go to LDS without passing registers.
template <int DT, int BM, int BN, int WM, int WN, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN) void fc_int8_product_kernel(const product_params p) {
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, MI = BM / WM / 32, NI = BN / WN / 32, WORDS = (BM + BN) * 8, EACH = WORDS / THREADS;
    extern __shared__ intx4 lds[];      // [2][BN + BM rows][8]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // tiles in bands of eight rows of tiles, column by column, each XCD (workgroups are dealt to eight in turn) a contiguous part of them
    const unsigned tiles = gridDim.x, per = tiles / 8, rest = tiles % 8, xcd = blockIdx.x % 8;
    const unsigned id = xcd * per + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
    const unsigned band = id / (8 * p.tiles_n), in_band = id % (8 * p.tiles_n);
    const unsigned height = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
    const long m0 = (long)(band * 8 + in_band % height) * BM;
    const int n0 = (int)(in_band / height) * BN;

    // word i of a stage: row i / 8 (those of w first), place i % 8
    const int8_t *from[EACH];
    int k_of[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int i = (e * WAVES + wave) * 64 + lane, row = i >> 3;
        k_of[e] = ((i & 7) ^ (row >> 1 & 7)) * 16;
        if (row < BN) from[e] = p.w + (n0 + row < p.N ? n0 + row : p.N - 1) * p.w_row + k_of[e];
        else from[e] = p.x + (m0 + row - BN < p.M ? m0 + row - BN : p.M - 1) * p.x_row + k_of[e];
    }
    intx4 held[DIRECT ? 1 : EACH];
    auto fetch = [&](int k, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            if constexpr (DIRECT) {
                const void *at = k + k_of[e] < p.K ? (const void *)(from[e] + k) : (const void *)&kZeroWord;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)at,
                                                 (__attribute__((address_space(3))) void *)(lds + buf * WORDS + (e * WAVES + wave) * 64), 16, 0, 0);
            } else {
                held[e] = row_word(from[e] - k_of[e], k + k_of[e], p.K);
            }
        }
    };
    auto store = [&](int buf) __attribute__((always_inline)) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int e = 0; e < EACH; e++) lds[buf * WORDS + (e * WAVES + wave) * 64 + lane] = held[e];
        }
    };
    intx16 sum[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) sum[i][j] = intx16{};
    const int wm = wave / WN, wn = wave % WN, r = lane & 31, half = lane >> 5, turn = r >> 1 & 7;
    const int a_row = wn * (BN / WN) + r, b_row = BN + wm * (BM / WM) + r;
    fetch(0, 0);
    store(0);
    const int stages = (p.K + kStage - 1) / kStage;
    for (int s = 0; s < stages; s++) {
        __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0): this wavefront's words of the stage are in LDS
        __syncthreads();
        if (s + 1 < stages) fetch((s + 1) * kStage, (s + 1) & 1);
        const intx4 *at = lds + (s & 1) * WORDS;
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
            const int place = (2 * kk + half) ^ turn;
            intx4 a[NI], b[MI];
#pragma unroll
            for (int j = 0; j < NI; j++) a[j] = at[(a_row + 32 * j) * 8 + place];
#pragma unroll
            for (int i = 0; i < MI; i++) b[i] = at[(b_row + 32 * i) * 8 + place];
#pragma unroll
            for (int i = 0; i < MI; i++)
#pragma unroll
                for (int j = 0; j < NI; j++) sum[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[j], b[i], sum[i][j], 0, 0, 0);
        }
        if (s + 1 < stages) store((s + 1) & 1);
    }
#pragma unroll
    for (int i = 0; i < MI; i++) {
        const long m = m0 + wm * (BM / WM) + 32 * i + r;
        if (m >= p.M) continue;
        const float xs = p.x_scale[m];
#pragma unroll
        for (int j = 0; j < NI; j++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int n = n0 + wn * (BN / WN) + 32 * j + 8 * g + 4 * half;
                const int four[4] = {sum[i][j][4 * g], sum[i][j][4 * g + 1], sum[i][j][4 * g + 2], sum[i][j][4 * g + 3]};
                if (n < p.N) put<DT>(p, m, n, four, xs);
            }
    }
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

template <int DT, int BM, int BN, int WM, int WN>
int run_tiles(fc_context *ctx, product_params &p, bool direct) {
    p.tiles_m = (int)((p.M + BM - 1) / BM);
    p.tiles_n = (p.N + BN - 1) / BN;
    constexpr size_t lds = 2 * (BM + BN) * kStage;
    const dim3 grid((unsigned)((long)p.tiles_m * p.tiles_n)), threads(64 * WM * WN);
    const auto kernel = direct ? fc_int8_product_kernel<DT, BM, BN, WM, WN, true> : fc_int8_product_kernel<DT, BM, BN, WM, WN, false>;
    if (lds > 65536) FC_HIP_CHECK(ctx, hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    kernel<<<grid, threads, lds, ctx->stream>>>(p);
    FC_LAUNCH_CHECK(ctx, "fc_int8_product_kernel");
    return FC_OK;
}

template <int DT, int MF>
int run_few(fc_context *ctx, const product_params &p) {
    constexpr int NF = 1, WAVES = 8;
    fc_int8_product_few_kernel<DT, MF, NF, WAVES><<<dim3((unsigned)((p.N + 16 * NF - 1) / (16 * NF)), (unsigned)((p.M + 16 * MF - 1) / (16 * MF))),
                                                    dim3(64 * WAVES), 0, ctx->stream>>>(p);
    FC_LAUNCH_CHECK(ctx, "fc_int8_product_few_kernel");
    return FC_OK;
}

template <int DT>
int run(fc_context *ctx, product_params &p, int tile, bool direct) {
    if (tile == 0) {
        if (p.M <= 16) return run_few<DT, 1>(ctx, p);
        if (p.M <= 32) return run_few<DT, 2>(ctx, p);
        return run_few<DT, 4>(ctx, p);
    }
    if (tile == 256) return run_tiles<DT, 256, 256, 2, 4>(ctx, p, direct);
    if (tile == 128) return run_tiles<DT, 128, 128, 2, 2>(ctx, p, direct);
    return run_tiles<DT, 64, 64, 2, 2>(ctx, p, direct);
}

bool same(const fc_int8_product_plan &a, const fc_int8_product_plan &b) {
    const fc_int8_product_shape &s = a.shape, &t = b.shape;
    return s.M == t.M && s.N == t.N && s.K == t.K && s.dtype == t.dtype && s.x_row == t.x_row && s.w_row == t.w_row && s.y_row == t.y_row &&
           a.tile == b.tile && a.ws_bytes == b.ws_bytes;
}

}  // namespace

extern "C" int fc_int8_product_make_plan(const fc_int8_product_shape *s, fc_int8_product_plan *plan) {
    if (!plan || !s || s->M < 1 || s->N < 1 || s->K < 1 || !fc_dtype_ok(s->dtype) || s->x_row < 0 || s->w_row < 0 || s->y_row < 0) return FC_ERR_INVALID;
    if (s->K > kMostTerms || s->M >= (1l << 31) || fc_count(s->M, s->N) >= (1l << 36)) return FC_ERR_UNSUPPORTED;
    *plan = {};
    plan->shape = *s;
    auto tiles = [&](long side) { return (s->M + side - 1) / side * ((s->N + side - 1) / side); };
    plan->tile = s->M <= 64 ? 0 : tiles(256) >= 256 ? 256 : tiles(128) >= 256 ? 128 : 64;
    return FC_OK;
}

extern "C" int fc_int8_product(fc_context *ctx, const fc_int8_product_plan *plan, const int8_t *x_dev, const float *x_scale_dev, const int8_t *w_dev,
                               const float *w_scale_dev, const float *bias_dev, void *y_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    fc_int8_product_plan own;
    if (!plan || fc_int8_product_make_plan(&plan->shape, &own) != FC_OK || !same(*plan, own))
        return fail(ctx, FC_ERR_INVALID, "fc_int8_product: not a plan of fc_int8_product_make_plan");
    const fc_int8_product_shape &s = plan->shape;
    if (!x_dev || !x_scale_dev || !w_dev || !w_scale_dev || !y_dev || (!ws_dev && plan->ws_bytes)) return fail(ctx, FC_ERR_INVALID, "fc_int8_product: null pointer");
    if ((((uint64_t)x_scale_dev | (uint64_t)w_scale_dev | (uint64_t)bias_dev | (uint64_t)ws_dev) & 3) || ((uint64_t)y_dev & (fc_elem_size(s.dtype) - 1)))
        return fail(ctx, FC_ERR_INVALID, "fc_int8_product: unaligned pointer");
    if (!fc_apart(s.M, s.y_row, s.N)) return fail(ctx, FC_ERR_INVALID, "fc_int8_product: rows of y overlap");
    product_params p = {};
    p.x = x_dev; p.w = w_dev; p.x_scale = x_scale_dev; p.w_scale = w_scale_dev; p.bias = bias_dev; p.y = y_dev;
    p.M = s.M; p.N = s.N; p.K = s.K; p.x_row = s.x_row; p.w_row = s.w_row; p.y_row = s.y_row;
    p.wide = ((s.N | s.y_row) & 3) == 0 && ((uint64_t)y_dev & (4 * fc_elem_size(s.dtype) - 1)) == 0;
    const bool direct = ((s.K | s.x_row | s.w_row) & 15) == 0 && (((uint64_t)x_dev | (uint64_t)w_dev) & 15) == 0;
    const fc_device_scope on(ctx);
    if (s.dtype == FC_F32) return run<FC_F32>(ctx, p, plan->tile, direct);
    if (s.dtype == FC_BF16) return run<FC_BF16>(ctx, p, plan->tile, direct);
    return run<FC_F16>(ctx, p, plan->tile, direct);
}
