// Products of 8-bit rows with scales for each row (token) and each column (channel):
//
//   y[m][n] = (sum over k of x[m][k] w[n][k]) * x_scale[m] * w_scale[n] + bias[n]
//
// Sums are 32-bit integers, exact up to 131071 terms whatever their order, so every kernel here gives the same bits.  x and w are rows of k: 16 bytes of a
// row are a lane's operand of v_mfma_i32_16x16x64_i8 and v_mfma_i32_32x32x32_i8 as they lie.  w is the first operand: a lane then holds four
// neighbouring channels of one token.
#include <math.h>

#include <type_traits>

#include "token_types.h"

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

constexpr int kMostTerms = 131071;      // of 128 * 128 each: 2^31 - 2^14
constexpr int kStage = 64;              // bytes of a row that a tile takes at once: 4 words of 16
constexpr int kFewStage = 128;          // bytes of a row that a wavefront takes at once where tokens are few

__device__ const intx4 kZeroWord = {0, 0, 0, 0};

struct product_params {
    const int8_t *x, *w;
    const float *x_scale, *w_scale, *bias;
    void *y;
    long M;
    int N, K;
    long x_row, w_row, y_row;
    int tiles_m, tiles_n;
    int *parts_at;           // [parts][M][N], where the reduction is cut
    int part;                // bytes of a row that a part takes
};

// 16 bytes of a row from k on, wherever they begin; zeros past its end.
__device__ __forceinline__ intx4 row_word(const int8_t *row, int k, int K) {
    intx4 v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else if (k < K && K >= 16) {      // the row's last 16, moved down
        unsigned __int128 last;
        __builtin_memcpy(&last, row + K - 16, 16);
        last >>= 8 * (k + 16 - K);
        __builtin_memcpy(&v, &last, 16);
    } else if (k < K) {
        unsigned u[4] = {0, 0, 0, 0};
        for (int i = 0; i < K - k; i++) u[i >> 2] |= (unsigned)(uint8_t)row[k + i] << (8 * (i & 3));
        v = {(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
    }
    return v;
}

// Four neighbours of a part's sums.
__device__ __forceinline__ void put_part(const product_params &p, long m, int n, intx4 sum) {
    int *to = p.parts_at + ((long)blockIdx.z * p.M + m) * p.N + n;
    if (n + 4 <= p.N) {
        __builtin_memcpy(to, &sum, 16);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < p.N) to[i] = sum[i];
}

// sum * xs * ws, and a bias: a sum below 2^31 times a scale above 2^96 may leave fp32's numbers although the other scale brings it back, so that one goes first then.
__device__ __forceinline__ float scaled(int sum, float xs, float ws) {
    const bool far = __builtin_fabsf(xs) > 0x1p96f;
    return (float)sum * (far ? ws : xs) * (far ? xs : ws);
}
__device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) {
    const bool far = __builtin_fabsf(xs) > 0x1p96f;
    return __builtin_fmaf((float)sum * (far ? ws : xs), far ? xs : ws, bias);
}

// Four neighbouring channels, from n on, of token m.
template <int DT>
__device__ __forceinline__ void put(const product_params &p, long m, int n, const int (&sum)[4], float xs) {
    typedef typename fc_elem<DT>::type E;
    E *y = (E *)p.y + m * p.y_row + n;
    if (n + 4 <= p.N) {
        float ws[4], bias[4] = {0.f, 0.f, 0.f, 0.f};
        __builtin_memcpy(ws, p.w_scale + n, sizeof ws);
        if (p.bias) __builtin_memcpy(bias, p.bias + n, sizeof bias);
        fc_vec<DT, 4> out;
#pragma unroll
        for (int i = 0; i < 4; i++) out.set(i, p.bias ? scaled(sum[i], xs, ws[i], bias[i]) : scaled(sum[i], xs, ws[i]));
        __builtin_memcpy(y, &out, sizeof out);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (n + i < p.N) y[i] = (E)(p.bias ? scaled(sum[i], xs, p.w_scale[n + i], p.bias[n + i]) : scaled(sum[i], xs, p.w_scale[n + i]));
}

// What a lane has of a product of 16 tokens and 16 channels: column, a token; four rows, channels.
template <int DT>
__device__ __forceinline__ void put_few(const product_params &p, long m, int n, intx4 s) {
    const int four[4] = {s[0], s[1], s[2], s[3]};
    if (m >= p.M || n >= p.N) return;
    if (p.parts_at) put_part(p, m, n, s);
    else put<DT>(p, m, n, four, p.x_scale[m]);
}

// Few tokens.  Bound by w, read once: a workgroup takes 16 * NF channels and up to 16 * MF tokens, its wavefronts take 128 bytes of the rows
// in turn, operands from memory straight into registers, and add up through LDS.  This is for rows that begin anywhere; 64 tokens, 8192 channels of 4096: 14.7 us.
template <int DT, int MF, int NF, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void fc_int8_product_few_kernel(const product_params p) {
    __shared__ intx4 part[WAVES][MF * NF][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16 * NF;
    const long m0 = (long)blockIdx.y * 16 * MF;
    const int8_t *w[NF], *x[MF];
    const int k0 = blockIdx.z * p.part, K = p.K - k0 < p.part ? p.K - k0 : p.part;
#pragma unroll
    for (int f = 0; f < NF; f++) w[f] = p.w + k0 + (n0 + 16 * f + r < p.N ? n0 + 16 * f + r : p.N - 1) * p.w_row;
#pragma unroll
    for (int f = 0; f < MF; f++) x[f] = p.x + k0 + (m0 + 16 * f + r < p.M ? m0 + 16 * f + r : p.M - 1) * p.x_row;
    intx4 sum[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) sum[i][j] = intx4{0, 0, 0, 0};
    // two steps' operands in registers: one is on its way while the other is used
    intx4 a[2][2][NF], b[2][2][MF];
    auto read = [&](int k, int turn) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int f = 0; f < NF; f++) __builtin_memcpy(&a[turn][h][f], w[f] + k + 64 * h + 16 * q, 16);
#pragma unroll
            for (int f = 0; f < MF; f++) __builtin_memcpy(&b[turn][h][f], x[f] + k + 64 * h + 16 * q, 16);
        }
    };
    auto use = [&](int turn) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < MF; i++)
#pragma unroll
                for (int j = 0; j < NF; j++) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[turn][h][j], b[turn][h][i], sum[i][j], 0, 0, 0);
    };
    constexpr int STEP = WAVES * kFewStage;
    int k = wave * kFewStage;
    if (k + kFewStage <= K) read(k, 0);
    for (; k + STEP + kFewStage <= K; k += 2 * STEP) {
        read(k + STEP, 1);
        use(0);
        if (k + 2 * STEP + kFewStage <= K) read(k + 2 * STEP, 0);
        use(1);
    }
    if (k + kFewStage <= K) {
        use(0);
        k += STEP;
    }
    if (k < K) {      // the last bytes
#pragma unroll
        for (int h = 0; h < 2; h++) {
            intx4 a[NF], b[MF];
#pragma unroll
            for (int f = 0; f < NF; f++) a[f] = row_word(w[f], k + 64 * h + 16 * q, K);
#pragma unroll
            for (int f = 0; f < MF; f++) b[f] = row_word(x[f], k + 64 * h + 16 * q, K);
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
        put_few<DT>(p, m0 + 16 * (f / NF) + r, n0 + 16 * (f % NF) + 4 * q, s);
    }
}

// The same where rows begin on and are multiples of 16 bytes.  Eight neighbouring lanes read 128 bytes of a row, which go to LDS without passing registers: an
// operand's own lanes lie in 16 rows each, and a load of them takes the L1 four times as long.  A wavefront has a ring of its own and waits for nobody.  64 tokens,
// 8192 channels of 4096: 8.3 us (33.5 MB of w, 4.0 TB/s); 16 tokens 5.2 us; 1 token, 16384 channels 13.0 us (5.2 TB/s); an empty launch takes about 4.5.
template <int DT, int MF, int NF, int WAVES, int BUFFERS>
__global__ __launch_bounds__(64 * WAVES) void fc_int8_product_ring_kernel(const product_params p) {
    static_assert(BUFFERS <= 2);
    constexpr int LOADS = 2 * (NF + MF), WORDS = LOADS * 64;
    extern __shared__ intx4 lds[];      // [WAVES][BUFFERS][16 * (NF + MF) rows][8]; then the wavefronts' sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16 * NF;
    const long m0 = (long)blockIdx.y * 16 * MF;
    const int k0 = blockIdx.z * p.part, K = p.K - k0 < p.part ? p.K - k0 : p.part;
    // load e: eight rows of the stage, those of w first; word c of a row lies at place c ^ (row % 8)
    const int k_of = ((lane & 7) ^ (lane >> 3)) * 16;
    const int8_t *const w = p.w + n0 * p.w_row + k0, *const x = p.x + m0 * p.x_row + k0;
    uint32_t off[LOADS];
#pragma unroll
    for (int e = 0; e < LOADS; e++) {
        const int row = 8 * (e < 2 * NF ? e : e - 2 * NF) + (lane >> 3);
        const long at = e < 2 * NF ? (n0 + row < p.N ? row : p.N - 1 - n0) * p.w_row : (m0 + row < p.M ? row : p.M - 1 - m0) * p.x_row;
        off[e] = (uint32_t)at + k_of;
    }
    const int all = (K + kFewStage - 1) / kFewStage, steps = all > wave ? (all - wave - 1) / WAVES + 1 : 0;
    // Workgroups begin at steps of their own: rows a power of two apart have their bytes of one step in few of the L2's channels.  64 tokens, 16384 channels of 8192:
    // 24.6 us, and 33.7 if all begin at the first.
    unsigned turn = steps ? (blockIdx.x / 8) % steps : 0;
    intx4 *const ring = lds + wave * BUFFERS * WORDS;
    auto fetch = [&](int s) __attribute__((always_inline)) {
        const int k = (wave + (int)turn * WAVES) * kFewStage;
        turn = turn + 1 < (unsigned)steps ? turn + 1 : 0;
        const int8_t *wk = uniform_ptr(w + k), *xk = uniform_ptr(x + k);
        intx4 *to = ring + s % BUFFERS * WORDS;
#pragma unroll
        for (int e = 0; e < LOADS; e++) {
            const void *at = (e < 2 * NF ? wk : xk) + off[e];
            if (k + kFewStage > K && k + k_of >= K) at = &kZeroWord;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)at, (__attribute__((address_space(3))) void *)(to + e * 64), 16, 0, 0);
        }
    };
    intx4 sum[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) sum[i][j] = intx4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < BUFFERS; s++)
        if (s < steps) fetch(s);
    for (int s = 0; s < steps; s++) {
        // all but the next step's loads have arrived
        if (BUFFERS > 1 && s + 1 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(BUFFERS > 1 ? LOADS : 0) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const intx4 *at = ring + s % BUFFERS * WORDS + r * 8;
        intx4 a[2][NF], b[2][MF];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int f = 0; f < NF; f++) a[h][f] = at[f * 128 + ((4 * h + q) ^ (r & 7))];
#pragma unroll
            for (int f = 0; f < MF; f++) b[h][f] = at[(NF + f) * 128 + ((4 * h + q) ^ (r & 7))];
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // read, before they are written over
        if (s + BUFFERS < steps) fetch(s + BUFFERS);
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < MF; i++)
#pragma unroll
                for (int j = 0; j < NF; j++) sum[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[h][j], b[h][i], sum[i][j], 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MF; i++)
#pragma unroll
        for (int j = 0; j < NF; j++) lds[(wave * MF * NF + i * NF + j) * 64 + lane] = sum[i][j];
    __syncthreads();
    for (int f = wave; f < MF * NF; f += WAVES) {
        intx4 s = lds[f * 64 + lane];
#pragma unroll
        for (int v = 1; v < WAVES; v++) s += lds[(v * MF * NF + f) * 64 + lane];
        put_few<DT>(p, m0 + 16 * (f / NF) + r, n0 + 16 * (f % NF) + 4 * q, s);
    }
}

// Many tokens: tiles of BM tokens x BN channels, WM x WN wavefronts, stages of 64 bytes of the rows in LDS, read two stages before they are ready and one
// more before they are used, so that a wavefront's first operands of a stage arrive under the products of the one before.  Word c of a stage's row lies
// at place c ^ (row / 4 % 4): 16 neighbouring rows' words of one k cover all banks.  DIRECT: rows begin on and are multiples of 16 bytes, which go to
// LDS without passing registers.  12544 x 8192 of 4096, bf16: 435 to 453 us, 1.86 to 1.94e15 operations a second; 8192 x 8192 of 8192 2.19e15.  The clock gives way to
// power: the same with zeros for values takes 349 us; 12288 rows (six tiles a unit instead of 49 / 8) 411; four wavefronts of 128 x 128 479, stages begun in turn by the workgroups 446 to 461.
template <int DT, int BM, int BN, int WM, int WN, int BUFFERS, bool DIRECT>
__global__ __launch_bounds__(64 * WM * WN, BM / WM * (BN / WN) > 8192 ? 1 : 2) void fc_int8_product_kernel(const product_params p) {
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, MI = BM / WM / 32, NI = BN / WN / 32, WORDS = (BM + BN) * 4, EACH = WORDS / THREADS;
    extern __shared__ intx4 lds[];      // [BUFFERS][BN + BM rows][4]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // tiles in bands of eight rows of tiles, column by column, each XCD (workgroups are dealt to eight in turn) a contiguous part of them
    const unsigned tiles = gridDim.x, per = tiles / 8, rest = tiles % 8, xcd = blockIdx.x % 8;
    const unsigned id = xcd * per + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
    const unsigned band = id / (8 * p.tiles_n), in_band = id % (8 * p.tiles_n);
    const unsigned height = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
    const long m0 = (long)(band * 8 + in_band % height) * BM;
    const int n0 = (int)(in_band / height) * BN;

    // word i of a stage: row i / 4 (those of w first), place i % 4.  DIRECT: 32-bit offsets from where the tile begins, which moves on with the stages.
    const int k_of = ((lane & 3) ^ (lane >> 4 & 3)) * 16;      // rows of an access begin at a multiple of 16
    const int k0 = blockIdx.z * p.part, K = p.K - k0 < p.part ? p.K - k0 : p.part;
    const int8_t *const w_tile = p.w + n0 * p.w_row + k0, *const x_tile = p.x + m0 * p.x_row + k0;
    uint32_t off[DIRECT ? EACH : 1];
    const int8_t *from[DIRECT ? 1 : EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int row = ((e * WAVES + wave) * 64 + lane) >> 2;
        const bool of_w = e * WAVES * 16 < BN;      // of the whole access: BN is a multiple of its rows
        const long at = of_w ? n0 + row < p.N ? row : p.N - 1 - n0 : m0 + row - BN < p.M ? row - BN : p.M - 1 - m0;
        if constexpr (DIRECT) off[e] = (uint32_t)(at * (of_w ? p.w_row : p.x_row)) + k_of;
        else from[e] = (of_w ? w_tile + at * p.w_row : x_tile + at * p.x_row) + k_of;
    }
    static_assert(BN % (16 * WAVES) == 0);
    const int stages = (K + kStage - 1) / kStage;
    intx4 held[DIRECT ? 1 : EACH];
    auto fetch = [&](int s, auto whole) __attribute__((always_inline)) {      // whole: the stage is known to be there, all of it
        const int k = s * kStage;
        if constexpr (DIRECT) {
            intx4 *to = lds + (s % BUFFERS) * WORDS + wave * 64;
            const int8_t *w = uniform_ptr(w_tile + k), *x = uniform_ptr(x_tile + k);
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                const void *at = (e * WAVES * 16 < BN ? w : x) + off[e];
                if (!whole && k + k_of >= K) at = &kZeroWord;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)at, (__attribute__((address_space(3))) void *)(to + e * THREADS),
                                                 16, 0, 0);
            }
        } else {
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                if (whole || k + kStage <= K) __builtin_memcpy(&held[e], from[e] + k, 16);
                else held[e] = row_word(from[e] - k_of, k + k_of, K);
            }
        }
    };
    auto store = [&](int s) __attribute__((always_inline)) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int e = 0; e < EACH; e++) lds[(s % BUFFERS) * WORDS + e * THREADS + wave * 64 + lane] = held[e];
        }
    };
    // This wavefront's words are in LDS but for those of `later` stages; then everybody's are, and everybody has read the stage before the last.  In one block of
    // assembly: a fence would wait for all loads on their way.
    auto ready = [&](bool later) __attribute__((always_inline)) {
        if (DIRECT && BUFFERS > 3 && later) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((BUFFERS - 3) * EACH) : "memory");
        else if (DIRECT) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    intx16 sum[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
        for (int j = 0; j < NI; j++) sum[i][j] = intx16{};
    const int wm = wave / WN, wn = wave % WN, r = lane & 31, half = lane >> 5, turn = r >> 2 & 3;
    const int a_row = (wn * (BN / WN) + r) * 4, b_row = (BN + wm * (BM / WM) + r) * 4;
    intx4 a[2][NI], b[2][MI];
    auto operands = [&](int s, int kk) __attribute__((always_inline)) {
        const intx4 *at = lds + (s % BUFFERS) * WORDS + ((2 * kk + half) ^ turn);
#pragma unroll
        for (int j = 0; j < NI; j++) a[kk][j] = at[a_row + 128 * j];
#pragma unroll
        for (int i = 0; i < MI; i++) b[kk][i] = at[b_row + 128 * i];
    };
    auto products = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int j = 0; j < NI; j++) sum[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[kk][j], b[kk][i], sum[i][j], 0, 0, 0);
    };
    // stage s is in use, s + 1 ready, the others on their way; without DIRECT, s + 2 in registers
    constexpr int AHEAD = DIRECT ? BUFFERS - 1 : 2;
    const std::false_type some;
    const std::true_type all;
    fetch(0, some);
    store(0);
    if (1 < stages) fetch(1, some);
    if (1 < stages) store(1);
    if (AHEAD > 2 || !DIRECT)
        if (2 < stages) fetch(2, some);
    ready(false);
    operands(0, 0);
    int s = 0;
    if (AHEAD < stages && DIRECT) fetch(AHEAD, some);
    operands(0, 1);
    products(0);
    if (1 < stages) operands(1, 0);
    products(1);
    for (s = 1; s + AHEAD < stages - 1; s++) {      // the last stage may not be whole
        store(s + 1);
        ready(true);      // stage s + 1
        fetch(s + AHEAD, all);
        operands(s, 1);
        products(0);
        operands(s + 1, 0);
        products(1);
    }
    for (; s < stages; s++) {
        if (s + 1 < stages) store(s + 1);
        ready(s + 2 < stages);
        if (s + AHEAD < stages) fetch(s + AHEAD, some);
        operands(s, 1);
        products(0);
        if (s + 1 < stages) operands(s + 1, 0);
        products(1);
    }
    // A lane has one token and, of every eight channels, four neighbours.  They are laid out as rows in LDS, 32 tokens of the wavefront at a time, and leave in
    // whole lines.
    if (p.parts_at) {
#pragma unroll
        for (int i = 0; i < MI; i++) {
            const long m = m0 + wm * (BM / WM) + 32 * i + r;
#pragma unroll
            for (int j = 0; j < NI; j++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int n = n0 + wn * (BN / WN) + 32 * j + 8 * g + 4 * half;
                    const intx4 four = {sum[i][j][4 * g], sum[i][j][4 * g + 1], sum[i][j][4 * g + 2], sum[i][j][4 * g + 3]};
                    if (m < p.M && n < p.N) put_part(p, m, n, four);
                }
        }
        return;
    }
    typedef typename fc_elem<DT>::type E;
    constexpr int VEC = 16 / (int)sizeof(E), COLS = BN / WN, PITCH = COLS * (int)sizeof(E) + 16, PER_ROW = COLS / VEC, AT_ONCE = 64 / PER_ROW;
    static_assert(WAVES * 32 * PITCH <= BUFFERS * WORDS * 16);
    const int n_wave = n0 + wn * COLS;
    float ws[NI][4][4], bias[NI][4][4];
#pragma unroll
    for (int j = 0; j < NI; j++)
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int n = n_wave + 32 * j + 8 * g + 4 * half;
            if (n0 + BN <= p.N) {
                __builtin_memcpy(ws[j][g], p.w_scale + n, 16);
                if (p.bias) __builtin_memcpy(bias[j][g], p.bias + n, 16);
            } else {
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const int at = n + v < p.N ? n + v : p.N - 1;
                    ws[j][g][v] = p.w_scale[at];
                    if (p.bias) bias[j][g][v] = p.bias[at];
                }
            }
        }
    float xs[MI];
#pragma unroll
    for (int i = 0; i < MI; i++) {
        const long m = m0 + wm * (BM / WM) + 32 * i + r;
        xs[i] = p.x_scale[m < p.M ? m : p.M - 1];
    }
    __syncthreads();      // everybody's operands are read
    char *mine = (char *)lds + wave * 32 * PITCH;
    const int row = lane / PER_ROW, col = lane % PER_ROW * VEC;
#pragma unroll
    for (int i = 0; i < MI; i++) {
#pragma unroll
        for (int j = 0; j < NI; j++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                fc_vec<DT, 4> out;
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const int whole = sum[i][j][4 * g + v];
                    out.set(v, p.bias ? scaled(whole, xs[i], ws[j][g][v], bias[j][g][v]) : scaled(whole, xs[i], ws[j][g][v]));
                }
                *(fc_vec<DT, 4> *)(mine + r * PITCH + (32 * j + 8 * g + 4 * half) * sizeof(E)) = out;
            }
        fc_wave_sync();
#pragma unroll
        for (int k = 0; k < 32 / AT_ONCE; k++) {
            const fc_vec<DT, VEC> out = *(const fc_vec<DT, VEC> *)(mine + (row + k * AT_ONCE) * PITCH + col * sizeof(E));
            const long m = m0 + wm * (BM / WM) + 32 * i + row + k * AT_ONCE;
            if (m >= p.M) continue;
            E *to = (E *)p.y + m * p.y_row + n_wave + col;
            if (n_wave + col + VEC <= p.N) {
                __builtin_memcpy(to, &out, 16);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; v++)
                    if (n_wave + col + v < p.N) to[v] = out.v[v];
            }
        }
        fc_wave_sync();
    }
}

// The parts' sums added up, scaled and stored, four channels a thread.
template <int DT>
__global__ __launch_bounds__(256) void fc_int8_product_join_kernel(const product_params p, int parts) {
    const int quads = (p.N + 3) / 4;
    const long i = (long)blockIdx.x * 256 + threadIdx.x, m = i / quads;
    const int n = (int)(i - m * quads) * 4;
    if (m >= p.M) return;
    int four[4] = {0, 0, 0, 0};
    const int *from = p.parts_at + m * p.N + n;
    const long part = p.M * p.N;
    for (int first = 0; first < parts; first += 4) {      // four on their way at once
        int v[4][4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int *at = from + (first + k < parts ? first + k : 0) * part;
            if (n + 4 <= p.N) {
                __builtin_memcpy(v[k], at, 16);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[k][j] = at[n + j < p.N ? j : 0];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) four[j] += first + k < parts ? v[k][j] : 0;
    }
    put<DT>(p, m, n, four, p.x_scale[m]);
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

// What the rows of a plan run on.
struct product_form {
    int tile;                // tokens and channels of a workgroup's tile; 0: few tokens
    int mf, nf;              // few tokens: blocks of 16 of a workgroup
    int parts;               // of the reduction
    double us;               // expected
};

long ceil_div(long a, long b) { return (a + b - 1) / b; }

constexpr int kFewTokens = 64;
constexpr long kUnits = 256;      // compute units

// Few tokens.  Wide workgroups read x seldom, many read w side by side: the widest of which there is one a unit.  8192 channels of 4096, 64 tokens: 64x32 8.4 us,
// 32x32 11.5, 16x32 16.5; 4096 channels 7.8, 6.3 and 8.6; 2048 channels 6.9, 5.4 and 5.0; 32 tokens of 8192 channels 7.3, 6.6 and 8.8; 16 tokens of 8192 channels
// 16x32 5.3 and 16x16 6.0.
product_form few_form(long M, int N) {
    const int forms[4][2] = {{4, 2}, {2, 2}, {1, 2}, {1, 1}};
    product_form f = {};
    for (const auto &v : forms) {
        f.mf = v[0];
        f.nf = v[1];
        if (f.mf > 1 && M <= 8 * f.mf) continue;
        if (ceil_div(M, 16 * f.mf) * ceil_div(N, 16 * f.nf) >= kUnits) break;
    }
    f.parts = 1;
    return f;
}

// Tiles.  Times of a call in us by tiles a compute unit, c, and 1024 bytes of the reduction, k, fitted to products of 256 to 12288 rows.
double tile_time(int tile, long M, int N, int K) {
    const double tiles = (double)(ceil_div(M, tile) * ceil_div(N, tile)), c = tiles / kUnits, k = K / 1024.0;
    if (tile == 64) return 3 + 0.4 * c + k * (c < 0.9 ? 2.2 : 2.4 * c);
    if (tile == 128) return 3 + 2.4 * c + k * (c < 0.8 ? 4.2 : 5.2 * c);
    return c > 1 ? ceil(c) * (10 + 14.5 * k) : 8 + 2 * c + k * (10 + 5 * c);
}

product_form best_tile(long M, int N, int K) {
    product_form f = {};
    f.parts = 1;
    for (int tile : {64, 128, 256}) {
        const double us = tile_time(tile, M, N, K);
        if (!f.tile || us < f.us) {
            f.tile = tile;
            f.us = us;
        }
    }
    return f;
}

// Workgroups that leave most of the chip idle cut a reduction of `least` bytes and more; adding the parts up is a launch more.  With and without: 1 token, 64
// channels of 65536 11.5 and 18.6 us, 512 channels of 16384 6.8 and 6.8, of 8192 8.0 and 4.7; 300 tokens, 520 channels of 8192 12.7 and 20.4; 200 tokens, 1000
// channels of 4096 10.2 and 12.2, of 2048 10.4 and 8.1.
void cut(product_form &f, long workgroups, int K, int least) {
    if (workgroups > kUnits / 4 || K < least) return;
    long parts = kUnits / workgroups;
    if (parts > K / 1024) parts = K / 1024;
    const long part = ceil_div(ceil_div(K, parts), 128) * 128;
    f.parts = (int)ceil_div(K, part);
}

template <int DT, int BM, int BN, int WM, int WN, int BUFFERS>
int run_tiles(fc_context *ctx, product_params p, int parts, bool direct) {
    p.tiles_m = (int)((p.M + BM - 1) / BM);
    p.tiles_n = (p.N + BN - 1) / BN;
    constexpr size_t lds = BUFFERS * (BM + BN) * kStage;
    const dim3 grid((unsigned)((long)p.tiles_m * p.tiles_n), 1, (unsigned)parts), threads(64 * WM * WN);
    const auto kernel = direct ? fc_int8_product_kernel<DT, BM, BN, WM, WN, BUFFERS, true> : fc_int8_product_kernel<DT, BM, BN, WM, WN, BUFFERS, false>;
    if (lds > 65536) FC_HIP_CHECK(ctx, hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    kernel<<<grid, threads, lds, ctx->stream>>>(p);
    FC_LAUNCH_CHECK(ctx, "fc_int8_product_kernel");
    return FC_OK;
}

template <int DT, int MF, int NF>
int run_few(fc_context *ctx, const product_params &p, int parts, bool direct) {
    const dim3 grid((unsigned)ceil_div(p.N, 16 * NF), (unsigned)ceil_div(p.M, 16 * MF), (unsigned)parts);
    if (direct) {
        constexpr int WAVES = 8, BUFFERS = MF == 4 ? 1 : 2;
        constexpr size_t lds = (size_t)WAVES * BUFFERS * 2 * (NF + MF) * 1024;
        static_assert(lds <= 160 * 1024 && lds >= (size_t)WAVES * MF * NF * 1024);
        const auto kernel = fc_int8_product_ring_kernel<DT, MF, NF, WAVES, BUFFERS>;
        if (lds > 65536) FC_HIP_CHECK(ctx, hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        kernel<<<grid, dim3(64 * WAVES), lds, ctx->stream>>>(p);
        FC_LAUNCH_CHECK(ctx, "fc_int8_product_ring_kernel");
        return FC_OK;
    }
    constexpr int WAVES = 8;
    fc_int8_product_few_kernel<DT, MF, NF, WAVES><<<grid, dim3(64 * WAVES), 0, ctx->stream>>>(p);
    FC_LAUNCH_CHECK(ctx, "fc_int8_product_few_kernel");
    return FC_OK;
}

template <int DT>
int run_form(fc_context *ctx, product_params p, const product_form &f, bool direct, void *ws) {
    p.part = (int)(ceil_div(ceil_div(p.K, f.parts), 128) * 128);
    p.parts_at = f.parts > 1 ? (int *)ws : nullptr;
    int rc;
    if (f.tile == 0)
        rc = f.mf == 4 ? run_few<DT, 4, 2>(ctx, p, f.parts, direct) : f.mf == 2 ? run_few<DT, 2, 2>(ctx, p, f.parts, direct) : f.nf == 2 ? run_few<DT, 1, 2>(ctx, p, f.parts, direct) : run_few<DT, 1, 1>(ctx, p, f.parts, direct);
    else
        rc = f.tile == 256   ? run_tiles<DT, 256, 256, 2, 4, 4>(ctx, p, f.parts, direct)
             : f.tile == 128 ? run_tiles<DT, 128, 128, 2, 2, 4>(ctx, p, f.parts, direct)
                             : run_tiles<DT, 64, 64, 2, 2, 4>(ctx, p, f.parts, direct);
    if (rc || f.parts == 1) return rc;
    fc_int8_product_join_kernel<DT><<<dim3((unsigned)ceil_div(p.M * ((p.N + 3) / 4), 256)), dim3(256), 0, ctx->stream>>>(p, f.parts);
    FC_LAUNCH_CHECK(ctx, "fc_int8_product_join_kernel");
    return FC_OK;
}

template <int DT>
int run(fc_context *ctx, const product_params &p, const fc_int8_product_plan *plan, bool direct, void *ws) {
    if (p.M <= kFewTokens) {
        product_form f = few_form(p.M, p.N);
        f.parts = plan->parts;
        return run_form<DT>(ctx, p, f, direct, ws);
    }
    product_form f = {};
    f.tile = plan->tile;
    f.parts = plan->parts;
    return run_form<DT>(ctx, p, f, direct, ws);
}

bool same(const fc_int8_product_plan &a, const fc_int8_product_plan &b) {
    const fc_int8_product_shape &s = a.shape, &t = b.shape;
    return s.M == t.M && s.N == t.N && s.K == t.K && s.dtype == t.dtype && s.x_row == t.x_row && s.w_row == t.w_row && s.y_row == t.y_row &&
           a.tile == b.tile && a.parts == b.parts && a.ws_bytes == b.ws_bytes;
}

}  // namespace

extern "C" int fc_int8_product_make_plan(const fc_int8_product_shape *s, fc_int8_product_plan *plan) {
    if (!plan || !s || s->M < 1 || s->N < 1 || s->K < 1 || !fc_dtype_ok(s->dtype) || s->x_row < 0 || s->w_row < 0 || s->y_row < 0) return FC_ERR_INVALID;
    if (s->K > kMostTerms || s->M >= (1l << 31) || fc_count(s->M, s->N) >= (1l << 36)) return FC_ERR_UNSUPPORTED;
    *plan = {};
    product_form f;
    if (s->M <= kFewTokens) {
        f = few_form(s->M, s->N);
        cut(f, ceil_div(s->M, 16 * f.mf) * ceil_div(s->N, 16 * f.nf), s->K, 32768);
    } else {
        f = best_tile(s->M, s->N, s->K);
        cut(f, ceil_div(s->M, f.tile) * ceil_div(s->N, f.tile), s->K, 4096);
    }
    // a launch has fewer than 2^32 threads
    const long threads = f.tile == 256 || !f.tile ? 512 : 256;
    const long workgroups = f.tile ? ceil_div(s->M, f.tile) * ceil_div(s->N, f.tile) : ceil_div(s->M, 16 * f.mf) * ceil_div(s->N, 16 * f.nf);
    if (workgroups * f.parts >= (1l << 32) / threads) return FC_ERR_UNSUPPORTED;
    plan->shape = *s;
    plan->tile = f.tile;
    plan->parts = f.parts;
    plan->ws_bytes = f.parts > 1 ? (size_t)f.parts * s->M * s->N * sizeof(int) : 0;
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
    // a tile's offsets are 32 bits
    const bool direct = ((s.K | s.x_row | s.w_row) & 15) == 0 && (((uint64_t)x_dev | (uint64_t)w_dev) & 15) == 0 && (s.x_row | s.w_row) < (1l << 23);
    const fc_device_scope on(ctx);
    if (s.dtype == FC_F32) return run<FC_F32>(ctx, p, plan, direct, ws_dev);
    if (s.dtype == FC_BF16) return run<FC_BF16>(ctx, p, plan, direct, ws_dev);
    return run<FC_F16>(ctx, p, plan, direct, ws_dev);
}
