// Linear attention in chunks of 32 tokens on the matrix cores.
//
// With S the state that enters a chunk, local tokens i, j and l the decay (forward; a backward run differs by one power of l):
//   o_i = scale * ( l^(i+1) S^T q_i + sum over j <= i of l^(i-j) (q_i . k_j) v_j )
//   S  <- l^C S + sum over j of l^(C-1-j) k_j v_j^T
// Of S nothing leaves the registers between the first token of a segment and its last; q, k and v are read once by a sequence in one piece whose values have up to
// 128 channels (q and k once more for each 128 further ones), and in segments k and v a second time.  A wavefront owns 32 columns of S for all of its
// rows, as accumulators of 32x32 products.  What makes them fit together without a turn through LDS: lane l of an accumulator
// holds column l % 32, rows 8*(r/4) + 4*(l/32) + r%4; lane l of an operand holds row (or column) l % 32, depths 8*(l/32) + e.
// The order of a product's depths is free as long as both operands keep the same, so with depth 8*g + e of sixteen named
// 8*(e/4) + 4*g + e%4 eight accumulators are an operand as they are.  P^T = K Q^T feeds O^T = V P^T, S feeds O^T = S^T Q^T.
// All operands lie in LDS in that order, 16 bytes a lane, so that a wavefront reads 1 KB in a row.
//
// Roundings.  A matrix core multiplies bf16 (8 bits) and adds in fp32.  Inputs are split into as many bf16 parts as they have bits
// for: bf16 one, half two, fp32 three, exactly.  What is formed between two products, P and S, goes in as two parts for the 16-bit types
// (16 bits, against the 8 or 11 of the output, whose rounding hides it; a third would be 8 products more of 50) and as three for fp32; l^n k, which is summed into the state, as three (24 bits:
// states are fp32).  Products of parts below the last bits that are kept are left out: for fp32 six of nine are made, which errs by 2^-24 of a product at most, 0.1 of
// that on average.
//
// Bound by the time of a chunk in a wavefront, since a state waits for the chunk before: at D = 128 in bf16 47 products of 32 cycles and 560 other vector
// instructions (splits, decays, the diagonal of P) a wavefront and chunk, the matrix cores busy a fifth of the time, in two wavefronts a SIMD that overlap one
// another's; the registers of a state, 64 of 231 at D = 128, allow no third (three spill: 324 us of training below become 450 and more).  fp32 with more than
// 64 rows has one only: three parts of everything are 102 KB of LDS, one workgroup a compute unit, and 44 registers spill (104 by single elements).
// 32 tokens a chunk: with 64 P and its
// operands would not fit beside the state, and P's products grow with the chunk.  Every wavefront of a workgroup needs the whole P, so each forms
// a part of it for all.  Segments make up for what one wavefront waits: see the rule beside the plan.
// 12544 tokens of 16 heads of 128 in bf16: states 38 us, their scan 14, answers 72, 117 to 120 with the launches, of 33 that a copy of as many bytes takes.  8 x 1225 tokens of 8 heads
// of 64 in fp32: 16, 5 and 36, 56 together, of 13.  8 x 3136 tokens of 16 heads of 64 with the backward pass in bf16: 323 us, of 90, in three runs of states (25 to
// 30 each), three scans (9 to 10) and four runs of answers (53 to 61).
#pragma once

#include <atomic>

#include "linear_attention.h"

constexpr int kLaChunk = 32;
// A state is held divided by a scale from 2 to kLaTop (kLaMost where a decay above 1 lets it grow).  Never by less than 2: then neither it, nor what
// a chunk adds to it, nor the first part of either comes near the largest float before the state itself does.  Never by much more: the third part
// of small values would be lost.  A wider range saves passes over the state where a head forgets within a chunk or two, 1 % at most (a top of 2^17: 12544 tokens 118 us
// for 119, the training below 324 for 326), but with 2^17 fp32 operands of 1e-30 keep 18 bits, with 4 those of 1e-33.
constexpr double kLaTop = 4, kLaLeast = 2, kLaMost = 65536;
constexpr float kLaLargest = 0x1.fep127f;      // of bf16
constexpr int kLaLoadsDone = 0x0f70;    // s_waitcnt: no load or store of global memory on its way
constexpr int kLaOnlyVector = 0x6;      // scheduling: vector and scalar arithmetic may pass, memory and matrix instructions not

typedef __bf16 la_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 la_bf16x4 __attribute__((ext_vector_type(4)));
typedef float la_f32x16 __attribute__((ext_vector_type(16)));
typedef float la_f32x4 __attribute__((ext_vector_type(4)));
typedef float la_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 la_bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t la_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t la_u32x4 __attribute__((ext_vector_type(4)));

// Operands as bf16 parts.  PARTS: of the inputs; FORMED: of what is formed between two products; KEPT: of what enters the state.
// Products of parts that together come ORDER or more parts late are left out (of those into the state, KEPT).
typedef la_bf16x8 la_frag;      // sixteen depths of 32 rows
typedef la_bf16x4 la_quad;      // four depths of a row, of four
constexpr int kLaFrag = 1024;   // bytes
template <int DT>
struct la_math {
    static constexpr int PARTS = DT == FC_F32 ? 3 : DT == FC_F16 ? 2 : 1, FORMED = DT == FC_F32 ? 3 : 2, KEPT = 3, ORDER = FORMED;
};
__device__ __forceinline__ la_f32x16 la_product(const la_frag &a, const la_frag &b, la_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ la_f32x4 la_product16(const la_frag &a, const la_frag &b, la_f32x4 c) {      // 16x16, 32 depths
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// PARTS bf16 parts of two values, each pair in one word: rounded, what that leaves rounded, and so on.  Bits that `keep` lacks are zeros in
// every part.  LARGE: values may lie so close to the largest float that they would round to infinity; then the first part is the largest bf16, and
// the others hold the rest, or an infinity or NaN itself.  (A value less its rounded self is one v_dot2_f32_bf16 on the pair as it is packed, too, a - 1 * hi.lo + 0 * hi.hi; with
// it the whole kernel takes 1.13 times as long.)
template <int PARTS, bool LARGE>
__device__ __forceinline__ void la_split_pair(float a, float b, uint32_t (&out)[PARTS], uint32_t keep = ~0u) {
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
        la_f32x2 x = {a, b};
        if (LARGE && p == 0) x = (la_f32x2){__builtin_amdgcn_fmed3f(a, -kLaLargest, kLaLargest), __builtin_amdgcn_fmed3f(b, -kLaLargest, kLaLargest)};
        out[p] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, la_bf16x2)) & keep;
        if (p + 1 < PARTS) {
            a -= __builtin_bit_cast(float, out[p] << 16);
            b -= __builtin_bit_cast(float, out[p] & 0xffff0000u);
        }
    }
}
// of four
template <int PARTS, bool LARGE>
__device__ __forceinline__ void la_split(const float (&x)[4], la_bf16x4 (&out)[PARTS]) {
    uint32_t lo[PARTS], hi[PARTS];
    la_split_pair<PARTS, LARGE>(x[0], x[1], lo);
    la_split_pair<PARTS, LARGE>(x[2], x[3], hi);
#pragma unroll
    for (int p = 0; p < PARTS; p++) out[p] = __builtin_bit_cast(la_bf16x4, (la_u32x2){lo[p], hi[p]});
}

// Byte offset of quad u of a row in a fragment.  The row's place is mixed with `mix` so that threads that write at once meet different banks;
// a wavefront that reads a fragment reads all of its places whatever the mix.
__device__ __forceinline__ int la_place(int row, int u, int mix) { return ((u & 1) * 32 + (row ^ mix)) * 16 + (u >> 1) * 8; }

// natural: row = token, sixteen channels a fragment.  turned: row = channel of 32, sixteen tokens a fragment.
__device__ __forceinline__ int la_natural(int token, int quad) {      // quad: channel / 4
    const int s = quad >> 2, u = quad & 3;
    return s * kLaFrag + la_place(token, u, (2 * s + (u & 1)) & 15);
}
__device__ __forceinline__ int la_turned(int channel, int quad) {     // quad: token / 4
    const int td = channel >> 5, row = channel & 31;
    return (td * 2 + (quad >> 2)) * kLaFrag + la_place(row, quad & 3, (td & 1) | (row >> 4) << 1);
}
__device__ __forceinline__ la_frag la_read(const char *frag, int lane, int mix) {
    return *(const la_frag *)(frag + ((lane & 32) + ((lane & 31) ^ mix)) * 16);
}
__device__ __forceinline__ la_frag la_read_natural(const char *base, int s, int lane) {
    return la_read(base + s * kLaFrag, lane, (2 * s + (lane >> 5)) & 15);
}
// Thirty-two depths, from two fragments, of sixteen tokens: an operand of a 16x16 product.
__device__ __forceinline__ la_frag la_read_natural16(const char *base, int s, int first, int lane) {
    const int f = 2 * s + (lane >> 5), g = lane >> 4 & 1;
    return *(const la_frag *)(base + f * kLaFrag + (g * 32 + ((first + (lane & 15)) ^ ((2 * f + g) & 15))) * 16);
}
__device__ __forceinline__ la_frag la_read_turned(const char *base, int td, int s, int lane) {
    return la_read(base + (td * 2 + s) * kLaFrag, lane, (td & 1) | (lane >> 4 & 1) << 1);
}

// Which four of a chunk's tokens and which four of D channels a thread has: sixteen threads side by side read 128 bytes of a token's channels,
// the sixteen after them those of the token eight further on, which together meet every bank of LDS once when they write.
// Threads past the last of a narrow operand have tokens past the chunk.
template <int D>
__device__ __forceinline__ int la_tokens_of(int item) {
    if (D < 64 || item >= 2 * D) return item / (D / 4);
    const int t = item >> 4 & 7;
    return (t & 1) << 1 | (t >> 1 & 1) | (t & 4);
}
template <int D>
__device__ __forceinline__ int la_channels_of(int item) {
    return D < 64 ? item % (D / 4) : (item & 15) | item >> 7 << 4;
}

// Four tokens times four channels of an operand, on their way from global memory to LDS.
template <int DT>
struct la_block {
    fc_vec<DT, 4> row[4];
};

// Where a thread finds its four tokens of four channels in each chunk.
// WIDE: four channels lie within one access.  Then a chunk is read through a buffer resource that begins at its first byte in memory (its
// last token in a backward run); a lane whose token or channels do not exist reads past its end, which gives zeros.
template <int DT, bool WIDE>
struct la_source {
    typedef typename fc_elem<DT>::type E;
    static constexpr uint32_t NOWHERE = 0x80000000u;
    const E *at;             // the first token of the four: of this thread, or if WIDE of the chunk, at its lowest address
    long next;               // elements to the next token
    uint32_t offset;
    int token, channels;     // of the four in the chunk; that are there from the thread's first on

    __device__ __forceinline__ void begin(const fc_la_operand &x, const fc_la_run &r, long b, int h, long first, int tq, int channel, int D) {
        next = r.reverse ? -x.token : x.token;
        token = 4 * tq;
        channels = D - channel;
        const E *head = (const E *)x.p + b * x.batch + (h / x.share) * x.head + first * x.token;
        if (WIDE) {
            at = head + (r.reverse ? (kLaChunk - 1) * next : 0);
            offset = channels > 0 && token < kLaChunk ? (uint32_t)((r.reverse ? kLaChunk - 4 - token : token) * x.token + channel) * (uint32_t)sizeof(E) : NOWHERE;
        } else {
            at = head + token * next + channel;
            offset = 0;
        }
    }
    // of a chunk of n tokens; moves on to the next one
    __device__ __forceinline__ void load(la_block<DT> &b, int n) {
        if (WIDE) {
            const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(const_cast<E *>(uniform_ptr(at)), 0, 0x7fffffff, 0x00020000);
            const int step = __builtin_amdgcn_readfirstlane((int)(next * (long)sizeof(E))), lowest = step < 0 ? -3 * step : 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t there = n == kLaChunk || token + i < n ? offset : NOWHERE;
                const int row = __builtin_amdgcn_readfirstlane(lowest + i * step);
                if constexpr (DT == FC_F32) b.row[i] = __builtin_bit_cast(row_type, __builtin_amdgcn_raw_buffer_load_b128(res, there, row, 0));
                else b.row[i] = __builtin_bit_cast(row_type, __builtin_amdgcn_raw_buffer_load_b64(res, there, row, 0));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) b.row[i].v[e] = token + i < n && e < channels ? at[i * next + e] : (E)0.f;
        }
        at += kLaChunk * next;
    }
    typedef fc_vec<DT, 4> row_type;
};

template <int PARTS, bool LARGE>
__device__ __forceinline__ void la_put(char *base, int plane, int at, const float (&x)[4]) {
    la_quad q[PARTS];
    la_split<PARTS, LARGE>(x, q);
#pragma unroll
    for (int p = 0; p < PARTS; p++) *(la_quad *)(base + p * plane + at) = q[p];
}
// Four inputs: bf16 as they lie in memory, others split.
template <int DT>
__device__ __forceinline__ void la_put_raw(char *base, int plane, int at, typename fc_elem<DT>::type a, typename fc_elem<DT>::type b,
                                           typename fc_elem<DT>::type c, typename fc_elem<DT>::type d) {
    if constexpr (DT == FC_BF16) *(la_quad *)(base + at) = (la_quad){a, b, c, d};
    else la_put<la_math<DT>::PARTS, DT == FC_F32>(base, plane, at, {(float)a, (float)b, (float)c, (float)d});
}

// Eight accumulators of a state from `first` on as an operand: held at half the state or less.
template <int FORMED>
__device__ __forceinline__ void la_formed(const la_f32x16 &x, int first, la_frag (&f)[FORMED]) {
    la_u32x4 w[FORMED];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t two[FORMED];
        la_split_pair<FORMED, false>(x[first + 2 * i], x[first + 2 * i + 1], two);
#pragma unroll
        for (int p = 0; p < FORMED; p++) w[p][i] = two[p];
    }
#pragma unroll
    for (int p = 0; p < FORMED; p++) f[p] = __builtin_bit_cast(la_frag, w[p]);
}

// Not 0 if any element of a block is an infinity or NaN: all exponent bits set, which one more in the last of them carries over.
template <int DT>
__device__ __forceinline__ uint32_t la_not_finite(const la_block<DT> &b) {
    constexpr uint32_t exponent = DT == FC_F32 ? 0x7f800000u : DT == FC_BF16 ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t last = DT == FC_F32 ? 0x00800000u : DT == FC_BF16 ? 0x00800080u : 0x04000400u;
    constexpr uint32_t carry = DT == FC_F32 ? 0x80000000u : 0x80008000u;
    constexpr int WORDS = sizeof(la_block<DT>) / 4;
    struct words {
        uint32_t w[WORDS];
    };
    const words x = __builtin_bit_cast(words, b);
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < WORDS; i++) bad |= (x.w[i] & exponent) + last;
    return bad & carry;
}

template <int DT>
__device__ __forceinline__ void la_answer(const fc_la_run &r, long at, float x) {
    if (r.o_fp32) ((float *)r.o)[at] = x;
    else ((typename fc_elem<DT>::type *)r.o)[at] = (typename fc_elem<DT>::type)x;
}

// Tokens of the chunk that begins at p0.
__device__ __forceinline__ int la_tokens(long p0, long end) { return (int)(end - p0 < kLaChunk ? end - p0 : kLaChunk); }

// KT tiles of 32 rows of the state (rows past Dk are zeros), NW wavefronts of 32 columns.  FULL: answers tokens; otherwise only
// forms the state that a segment adds.
template <int DT, int KT, int NW, bool FULL, bool WIDE>
__global__ __launch_bounds__(64 * NW, 2) void fc_linear_attention_chunk_kernel(const fc_la_run r, int segments, long segment, int slices, float *parts) {
    typedef la_math<DT> M;
    typedef typename fc_elem<DT>::type E;
    constexpr int THREADS = 64 * NW, DK = 32 * KT, DV = 32 * NW;
    constexpr int QK_PLANE = 2 * KT * kLaFrag, V_PLANE = 2 * NW * kLaFrag;
    constexpr int Q_BYTES = FULL ? M::PARTS * QK_PLANE : 0;
    constexpr int QK_ITEMS = (8 * DK / 4 + THREADS - 1) / THREADS, V_ITEMS = 8 * DV / 4 / THREADS;
    extern __shared__ char lds[];
    char *const qs = lds, *const ks = qs + Q_BYTES, *const kt = ks + Q_BYTES, *const vt = kt + M::KEPT * QK_PLANE;
    char *const pt = vt + M::PARTS * V_PLANE;                       // P, rows of 32 answers, if FULL
    double *const exact = (double *)(FULL ? pt + M::FORMED * 2 * kLaFrag : pt + M::KEPT * QK_PLANE + M::PARTS * V_PLANE);      // decay^0 .. decay^32
    float *const power = (float *)(exact + kLaChunk + 1);           // the same, times what enters the state
    int *const odd = (int *)(power + kLaChunk + 1);                 // whether a value of the chunk is not finite,
    int *const since = odd + 1;                                     // and from which token on, for each column

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5;
    unsigned block = blockIdx.x;
    const int slice = block % slices;
    block /= slices;
    const int running = FULL ? segments : segments - 1;      // what the last one adds is asked for by none
    const int seg = block % running;
    const long bh = block / running, b = bh / r.H;
    const int h = (int)(bh - b * r.H);
    const int col0 = slice * DV, col = col0 + 32 * wave + (lane & 31);
    const long len = fc_la_length(r, b);
    const long begin = seg * segment, end = begin + segment < len ? begin + segment : len;
    if (!FULL && begin >= end) return;
    const float ld = r.log_decay[h];
    // this thread's tokens and channels of every operand, a chunk at a time
    const long first = r.reverse ? len - 1 - begin : begin;
    la_source<DT, WIDE> q_from[FULL ? QK_ITEMS : 1], k_from[QK_ITEMS], v_from[V_ITEMS];
    la_block<DT> q_in[FULL ? QK_ITEMS : 1], k_in[QK_ITEMS], k_now[QK_ITEMS], v_in[V_ITEMS];
#pragma unroll
    for (int it = 0; it < QK_ITEMS; it++) {
        const int tq = la_tokens_of<DK>(tid + it * THREADS), cq = la_channels_of<DK>(tid + it * THREADS);
        if (FULL) q_from[it].begin(r.q, r, b, h, first, tq, 4 * cq, r.Dk);
        k_from[it].begin(r.k, r, b, h, first, tq, 4 * cq, r.Dk);
    }
#pragma unroll
    for (int it = 0; it < V_ITEMS; it++) {
        const int tq = la_tokens_of<DV>(tid + it * THREADS), cq = la_channels_of<DV>(tid + it * THREADS);
        v_from[it].begin(r.v, r, b, h, first, tq, col0 + 4 * cq, r.Dv);
    }
    auto load_qk = [&](long p0) __attribute__((always_inline)) {
        const int n = la_tokens(p0, end);
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++) {
            if (FULL) q_from[it].load(q_in[it], n);
            k_from[it].load(k_in[it], n);
        }
    };
    auto load_v = [&](long p0) __attribute__((always_inline)) {
        const int n = la_tokens(p0, end);
#pragma unroll
        for (int it = 0; it < V_ITEMS; it++) v_from[it].load(v_in[it], n);
    };
    load_qk(begin);
    load_v(begin);
    // the state: rows 32*t + 8*(e/4) + 4*g + e%4 of column col, zeros in place of what it does not have
    la_f32x16 S[KT];
    const float *from_state = segments > 1 ? parts + (bh * segments + seg) * (long)r.Dk * r.Dv : r.state_in ? r.state_in + bh * r.state_head : nullptr;
    {
        const float held = begin < end ? (float)(1.0 / kLaTop) : 1.f;
        const uint32_t srow = (uint32_t)(segments > 1 ? r.part_row : r.state_row), scol = (uint32_t)(segments > 1 ? r.part_col : r.state_col);
        const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(uniform_ptr(from_state)), 0, from_state ? 0x7fffffff : 0, 0x00020000);
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int row = 32 * t + 8 * (e / 4) + 4 * g + e % 4;
                S[t][e] = 0.f;
                if (FULL) S[t][e] = held * __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(res, row < r.Dk && col < r.Dv ? 4 * (row * srow + col * scol) : 0x80000000u, 0, 0));
            }
    }
    if (FULL)
        for (int i = tid; i < M::FORMED * 2 * kLaFrag / 4; i += THREADS) ((uint32_t *)pt)[i] = 0;

    if (tid <= kLaChunk) {
        const double l = tid ? exp((double)ld * tid) : 1.0;
        exact[tid] = l;
        power[tid] = (float)l * r.scale_in;
    }
    if (FULL) {
        if (tid == 0) *odd = 0;
        for (int c = tid; c < DV; c += THREADS) since[c] = kLaChunk;
    }
    __syncthreads();
    // P^T in blocks of 16x16, the one above the diagonal left as zeros: this wavefront's, with the powers between their tokens.  A later
    // token is left out of P by its bits, not multiplied by zero: it may hold anything.
    constexpr int BLOCKS = FULL ? (3 + NW - 1) / NW : 1;
    float near[BLOCKS][4], from = 0.f;
    uint32_t earlier[BLOCKS][2];
    const int i_tok = lane & 31;
    if (FULL) {
#pragma unroll
        for (int n = 0; n < BLOCKS; n++) {
            const int t = wave + n * NW, j0 = t == 2 ? 16 : 0, i0 = t >= 1 ? 16 : 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = i0 + (lane & 15) - (j0 + 4 * (lane >> 4) + e);
                near[n][e] = d < 0 ? 0.f : power[d] * r.scale_out;
                if (e % 2 == 0) earlier[n][e / 2] = (d >= 0 ? 0x0000ffffu : 0u) | (d >= 1 ? 0xffff0000u : 0u);
            }
        }
        from = (float)exact[i_tok + 1 - r.reverse] * r.scale_out;
    }
    // The state is scale * S: what decays is the scale, one number, and what a chunk adds is divided by it, until it is small
    // enough to be worth a pass over S.  Where no token comes it passes as it is.
    double scale = begin < end ? kLaTop : 1.0;

    // token i of four of q and k
    auto put_natural = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++) {
            const int tq = la_tokens_of<DK>(tid + it * THREADS), cq = la_channels_of<DK>(tid + it * THREADS);
            if (8 * DK / 4 < THREADS && tq >= 8) continue;
            const int at = la_natural(4 * tq + i, cq);
            la_put_raw<DT>(qs, QK_PLANE, at, q_in[it].row[i].v[0], q_in[it].row[i].v[1], q_in[it].row[i].v[2], q_in[it].row[i].v[3]);
            la_put_raw<DT>(ks, QK_PLANE, at, k_in[it].row[i].v[0], k_in[it].row[i].v[1], k_in[it].row[i].v[2], k_in[it].row[i].v[3]);
        }
    };
    // channel e of four of what k adds to the state; w: what its four tokens are worth at the end of the chunk
    float w[QK_ITEMS][4];
    auto weigh = [&](int n, float add) __attribute__((always_inline)) {
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = n - 1 - 4 * la_tokens_of<DK>(tid + it * THREADS) - i + r.reverse;
                w[it][i] = power[d < 0 ? 0 : d > kLaChunk ? kLaChunk : d] * add;      // tokens past n are zeros
            }
    };
    auto put_weighed = [&](char *to, int e) __attribute__((always_inline)) {
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++) {
            const int tq = la_tokens_of<DK>(tid + it * THREADS), cq = la_channels_of<DK>(tid + it * THREADS);
            if (8 * DK / 4 < THREADS && tq >= 8) continue;
            la_put<M::KEPT, false>(to, QK_PLANE, la_turned(4 * cq + e, tq),
                                {k_now[it].row[0].get(e) * w[it][0], k_now[it].row[1].get(e) * w[it][1], k_now[it].row[2].get(e) * w[it][2],
                                 k_now[it].row[3].get(e) * w[it][3]});
        }
    };
    // A value that is not finite would meet the zeros of the tokens before it.  It is taken out here; its column is NaN from its token on.
    auto finite_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int it = 0; it < V_ITEMS; it++) {
            if (!la_not_finite<DT>(v_in[it])) continue;
            const int tq = la_tokens_of<DV>(tid + it * THREADS), cq = la_channels_of<DV>(tid + it * THREADS);
            *odd = 1;
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = v_in[it].row[i].get(e);
                    if (x - x == 0.f) continue;
                    atomicMin(&since[4 * cq + e], 4 * tq + i);
                    v_in[it].row[i].v[e] = (E)0.f;
                }
        }
    };
    // channel e of four of v
    auto put_v = [&](char *to, int e) __attribute__((always_inline)) {
#pragma unroll
        for (int it = 0; it < V_ITEMS; it++) {
            const int tq = la_tokens_of<DV>(tid + it * THREADS), cq = la_channels_of<DV>(tid + it * THREADS);
            la_put_raw<DT>(to, V_PLANE, la_turned(4 * cq + e, tq), v_in[it].row[0].v[e], v_in[it].row[1].v[e],
                                     v_in[it].row[2].v[e], v_in[it].row[3].v[e]);
        }
    };
    la_frag vf[2][M::PARTS];
    auto read_v = [&](const char *from) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int p = 0; p < M::PARTS; p++) vf[s][p] = la_read_turned(from + p * V_PLANE, wave, s, lane);
    };
    // The state takes a chunk in; what(i) goes on meanwhile, in 2 * KT steps.
    auto take_in = [&](const char *from, auto &&what) __attribute__((always_inline)) {
        la_frag kf[2][M::KEPT];
        auto fetch = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int a = 0; a < M::KEPT; a++) kf[i & 1][a] = la_read_turned(from + a * QK_PLANE, i / 2, i % 2, lane);
        };
        fetch(0);
#pragma unroll
        for (int i = 0; i < 2 * KT; i++) {
            if (i + 1 < 2 * KT) fetch(i + 1);
            __builtin_amdgcn_sched_barrier(kLaOnlyVector);      // reads ahead of the products that do not need them
#pragma unroll
            for (int a = 0; a < M::KEPT; a++)
#pragma unroll
                for (int c = 0; c < M::PARTS; c++)
                    if (a + c < M::KEPT) S[i / 2] = la_product(kf[i & 1][a], vf[i % 2][c], S[i / 2]);
            what(i);
            __builtin_amdgcn_sched_barrier(kLaOnlyVector);
        }
    };
    // What a chunk of n tokens does to the scale.
    double decayed = 1.0;
    bool settle = false;
    float add = 1.f, from_now = 0.f;
    auto rescale = [&](int n) __attribute__((always_inline)) {
        from_now = from * (float)scale;
        decayed = scale * exact[n];
        settle = decayed < kLaLeast || decayed > kLaMost;
        scale = settle ? kLaTop : decayed;
        add = (float)(1.0 / scale);
    };
    auto settle_state = [&]() __attribute__((always_inline)) {
        if (settle) {
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) S[t][e] *= (float)(decayed * (1.0 / kLaTop));
        }
    };

    if constexpr (!FULL) {
        // One barrier a chunk: while the state takes in one, the next is laid out in the other half of LDS.
        constexpr int HALF = M::KEPT * QK_PLANE + M::PARTS * V_PLANE;
        char *const halves = kt;
        int n = la_tokens(begin, end);
        rescale(n);
        weigh(n, add);
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++) k_now[it] = k_in[it];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            put_weighed(halves, e);
            put_v(halves + M::KEPT * QK_PLANE, e);
        }
        load_qk(begin + kLaChunk);
        load_v(begin + kLaChunk);
        bool settle_now = settle;
        double decayed_now = decayed;
        int half = 0;
#pragma unroll 1
        for (long p0 = begin; p0 < end; p0 += kLaChunk) {
            __syncthreads();
            const char *const now = halves + half * HALF;
            half ^= 1;
            char *const next = halves + half * HALF;
            read_v(now + M::KEPT * QK_PLANE);
            // the scale of this chunk, and then that of the next one
            settle = settle_now;
            decayed = decayed_now;
            settle_state();
            n = la_tokens(p0 + kLaChunk, end);
            if (n > 0) {
                rescale(n);
                settle_now = settle;
                decayed_now = decayed;
                weigh(n, add);
#pragma unroll
                for (int it = 0; it < QK_ITEMS; it++) k_now[it] = k_in[it];
            }
            take_in(now, [&](int i) __attribute__((always_inline)) {
                if (n > 0) {
#pragma unroll
                    for (int e = i * 4 / (2 * KT); e < (i + 1) * 4 / (2 * KT); e++) {
                        put_weighed(next, e);
                        put_v(next + M::KEPT * QK_PLANE, e);
                    }
                }
            });
            load_qk(p0 + 2 * kLaChunk);
            load_v(p0 + 2 * kLaChunk);
        }
    } else {
        // Two barriers a chunk.  Between the first and the second q and k are read, and what k adds and v are laid out for
        // the state; after the second these are read, and the next chunk's q and k laid out.  So either half has work for the vector unit
        // beside the matrix cores'.
        const long o_size = r.o_fp32 ? 4 : (long)sizeof(E), o_row = r.o_token * o_size;
        const long o_step = r.reverse ? -kLaChunk * o_row : kLaChunk * o_row;
        const uint32_t o_offset = (uint32_t)((r.reverse ? kLaChunk - 1 - i_tok : i_tok) * o_row + 32 * wave * o_size);
        char *o_at = (char *)r.o + (b * r.o_batch + h * r.o_head + col0) * o_size + (r.reverse ? first - (kLaChunk - 1) : first) * o_row;
#pragma unroll
        for (int i = 0; i < 4; i++) put_natural(i);
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++) k_now[it] = k_in[it];
        load_qk(begin + kLaChunk);
        __builtin_amdgcn_s_waitcnt(kLaLoadsDone);
#pragma unroll 1
        for (long p0 = begin; p0 < end; p0 += kLaChunk) {
            const int n = la_tokens(p0, end);
            rescale(n);
            weigh(n, add);
            __syncthreads();
            la_f32x16 O;
            la_f32x4 P[BLOCKS];
#pragma unroll
            for (int e = 0; e < 16; e++) O[e] = 0.f;
#pragma unroll
            for (int n = 0; n < BLOCKS; n++) P[n] = (la_f32x4){0.f, 0.f, 0.f, 0.f};
            {
                la_frag qf[2][M::PARTS], sf[M::FORMED], qp[BLOCKS][M::PARTS], kp[BLOCKS][M::PARTS];
                auto fetch = [&](int s) __attribute__((always_inline)) {
#pragma unroll
                    for (int p = 0; p < M::PARTS; p++) qf[s & 1][p] = la_read_natural(qs + p * QK_PLANE, s, lane);
                };
                finite_v();
                fetch(0);
#pragma unroll
                for (int s = 0; s < 2 * KT; s++) {
                    if (s + 1 < 2 * KT) fetch(s + 1);
                    if (s % 2 == 0) {
#pragma unroll
                        for (int n = 0; n < BLOCKS; n++) {
                            const int t = wave + n * NW;
                            if (t >= 3) continue;
#pragma unroll
                            for (int p = 0; p < M::PARTS; p++) {
                                qp[n][p] = la_read_natural16(qs + p * QK_PLANE, s / 2, t >= 1 ? 16 : 0, lane);
                                kp[n][p] = la_read_natural16(ks + p * QK_PLANE, s / 2, t == 2 ? 16 : 0, lane);
                            }
                        }
                    }
                    __builtin_amdgcn_sched_barrier(kLaOnlyVector);
                    la_formed<M::FORMED>(S[s / 2], 8 * (s % 2), sf);
#pragma unroll
                    for (int a = 0; a < M::FORMED; a++)
#pragma unroll
                        for (int c = 0; c < M::PARTS; c++)
                            if (a + c < M::ORDER) O = la_product(sf[a], qf[s & 1][c], O);
                    if (s % 2 == 1) {      // read a step ago
#pragma unroll
                        for (int n = 0; n < BLOCKS; n++) {
                            if (wave + n * NW >= 3) continue;
#pragma unroll
                            for (int a = 0; a < M::PARTS; a++)
#pragma unroll
                                for (int c = 0; c < M::PARTS; c++)
                                    if (a + c < M::ORDER) P[n] = la_product16(kp[n][a], qp[n][c], P[n]);
                        }
                    }
#pragma unroll
                    for (int e = s * 4 / (2 * KT); e < (s + 1) * 4 / (2 * KT); e++) {
                        put_weighed(kt, e);
                        put_v(vt, e);
                    }
                    __builtin_amdgcn_sched_barrier(kLaOnlyVector);
                }
            }
#pragma unroll
            for (int n = 0; n < BLOCKS; n++) {
                const int t = wave + n * NW;
                if (t >= 3) continue;
                uint32_t lo[M::FORMED], hi[M::FORMED];
                la_split_pair<M::FORMED, true>(P[n][0] * near[n][0], P[n][1] * near[n][1], lo, earlier[n][0]);
                la_split_pair<M::FORMED, true>(P[n][2] * near[n][2], P[n][3] * near[n][3], hi, earlier[n][1]);
                char *const to = pt + (t == 2 ? kLaFrag : 0) + la_place((t >= 1 ? 16 : 0) + (lane & 15), lane >> 4, 0);
#pragma unroll
                for (int p = 0; p < M::FORMED; p++) *(la_u32x2 *)(to + p * 2 * kLaFrag) = (la_u32x2){lo[p], hi[p]};
            }
            load_v(p0 + kLaChunk);      // nothing past the last chunk
            __syncthreads();
            read_v(vt);
            la_frag pf[2][M::FORMED];
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int p = 0; p < M::FORMED; p++) pf[s][p] = la_read(pt + (2 * p + s) * kLaFrag, lane, 0);
            const bool any_odd = *odd;
            settle_state();
            take_in(kt, [&](int i) __attribute__((always_inline)) {
#pragma unroll
                for (int e = i * 4 / (2 * KT); e < (i + 1) * 4 / (2 * KT); e++) put_natural(e);
            });
#pragma unroll
            for (int it = 0; it < QK_ITEMS; it++) k_now[it] = k_in[it];
            load_qk(p0 + 2 * kLaChunk);
#pragma unroll
            for (int e = 0; e < 16; e++) O[e] *= from_now;
#pragma unroll
            for (int s = 0; s < 2; s++) {
#pragma unroll
                for (int a = 0; a < M::PARTS; a++)
#pragma unroll
                    for (int c = 0; c < M::FORMED; c++)
                        if (a + c < M::ORDER) O = la_product(vf[s][a], pf[s][c], O);
            }
            if (any_odd) {
                const bool lost = since[32 * wave + i_tok] < kLaChunk;
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) S[t][e] = lost ? __builtin_nanf("") : S[t][e];
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (i_tok >= since[32 * wave + 8 * (e / 4) + 4 * g + e % 4]) O[e] = __builtin_nanf("");
                __syncthreads();
                if (tid == 0) *odd = 0;
                for (int c = tid; c < DV; c += THREADS) since[c] = kLaChunk;
            }
            // lane: token i_tok, columns 8*(e/4) + 4*g + e%4 of the wavefront's 32
            if (WIDE) {
                const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(o_at), 0, 0x7fffffff, 0x00020000);
                const int c = col0 + 32 * wave;
                const uint32_t nowhere = la_source<DT, true>::NOWHERE;
                if (DT == FC_F32 || r.o_fp32) {
#pragma unroll
                    for (int a = 0; a < 4; a++)
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(la_u32x4, (la_f32x4){O[4 * a], O[4 * a + 1], O[4 * a + 2], O[4 * a + 3]}),
                                                               res, i_tok < n && c + 8 * a + 4 * g < r.Dv ? o_offset + 16 * g : nowhere, 32 * a, 0);
                } else if constexpr (DT != FC_F32) {
                    // 16 bytes of a token a lane: the lower half of the wavefront takes columns 0 and 8 on from both, the upper
                    // half 16 and 24 on
                    la_u32x2 x[4];
#pragma unroll
                    for (int a = 0; a < 4; a++) {
                        fc_vec<DT, 4> y;
#pragma unroll
                        for (int e = 0; e < 4; e++) y.set(e, O[4 * a + e]);
                        x[a] = __builtin_bit_cast(la_u32x2, y);
                    }
#pragma unroll
                    for (int a = 0; a < 2; a++) {
                        const auto first = __builtin_amdgcn_permlane32_swap(x[a][0], x[a + 2][0], false, false);
                        const auto second = __builtin_amdgcn_permlane32_swap(x[a][1], x[a + 2][1], false, false);
                        const int from = c + 8 * a + 16 * g;
                        const uint32_t there = i_tok < n && from < r.Dv ? o_offset + 32 * g : nowhere;
                        if (r.Dv % 8 == 0)
                            __builtin_amdgcn_raw_buffer_store_b128((la_u32x4){first[0], second[0], first[1], second[1]}, res, there, 16 * a, 0);
                        else {      // four columns at the end
                            __builtin_amdgcn_raw_buffer_store_b64((la_u32x2){first[0], second[0]}, res, there, 16 * a, 0);
                            __builtin_amdgcn_raw_buffer_store_b64((la_u32x2){first[1], second[1]}, res, from + 4 < r.Dv ? there : nowhere, 16 * a + 8, 0);
                        }
                    }
                }
                o_at += o_step;
            } else if (i_tok < n) {
                const long t = r.reverse ? len - 1 - p0 - i_tok : p0 + i_tok;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int c = col0 + 32 * wave + 8 * (e / 4) + 4 * g + e % 4;
                    if (c >= r.Dv) continue;
                    la_answer<DT>(r, b * r.o_batch + t * r.o_token + h * r.o_head + c, O[e]);
                }
            }
        }
    }

    float *to_state = FULL ? (seg == segments - 1 && r.state_out ? r.state_out + bh * r.state_head : nullptr)
                           : parts + (bh * segments + seg) * (long)r.Dk * r.Dv;
    if (to_state) {
        const long orow = FULL ? r.state_row : r.Dv, ocol = FULL ? r.state_col : 1;
        int g_out = g;
        asm("" : "+v"(g_out));      // or the conditions of the load above would be kept through the loop, more than the scalar registers hold
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int row = 32 * t + 8 * (e / 4) + 4 * g_out + e % 4;
                if (row < r.Dk && col < r.Dv) to_state[row * orow + col * ocol] = S[t][e] * (float)scale;
            }
    }
    if (!FULL) return;
    // tokens past the end of a shorter sequence
    const long zero0 = begin > len ? begin : len, zero1 = begin + segment < r.T ? begin + segment : r.T;
    for (long t = zero0 + (tid >> 5); t < zero1; t += THREADS / 32) {
#pragma unroll
        for (int a = 0; a < NW; a++) {
            const int c = col0 + 32 * a + (tid & 31);
            if (c >= r.Dv) continue;
            la_answer<DT>(r, b * r.o_batch + t * r.o_token + h * r.o_head + c, 0.f);
        }
    }
}

template <int DT, int KT, int NW>
constexpr size_t la_lds_bytes(bool full) {
    typedef la_math<DT> M;
    const size_t qk = (size_t)2 * KT * kLaFrag, v = (size_t)2 * NW * kLaFrag;
    return (full ? 2 * M::PARTS * qk + M::FORMED * 2 * kLaFrag : M::KEPT * qk + M::PARTS * v) + M::KEPT * qk + M::PARTS * v + (kLaChunk + 1) * (sizeof(double) + sizeof(float)) + (1 + 32 * NW) * sizeof(int);
}

// More LDS than 64 KB has to be asked for, once for each kernel and device.
template <int DT, int KT, int NW, bool FULL, bool WIDE>
int la_launch_as(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    static std::atomic<uint64_t> granted{0};
    const size_t lds = la_lds_bytes<DT, KT, NW>(FULL);
    const auto kernel = fc_linear_attention_chunk_kernel<DT, KT, NW, FULL, WIDE>;
    const uint64_t bit = ctx->device < 64 ? 1ull << ctx->device : 0;
    if (lds > 65536 && !(granted.load() & bit)) {
        FC_HIP_CHECK(ctx, hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        granted.fetch_or(bit);
    }
    const int slices = (r.Dv + 32 * NW - 1) / (32 * NW);
    const unsigned blocks = (unsigned)(heads * (FULL ? segments : segments - 1) * slices);
    kernel<<<dim3(blocks), dim3(64 * NW), lds, ctx->stream>>>(r, segments, segment, slices, parts);
    FC_LAUNCH_CHECK(ctx, "fc_linear_attention_chunk_kernel");
    return FC_OK;
}

template <int DT, int KT, int NW, bool FULL>
int la_launch_one(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    return r.wide ? la_launch_as<DT, KT, NW, FULL, true>(ctx, r, heads, segments, segment, parts)
                  : la_launch_as<DT, KT, NW, FULL, false>(ctx, r, heads, segments, segment, parts);
}

template <int DT, bool FULL>
int la_launch(fc_context *ctx, const fc_la_run &r, long heads, int segments, long segment, float *parts) {
    if (fc_la_wavefronts(DT, r.Dk, r.Dv, r.wide) == 2) {
        if (r.Dk <= 32) return la_launch_one<DT, 1, 2, FULL>(ctx, r, heads, segments, segment, parts);
        if constexpr (DT == FC_F16) return la_launch_as<DT, 2, 2, FULL, true>(ctx, r, heads, segments, segment, parts);
        if constexpr (DT == FC_BF16) return la_launch_one<DT, 2, 2, FULL>(ctx, r, heads, segments, segment, parts);
    }
    if (r.Dk <= 32) return la_launch_one<DT, 1, 4, FULL>(ctx, r, heads, segments, segment, parts);
    if (r.Dk <= 64) return la_launch_one<DT, 2, 4, FULL>(ctx, r, heads, segments, segment, parts);
    return la_launch_one<DT, 4, 4, FULL>(ctx, r, heads, segments, segment, parts);
}
