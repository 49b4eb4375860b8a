// Linear attention in chunks of 32 tokens on the matrix cores.
//
// With S the state that enters a chunk, local tokens i, j and l the decay (forward; a backward run differs by one power of l):
//   o_i = scale * ( l^(i+1) S^T q_i + sum over j <= i of l^(i-j) (q_i . k_j) v_j )
//   S  <- l^C S + sum over j of l^(C-1-j) k_j v_j^T
// One pass: every q, k, v is read once, and of S nothing leaves the registers.  A wavefront owns 32 columns of S for all of its
// rows, as accumulators of 32x32 products.  What makes them fit together without a turn through LDS: lane l of an accumulator
// holds column l % 32, rows 8*(r/4) + 4*(l/32) + r%4; lane l of an operand holds row (or column) l % 32, depths 8*(l/32) + e.
// The order of a product's depths is free as long as both operands keep the same, so with depth 8*g + e of sixteen named
// 8*(e/4) + 4*g + e%4 eight accumulators are an operand as they are.  P^T = K Q^T feeds O^T = V P^T, S feeds O^T = S^T Q^T.
// All operands lie in LDS in that order, 16 bytes a lane, so that a wavefront reads 1 KB in a row.
//
// Roundings.  A matrix core multiplies bf16 (8 bits) and adds in fp32.  Inputs are split into as many bf16 parts as they have bits
// for: bf16 one, half two, exactly.  What is formed between two products, P and S, goes in as two parts (16 bits, against the 8 or
// 11 of the output); l^n k, which is summed into the state, as three (24 bits: states are fp32).  Parts whose product is below the last
// one kept are left out.  fp32 runs on fp32 matrix instructions, one part each.
#pragma once

#include <atomic>

#include "linear_attention.h"

constexpr int kLaChunk = 32;

typedef __bf16 la_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 la_bf16x4 __attribute__((ext_vector_type(4)));
typedef float la_f32x16 __attribute__((ext_vector_type(16)));
typedef float la_f32x4 __attribute__((ext_vector_type(4)));
typedef float la_f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t la_u32x4 __attribute__((ext_vector_type(4)));

// Sixteen depths of 32 rows, in LDS: UNITS 16-byte words a lane, and the products of two such operands.
template <int DT>
struct la_math {
    typedef __bf16 unit;
    typedef la_bf16x8 frag;
    typedef la_bf16x4 quad;      // four consecutive depths
    static constexpr int PARTS = DT == FC_F16 ? 2 : 1, FORMED = 2, KEPT = 3;
    static constexpr int FRAG_BYTES = 1024;
    static __device__ __forceinline__ la_f32x16 product(const frag &a, const frag &b, la_f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct la_math<FC_F32> {
    typedef float unit;
    struct frag {
        la_f32x4 half[2];
    };
    typedef la_f32x4 quad;
    static constexpr int PARTS = 1, FORMED = 1, KEPT = 1;
    static constexpr int FRAG_BYTES = 2048;
    static __device__ __forceinline__ la_f32x16 product(const frag &a, const frag &b, la_f32x16 c) {
#pragma unroll
        for (int e = 0; e < 8; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.half[e / 4][e % 4], b.half[e / 4][e % 4], c, 0, 0, 0);
        return c;
    }
};

// PARTS parts of four values
template <int PARTS>
__device__ __forceinline__ void la_split(const float (&x)[4], la_bf16x4 (&out)[PARTS]) {
    float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
        out[p] = __builtin_convertvector((la_f32x4){r[0], r[1], r[2], r[3]}, la_bf16x4);
        if (p + 1 < PARTS) {
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] -= (float)out[p][i];
        }
    }
}
template <int PARTS>
__device__ __forceinline__ void la_split(const float (&x)[4], la_f32x4 (&out)[PARTS]) {
    out[0] = (la_f32x4){x[0], x[1], x[2], x[3]};
}

// Byte offset of four consecutive depths (quad u of four in sixteen) of a row in a fragment.  The row's place is mixed with
// `mix` so that lanes that write the same row of many fragments, or every fourth row, meet different banks; a wavefront that
// reads a fragment reads all of its places whatever the mix.
template <int DT>
__device__ __forceinline__ int la_place(int row, int u, int mix) {
    const int g = u & 1, half = u >> 1, slot = g * 32 + (row ^ mix);
    return DT == FC_F32 ? half * 1024 + slot * 16 : slot * 16 + half * 8;
}

// Fragments of an operand: PARTS planes of `frags`.
// natural: row = token, sixteen channels a fragment.  turned: row = channel of 32, sixteen tokens a fragment.
template <int DT>
struct la_tile {
    static __device__ __forceinline__ int natural(int token, int quad) {      // quad: channel / 4
        const int s = quad >> 2, u = quad & 3;
        const int mix = DT == FC_F32 ? (4 * s + u) & 15 : (2 * s + (u & 1)) & 15;
        return s * la_math<DT>::FRAG_BYTES + la_place<DT>(token, u, mix);
    }
    static __device__ __forceinline__ int turned(int channel, int quad) {     // quad: token / 4
        const int td = channel >> 5;
        return (td * 2 + (quad >> 2)) * la_math<DT>::FRAG_BYTES + la_place<DT>(channel & 31, quad & 3, td & 3);
    }
    static __device__ __forceinline__ void read(const char *base, int lane, int mix0, int mix1, typename la_math<DT>::frag &f) {
        if constexpr (DT == FC_F32) {
            f.half[0] = *(const la_f32x4 *)(base + ((lane & 32) + ((lane & 31) ^ mix0)) * 16);
            f.half[1] = *(const la_f32x4 *)(base + 1024 + ((lane & 32) + ((lane & 31) ^ mix1)) * 16);
        } else {
            f = *(const la_bf16x8 *)(base + ((lane & 32) + ((lane & 31) ^ mix0)) * 16);
        }
    }
    static __device__ __forceinline__ void read_natural(const char *base, int s, int lane, typename la_math<DT>::frag &f) {
        const int g = lane >> 5;
        const int m0 = DT == FC_F32 ? (4 * s + g) & 15 : (2 * s + g) & 15, m1 = (4 * s + 2 + g) & 15;
        read(base + s * la_math<DT>::FRAG_BYTES, lane, m0, m1, f);
    }
    static __device__ __forceinline__ void read_turned(const char *base, int td, int s, int lane, typename la_math<DT>::frag &f) {
        read(base + (td * 2 + s) * la_math<DT>::FRAG_BYTES, lane, td & 3, td & 3, f);
    }
};

// Four tokens times four channels of an operand, on their way from global memory to LDS.
template <int DT>
struct la_block {
    fc_vec<DT, 4> row[4];
};

// The rows of `n` that are there of four, from `src` on, `next` elements apart, of channels that are there below `channels`; zeros in
// the place of the others.  WIDE: four channels are there or none is, and lie within one access.
template <int DT, bool WIDE>
__device__ __forceinline__ void la_load(la_block<DT> &b, const typename fc_elem<DT>::type *src, long next, int n, int channels) {
    typedef typename fc_elem<DT>::type E;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (WIDE) {
            fc_vec<DT, 4> v = {};
            if (i < n && channels > 0) v = *(const fc_vec<DT, 4> *)(src + i * next);
            b.row[i] = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) b.row[i].v[e] = i < n && e < channels ? src[i * next + e] : (E)0.f;
        }
    }
}

template <int DT, int PARTS>
__device__ __forceinline__ void la_put(char *base, int plane, int at, const float (&x)[4]) {
    typename la_math<DT>::quad q[PARTS];
    la_split<PARTS>(x, q);
#pragma unroll
    for (int p = 0; p < PARTS; p++) *(typename la_math<DT>::quad *)(base + p * plane + at) = q[p];
}

// Four values as they lie in memory, or split.
template <int DT, int PARTS>
__device__ __forceinline__ void la_put_raw(char *base, int plane, int at, typename fc_elem<DT>::type a, typename fc_elem<DT>::type b,
                                           typename fc_elem<DT>::type c, typename fc_elem<DT>::type d) {
    if constexpr (DT == FC_F16) la_put<DT, PARTS>(base, plane, at, {(float)a, (float)b, (float)c, (float)d});
    else *(typename la_math<DT>::quad *)(base + at) = (typename la_math<DT>::quad){a, b, c, d};
}

// Eight accumulators from `first` on as an operand.
template <int DT>
__device__ __forceinline__ void la_formed(const la_f32x16 &x, int first, typename la_math<DT>::frag (&f)[la_math<DT>::FORMED]) {
    if constexpr (DT == FC_F32) {
#pragma unroll
        for (int e = 0; e < 8; e++) f[0].half[e / 4][e % 4] = x[first + e];
    } else {
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] = x[first + e];
        f[0] = __builtin_convertvector((la_f32x8){r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]}, la_bf16x8);
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] -= (float)f[0][e];
        f[1] = __builtin_convertvector((la_f32x8){r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]}, la_bf16x8);
    }
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

// KT tiles of 32 rows of the state (rows past Dk are zeros), NW wavefronts of 32 columns.  FULL: answers tokens; otherwise only
// forms the state that a segment adds.
template <int DT, int KT, int NW, bool FULL, bool WIDE>
__global__ __launch_bounds__(64 * NW, KT <= 4 ? 2 : 1) void fc_linear_attention_chunk_kernel(const fc_la_run r, int segments, long segment, int slices, float *parts) {
    typedef la_math<DT> M;
    typedef typename M::frag frag;
    typedef typename fc_elem<DT>::type E;
    constexpr int THREADS = 64 * NW, DK = 32 * KT, DV = 32 * NW;
    constexpr int QK_PLANE = 2 * KT * M::FRAG_BYTES, V_PLANE = 2 * NW * M::FRAG_BYTES;
    constexpr int Q_BYTES = FULL ? M::PARTS * QK_PLANE : 0;
    constexpr int QK_ITEMS = (8 * DK / 4 + THREADS - 1) / THREADS, V_ITEMS = 8 * DV / 4 / THREADS;
    extern __shared__ char lds[];
    char *const qs = lds, *const ks = qs + Q_BYTES, *const kt = ks + Q_BYTES, *const vt = kt + M::KEPT * QK_PLANE;
    double *const exact = (double *)(vt + M::PARTS * V_PLANE);      // decay^0 .. decay^32
    float *const power = (float *)(exact + kLaChunk + 1);           // the same, times what enters the state
    int *const odd = (int *)(power + kLaChunk + 1);                 // whether a value of the chunk is not finite,
    int *const since = odd + 1;                                     // and from which token on, for each column

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 5;
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
    // powers between two tokens of a chunk, zero towards an earlier one, and from the state to a token
    float near[16], from;
    const int i_tok = lane & 31;
    if (FULL) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int d = i_tok - (8 * (e / 4) + 4 * g + e % 4);
            near[e] = d < 0 ? 0.f : power[d] * r.scale_out;
        }
        from = (float)exact[i_tok + 1 - r.reverse] * r.scale_out;
    }
    double left = 1.0;      // what the roundings of the chunks' decays have left out so far

    // the state: rows 32*t + 8*(e/4) + 4*g + e%4 of column col
    la_f32x16 S[KT];
    const float *from_state = segments > 1 ? parts + (bh * segments + seg) * (long)r.Dk * r.Dv : r.state_in ? r.state_in + bh * r.Dk * r.Dv : nullptr;
    const long srow = segments > 1 ? r.Dv : r.state_row, scol = segments > 1 ? 1 : r.state_col;
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int row = 32 * t + 8 * (e / 4) + 4 * g + e % 4;
            S[t][e] = FULL && from_state && row < r.Dk && col < r.Dv ? from_state[row * srow + col * scol] : 0.f;
        }

    // this thread's rows and channels of every operand, a chunk at a time
    const long step = r.reverse ? -1 : 1, first = r.reverse ? len - 1 - begin : begin;
    const E *qp[FULL ? QK_ITEMS : 1], *kp[QK_ITEMS], *vp[V_ITEMS];
    int qk_tok[QK_ITEMS], v_tok[V_ITEMS], qk_channels[QK_ITEMS], v_channels[V_ITEMS];
#pragma unroll
    for (int it = 0; it < QK_ITEMS; it++) {
        const int item = tid + it * THREADS, tq = item / (DK / 4), cq = item - tq * (DK / 4);
        qk_tok[it] = 4 * tq;
        qk_channels[it] = r.Dk - 4 * cq;
        if (FULL) qp[it] = (const E *)r.q.p + b * r.q.batch + (h / r.q.share) * r.q.head + (first + step * 4 * tq) * r.q.token + 4 * cq;
        kp[it] = (const E *)r.k.p + b * r.k.batch + (h / r.k.share) * r.k.head + (first + step * 4 * tq) * r.k.token + 4 * cq;
    }
#pragma unroll
    for (int it = 0; it < V_ITEMS; it++) {
        const int item = tid + it * THREADS, tq = item / (DV / 4), cq = item - tq * (DV / 4);
        v_tok[it] = 4 * tq;
        v_channels[it] = r.Dv - col0 - 4 * cq;
        vp[it] = (const E *)r.v.p + b * r.v.batch + (h / r.v.share) * r.v.head + (first + step * 4 * tq) * r.v.token + col0 + 4 * cq;
    }
    const long q_next = step * r.q.token, k_next = step * r.k.token, v_next = step * r.v.token;
    la_block<DT> qb[FULL ? QK_ITEMS : 1], kb[QK_ITEMS], vb[V_ITEMS];
    auto load = [&](long p0) {
        const int n = (int)(end - p0 < kLaChunk ? end - p0 : kLaChunk);
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++) {
            if (FULL) {
                la_load<DT, WIDE>(qb[it], qp[it], q_next, n - qk_tok[it], qk_channels[it]);
                qp[it] += kLaChunk * q_next;
            }
            la_load<DT, WIDE>(kb[it], kp[it], k_next, n - qk_tok[it], qk_channels[it]);
            kp[it] += kLaChunk * k_next;
        }
#pragma unroll
        for (int it = 0; it < V_ITEMS; it++) {
            la_load<DT, WIDE>(vb[it], vp[it], v_next, n - v_tok[it], v_channels[it]);
            vp[it] += kLaChunk * v_next;
        }
    };

    if (begin < end) load(begin);
    for (long p0 = begin; p0 < end; p0 += kLaChunk) {
        const int n = (int)(end - p0 < kLaChunk ? end - p0 : kLaChunk);
        __syncthreads();      // the chunk before is read
#pragma unroll
        for (int it = 0; it < QK_ITEMS; it++) {
            const int item = tid + it * THREADS, tq = item / (DK / 4), cq = item - tq * (DK / 4);
            if (tq >= 8) break;
            if (FULL) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int at = la_tile<DT>::natural(4 * tq + i, cq);
                    la_put_raw<DT, M::PARTS>(qs, QK_PLANE, at, qb[it].row[i].v[0], qb[it].row[i].v[1], qb[it].row[i].v[2], qb[it].row[i].v[3]);
                    la_put_raw<DT, M::PARTS>(ks, QK_PLANE, at, kb[it].row[i].v[0], kb[it].row[i].v[1], kb[it].row[i].v[2], kb[it].row[i].v[3]);
                }
            }
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = n - 1 - 4 * tq - i + r.reverse;
                w[i] = power[d < 0 ? 0 : d];      // rows past n are zeros
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                la_put<DT, M::KEPT>(kt, QK_PLANE, la_tile<DT>::turned(4 * cq + e, tq),
                                    {kb[it].row[0].get(e) * w[0], kb[it].row[1].get(e) * w[1], kb[it].row[2].get(e) * w[2], kb[it].row[3].get(e) * w[3]});
        }
#pragma unroll
        for (int it = 0; it < V_ITEMS; it++) {
            const int item = tid + it * THREADS, tq = item / (DV / 4), cq = item - tq * (DV / 4);
            if (FULL && la_not_finite<DT>(vb[it])) {
                // A value that is not finite would meet the zeros of the tokens before it.  It is taken out here; its column
                // is NaN from its token on.
                *odd = 1;
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = vb[it].row[i].get(e);
                        if (x - x == 0.f) continue;
                        atomicMin(&since[4 * cq + e], 4 * tq + i);
                        vb[it].row[i].v[e] = (E)0.f;
                    }
            }
#pragma unroll
            for (int e = 0; e < 4; e++)
                la_put_raw<DT, M::PARTS>(vt, V_PLANE, la_tile<DT>::turned(4 * cq + e, tq), vb[it].row[0].v[e], vb[it].row[1].v[e],
                                         vb[it].row[2].v[e], vb[it].row[3].v[e]);
        }
        __syncthreads();
        if (p0 + kLaChunk < end) load(p0 + kLaChunk);

        frag vf[2][M::PARTS];
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int p = 0; p < M::PARTS; p++) la_tile<DT>::read_turned(vt + p * V_PLANE, wave, s, lane, vf[s][p]);
        if (FULL) {
            la_f32x16 P, O;
#pragma unroll
            for (int e = 0; e < 16; e++) P[e] = O[e] = 0.f;
#pragma unroll
            for (int s = 0; s < 2 * KT; s++) {
                frag qf[M::PARTS], kf[M::PARTS], sf[M::FORMED];
#pragma unroll
                for (int p = 0; p < M::PARTS; p++) {
                    la_tile<DT>::read_natural(qs + p * QK_PLANE, s, lane, qf[p]);
                    la_tile<DT>::read_natural(ks + p * QK_PLANE, s, lane, kf[p]);
                }
#pragma unroll
                for (int a = 0; a < M::PARTS; a++)
#pragma unroll
                    for (int c = 0; c < M::PARTS; c++)
                        if (a + c < 2) P = M::product(kf[a], qf[c], P);
                la_formed<DT>(S[s / 2], 8 * (s % 2), sf);
#pragma unroll
                for (int a = 0; a < M::FORMED; a++)
#pragma unroll
                    for (int c = 0; c < M::PARTS; c++)
                        if (a + c < 2) O = M::product(sf[a], qf[c], O);
            }
#pragma unroll
            for (int e = 0; e < 16; e++) {
                O[e] *= from;
                // a later token's zero leaves nothing of P, whatever that holds
                asm("" : "+v"(near[e]));      // compared here: sixteen masks kept from chunk to chunk would not fit the scalar registers
                P[e] = near[e] != 0.f ? P[e] * near[e] : 0.f;
            }
            frag pf[2][M::FORMED];
#pragma unroll
            for (int s = 0; s < 2; s++) la_formed<DT>(P, 8 * s, pf[s]);
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int a = 0; a < M::PARTS; a++)
#pragma unroll
                    for (int c = 0; c < M::FORMED; c++)
                        if (a + c < 2) O = M::product(vf[s][a], pf[s][c], O);
            if (*odd) {
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (i_tok >= since[32 * wave + 8 * (e / 4) + 4 * g + e % 4]) O[e] = __builtin_nanf("");
            }
            // lane: token i_tok, columns 8*(e/4) + 4*g + e%4 of the wavefront's 32
            if (i_tok < n) {
                const long t = r.reverse ? len - 1 - p0 - i_tok : p0 + i_tok;
#pragma unroll
                for (int a = 0; a < 4; a++) {
                    const int c = col0 + 32 * wave + 8 * a + 4 * g;
                    if (r.o32) {
                        float *dst = r.o32 + ((b * r.T + t) * r.H + h) * r.Dv + c;
                        if (WIDE && c < r.Dv) {
                            *(float4 *)dst = make_float4(O[4 * a], O[4 * a + 1], O[4 * a + 2], O[4 * a + 3]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (c + e < r.Dv) dst[e] = O[4 * a + e];
                        }
                    } else {
                        E *dst = (E *)r.o + b * r.o_batch + t * r.o_token + h * r.o_head + c;
                        if (WIDE && c < r.Dv) {
                            fc_vec<DT, 4> x;
#pragma unroll
                            for (int e = 0; e < 4; e++) x.set(e, O[4 * a + e]);
                            *(fc_vec<DT, 4> *)dst = x;
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (c + e < r.Dv) dst[e] = (E)O[4 * a + e];
                        }
                    }
                }
            }
        }
        // The decay of a chunk in fp32, rounded so that the product over the chunks keeps to the true power.
        const double want = exact[n] * left;
        const float decay = (float)want;
        if (decay != 0.f) left = want / (double)decay;
#pragma unroll
        for (int t = 0; t < KT; t++) {
#pragma unroll
            for (int e = 0; e < 16; e++) S[t][e] *= decay;
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int a = 0; a < M::KEPT; a++) {
                    frag kf;
                    la_tile<DT>::read_turned(kt + a * QK_PLANE, t, s, lane, kf);
#pragma unroll
                    for (int c = 0; c < M::PARTS; c++)
                        if (a + c < 3) S[t] = M::product(kf, vf[s][c], S[t]);
                }
        }
        if (FULL && *odd) {
            const bool lost = since[32 * wave + i_tok] < kLaChunk;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) S[t][e] = lost ? __builtin_nanf("") : S[t][e];
            __syncthreads();
            if (tid == 0) *odd = 0;
            for (int c = tid; c < DV; c += THREADS) since[c] = kLaChunk;
        }
    }

    float *to_state = FULL ? (seg == segments - 1 && r.state_out ? r.state_out + bh * r.Dk * r.Dv : nullptr)
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
                if (row < r.Dk && col < r.Dv) to_state[row * orow + col * ocol] = S[t][e];
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
            if (r.o32) r.o32[((b * r.T + t) * r.H + h) * r.Dv + c] = 0.f;
            else ((E *)r.o)[b * r.o_batch + t * r.o_token + h * r.o_head + c] = (E)0.f;
        }
    }
}

template <int DT, int KT, int NW>
constexpr size_t la_lds_bytes(bool full) {
    typedef la_math<DT> M;
    return (size_t)2 * KT * M::FRAG_BYTES * ((full ? 2 * M::PARTS : 0) + M::KEPT) + (size_t)2 * NW * M::FRAG_BYTES * M::PARTS + (kLaChunk + 1) * (sizeof(double) + sizeof(float)) + (1 + 32 * NW) * sizeof(int);
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
    // two wavefronts where the state has no more than 64 columns
    if (r.Dv <= 64) {
        if (r.Dk <= 32) return la_launch_one<DT, 1, 2, FULL>(ctx, r, heads, segments, segment, parts);
        if (r.Dk <= 64) return la_launch_one<DT, 2, 2, FULL>(ctx, r, heads, segments, segment, parts);
        if (r.Dk <= 128) return la_launch_one<DT, 4, 2, FULL>(ctx, r, heads, segments, segment, parts);
        return la_launch_one<DT, 8, 2, FULL>(ctx, r, heads, segments, segment, parts);
    }
    if (r.Dk <= 32) return la_launch_one<DT, 1, 4, FULL>(ctx, r, heads, segments, segment, parts);
    if (r.Dk <= 64) return la_launch_one<DT, 2, 4, FULL>(ctx, r, heads, segments, segment, parts);
    if (r.Dk <= 128) return la_launch_one<DT, 4, 4, FULL>(ctx, r, heads, segments, segment, parts);
    return la_launch_one<DT, 8, 4, FULL>(ctx, r, heads, segments, segment, parts);
}
