// Rotary positions with several axes: every pair (a, b) of a head's channels is turned by position * inv_freq,
//   (a, b) -> (a cos - b sin, b cos + a sin),
// the position being the token's time, row or column by the pair's axis.  The gradient is the turn by the negative angle.
//
// Bound by memory: 6 operations a pair against 4 to 16 bytes read and written.  The cosines of a token are the same for all of
// its heads, so a workgroup takes a few whole tokens: each thread forms a few of their angles, once, into LDS, and then all
// threads walk over the heads of q and k, 16 bytes a lane and access.
// 2 sequences of 16x28x28 tokens with 32 and 8 heads of 128 in bf16 (514 MB read and written): 94 us, 5.5 TB/s.  One token each of 32 sequences: 4.4 us, one
// after another the waits for a position, its angle and the channels.
#include "token_types.h"

namespace {

constexpr int kThreads = 256;
constexpr long kMostThreads = 1l << 32;      // of a launch, not reached
constexpr int kMostTokens = 2;      // of a workgroup: 2 x 12544 tokens of 40 heads 93 us, with 4 98 and with 8 104

struct rotary_params {
    const void *q, *k;
    void *qo, *ko;
    const int32_t *positions;
    const float *inv_freq;
    long tokens;              // B * T
    long T;
    int Hq, heads;            // heads: of q and k together
    int R;                    // pairs
    int axes;
    int end[FC_ROTARY_AXES];  // first pair past each axis
    int units, turning;       // accesses of a head's channels: all of them (a pair of halves counts as one), and those that turn
    fc_fastdiv by_units, by_heads;
    float sign;
    long pos_batch;
    long qb, qt, qh, kb, kt, kh, qob, qot, qoh, kob, kot, koh;
};

// VEC elements an access; the workgroup takes `group` tokens.
template <int DT, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void fc_rotary_kernel(const rotary_params p, int group) {
    extern __shared__ float2 table[];      // [group][R, made even]: cosine and sine
    typedef fc_vec<DT, VEC> V;
    typedef typename fc_elem<DT>::type E;
    const long t0 = (long)blockIdx.x * group;      // counted over all sequences
    const int here = (int)(p.tokens - t0 < group ? p.tokens - t0 : group);
    const int pitch = (p.R + 1) & ~1;
    // where the tokens' heads begin
    struct place {
        const void *from;
        void *to;
    };
    __shared__ place qs[kMostTokens], ks[kMostTokens];
    if ((int)threadIdx.x < here) {
        const long bt = t0 + threadIdx.x, b = bt / p.T, t = bt - b * p.T;
        qs[threadIdx.x] = {(const E *)p.q + b * p.qb + t * p.qt, (E *)p.qo + b * p.qob + t * p.qot};
        ks[threadIdx.x] = {(const E *)p.k + b * p.kb + t * p.kt, (E *)p.ko + b * p.kob + t * p.kot};
    }
    for (int i = threadIdx.x; i < here * p.R; i += kThreads) {
        const int lt = i / p.R, j = i - lt * p.R;
        const long bt = t0 + lt, b = bt / p.T, t = bt - b * p.T;
        int axis = 0;
        while (axis < p.axes - 1 && j >= p.end[axis]) axis++;
        // in turns, of which the whole ones are dropped before anything is rounded to 32 bits: any int32 position keeps
        // its angle to 2^-20 of a turn and better
        const double turns = (double)p.positions[b * p.pos_batch + t * p.axes + axis] * (double)p.inv_freq[j] * 0.15915494309189533577;
        const float part = (float)(turns - rint(turns));
        float s, c;
        sincospif(2.f * part, &s, &c);
        table[lt * pitch + j] = make_float2(c, p.sign * s);
    }
    __syncthreads();
    const int tasks = here * p.heads * p.units;
    constexpr int AT_ONCE = 2;      // accesses read before the first is turned
    for (int first = threadIdx.x; first < tasks; first += AT_ONCE * kThreads) {
        V x[AT_ONCE], y[AT_ONCE];
        E *dst[AT_ONCE];
        int turn[AT_ONCE];      // where its token's begin in the table
        int unit[AT_ONCE];
#pragma unroll
        for (int n = 0; n < AT_ONCE; n++) {
            const int i = first + n * kThreads;
            unit[n] = -1;
            if (i >= tasks) continue;
            const int th = (int)fc_div((uint32_t)i, p.by_units), u = i - th * p.units;
            const int lt = (int)fc_div((uint32_t)th, p.by_heads), h = th - lt * p.heads;
            const bool of_k = h >= p.Hq;
            const place at = of_k ? ks[lt] : qs[lt];
            const E *src = (const E *)at.from + (of_k ? (h - p.Hq) * p.kh : h * p.qh);
            dst[n] = (E *)at.to + (of_k ? (h - p.Hq) * p.koh : h * p.qoh);
            unit[n] = u;
            turn[n] = lt * pitch;
            if (u >= p.turning) {      // channels past the pairs
                x[n] = fc_load_global<V>(src + 2 * p.R + (u - p.turning) * VEC);
            } else if (INTERLEAVED && VEC == 1) {      // odd strides or sizes: the pair by single elements
                x[n] = fc_load_global<V>(src + 2 * u);
                y[n] = fc_load_global<V>(src + 2 * u + 1);
            } else {
                x[n] = fc_load_global<V>(src + u * VEC);
                if (!INTERLEAVED) y[n] = fc_load_global<V>(src + p.R + u * VEC);
            }
        }
#pragma unroll
        for (int n = 0; n < AT_ONCE; n++) {
            const int u = unit[n];
            if (u < 0) continue;
            if (u >= p.turning) {
                fc_store_global(dst[n] + 2 * p.R + (u - p.turning) * VEC, x[n]);
                continue;
            }
            constexpr int PAIRS = INTERLEAVED && VEC > 1 ? VEC / 2 : VEC;
            struct alignas(PAIRS % 2 ? 8 : 16) pairs {
                float2 v[PAIRS];
            };
            const pairs t = *(const pairs *)(table + turn[n] + u * PAIRS);
            if (INTERLEAVED && VEC > 1) {
#pragma unroll
                for (int j = 0; j < PAIRS; j++) {
                    const float a0 = x[n].get(2 * j), a1 = x[n].get(2 * j + 1);
                    x[n].set(2 * j, a0 * t.v[j].x - a1 * t.v[j].y);
                    x[n].set(2 * j + 1, a1 * t.v[j].x + a0 * t.v[j].y);
                }
                fc_store_global(dst[n] + u * VEC, x[n]);
            } else {
#pragma unroll
                for (int j = 0; j < PAIRS; j++) {
                    const float a0 = x[n].get(j), a1 = y[n].get(j);
                    x[n].set(j, a0 * t.v[j].x - a1 * t.v[j].y);
                    y[n].set(j, a1 * t.v[j].x + a0 * t.v[j].y);
                }
                fc_store_global(dst[n] + (INTERLEAVED ? 2 * u : u * VEC), x[n]);
                fc_store_global(dst[n] + (INTERLEAVED ? 2 * u + 1 : p.R + u * VEC), y[n]);
            }
        }
    }
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

template <int DT, int VEC>
void launch(fc_context *ctx, const rotary_params &p, bool interleaved, int group, unsigned blocks, size_t lds) {
    if (interleaved) fc_rotary_kernel<DT, VEC, true><<<dim3(blocks), dim3(kThreads), lds, ctx->stream>>>(p, group);
    else fc_rotary_kernel<DT, VEC, false><<<dim3(blocks), dim3(kThreads), lds, ctx->stream>>>(p, group);
}

template <int DT>
void launch_width(fc_context *ctx, const rotary_params &p, bool interleaved, int vec, int group, unsigned blocks, size_t lds) {
    if constexpr (DT != FC_F32)
        if (vec == 8) return launch<DT, 8>(ctx, p, interleaved, group, blocks, lds);
    if (vec == 4) return launch<DT, 4>(ctx, p, interleaved, group, blocks, lds);
    if (vec == 2) return launch<DT, 2>(ctx, p, interleaved, group, blocks, lds);
    launch<DT, 1>(ctx, p, interleaved, group, blocks, lds);
}

}  // namespace

extern "C" int fc_rotary(fc_context *ctx, const fc_rotary_shape *s, const void *q_dev, const void *k_dev, const int32_t *positions_dev,
                         const float *inv_freq_dev, int inverse, void *q_out_dev, void *k_out_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (!s || s->B < 1 || s->T < 1 || s->Hq < 1 || s->Hk < 0 || s->D < 1 || !fc_dtype_ok(s->dtype) || s->axes < 1 || s->axes > FC_ROTARY_AXES)
        return fail(ctx, FC_ERR_INVALID, "fc_rotary: bad shape");
    long R = 0;
    for (int a = 0; a < s->axes; a++) {
        if (s->pairs[a] < 0) return fail(ctx, FC_ERR_INVALID, "fc_rotary: a negative number of pairs");
        R += s->pairs[a];
    }
    if (R < 1 || 2 * R > s->D) return fail(ctx, FC_ERR_INVALID, "fc_rotary: pairs that do not fit a head");
    if (!q_dev || !q_out_dev || !positions_dev || !inv_freq_dev || (s->Hk > 0 && (!k_dev || !k_out_dev)))
        return fail(ctx, FC_ERR_INVALID, "fc_rotary: null pointer");
    const long strides[13] = {s->positions_batch, s->q_batch, s->q_token, s->q_head, s->k_batch, s->k_token, s->k_head,
                              s->qo_batch, s->qo_token, s->qo_head, s->ko_batch, s->ko_token, s->ko_head};
    for (long v : strides)
        if (v < 0) return fail(ctx, FC_ERR_INVALID, "fc_rotary: negative stride");
    const size_t es = fc_elem_size(s->dtype);
    uint64_t addr = (uint64_t)q_dev | (uint64_t)q_out_dev;
    uint64_t bits = s->q_batch | s->q_token | s->q_head | s->qo_batch | s->qo_token | s->qo_head;
    if (s->Hk > 0) {
        addr |= (uint64_t)k_dev | (uint64_t)k_out_dev;
        bits |= s->k_batch | s->k_token | s->k_head | s->ko_batch | s->ko_token | s->ko_head;
    }
    if ((addr & (es - 1)) || (((uint64_t)positions_dev | (uint64_t)inv_freq_dev) & 3)) return fail(ctx, FC_ERR_INVALID, "fc_rotary: unaligned pointer");
    const long heads = (long)s->Hq + s->Hk, tokens = fc_count(s->B, s->T);
    int group = kMostTokens;
    while (group > 1 && tokens < 1024L * group) group >>= 1;
    // a last workgroup may have one token of two: 2^25 - 2 tokens are the most
    if (s->D > 1024 || heads > 65536 || tokens < 0 || (tokens + group - 1) / group >= kMostThreads / kThreads)
        return fail(ctx, FC_ERR_UNSUPPORTED, "fc_rotary: more than 1024 channels, 65536 heads or 2^25 - 2 tokens");
    if (!fc_apart(s->B, s->qo_batch, s->D) || !fc_apart(s->T, s->qo_token, s->D) || !fc_apart(s->Hq, s->qo_head, s->D) ||
        (s->Hk > 0 && (!fc_apart(s->B, s->ko_batch, s->D) || !fc_apart(s->T, s->ko_token, s->D) || !fc_apart(s->Hk, s->ko_head, s->D))))
        return fail(ctx, FC_ERR_INVALID, "fc_rotary: heads of an output overlap");
    const int vec = fc_widest(s->dtype, bits | (uint64_t)s->D | (uint64_t)(s->interleaved ? 2 * R : R), addr);
    rotary_params p;
    p.q = q_dev; p.k = k_dev; p.qo = q_out_dev; p.ko = k_out_dev;
    p.positions = positions_dev; p.inv_freq = inv_freq_dev;
    p.tokens = tokens; p.T = s->T; p.Hq = s->Hq; p.heads = (int)heads; p.R = (int)R; p.axes = s->axes;
    int end = 0;
    for (int a = 0; a < FC_ROTARY_AXES; a++) {
        if (a < s->axes) end += s->pairs[a];
        p.end[a] = end;
    }
    p.turning = (int)((s->interleaved && vec > 1 ? 2 * R : R) / vec);
    p.units = p.turning + (int)((s->D - 2 * R) / vec);
    p.by_units = fc_make_fastdiv((uint32_t)p.units);
    p.by_heads = fc_make_fastdiv((uint32_t)heads);
    p.sign = inverse ? -1.f : 1.f;
    p.pos_batch = s->positions_batch;
    p.qb = s->q_batch; p.qt = s->q_token; p.qh = s->q_head; p.kb = s->k_batch; p.kt = s->k_token; p.kh = s->k_head;
    p.qob = s->qo_batch; p.qot = s->qo_token; p.qoh = s->qo_head; p.kob = s->ko_batch; p.kot = s->ko_token; p.koh = s->ko_head;
    const unsigned blocks = (unsigned)((tokens + group - 1) / group);
    const size_t lds = (size_t)group * ((R + 1) & ~1l) * sizeof(float2);
    const bool il = s->interleaved != 0;
    if (s->dtype == FC_F32) launch_width<FC_F32>(ctx, p, il, vec, group, blocks, lds);
    else if (s->dtype == FC_BF16) launch_width<FC_BF16>(ctx, p, il, vec, group, blocks, lds);
    else launch_width<FC_F16>(ctx, p, il, vec, group, blocks, lds);
    FC_LAUNCH_CHECK(ctx, "fc_rotary_kernel");
    return FC_OK;
}
