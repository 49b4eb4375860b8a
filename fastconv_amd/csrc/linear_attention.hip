// Linear attention with a decay for each head: entry points, and the recurrence for few tokens.  See linear_attention.h for the
// formulas.
#include "linear_attention.h"

namespace {

constexpr int kThreads = 256;
constexpr long kMostThreads = 1l << 32;      // of a launch, not reached; a head has up to 8 workgroups
constexpr int kMaxDim = 256;
// Up to so many tokens run through the recurrence, about 1 us each; a chunk costs 11 to 15 us with one token or 32.  1 sequence of 16 heads of 128
// in bf16: 4 tokens 8.3 and 11.4 us, 8 tokens 12.2 and 11.3; 8 sequences 10.1 and 12.4, 14.6 and 12.5; 64 of 16 heads of 64 16.5 and 13.5, 24.1 and 13.6;
// 8 of 8 heads of 128 in fp32 8.3 and 15.3, 12.2 and 15.4.
constexpr long kMostSteps = 6;
// Heads from which the recurrence takes 128 columns a workgroup.  Heads of 128, one token, 32 columns and 128: 16 heads 5.6 and 9.6 us, 256 heads 9.7 and
// 12.2, 1024 heads 34 and 26.
constexpr long kWholeRows = 512;
// A sequence is cut up to fill the chip: 16 heads of 128, 12544 tokens in bf16 140 us for 1024 wavefronts, 121 for 2048 and 145 for 4096; with a
// backward pass, 8 x 16 heads of 64 and 3136 tokens 422, 330 and 393.  In fp32, whose heads of 64 take four wavefronts, 8 heads and 11760 tokens 79 us for 1536,
// 70 for 2048, 83 for 3072 and 86 for 4096; 32 x 8 heads and 2048 tokens 239 uncut, 252 in 3 parts, 257 in 4.
constexpr long kWavefronts = 2048;
// A cut costs two launches, k and v read twice, and a state a segment, written and read twice.  In two parts it loses (32 x 16 heads of 64, 4096
// tokens: 388 us against 351 uncut; 1024 tokens 124 and 97), in three it gains (21 x 16 heads, 2048 tokens: 139 and 178).
constexpr long kLeastSegments = 3;
// Segments of two chunks, but where states are larger than what a segment reads and many: of four.  8 sequences of 1225 tokens, 8 heads of 64x128, in fp32
// 71 us in 8 segments of 5 chunks, 75 in 4 and 119 in 2; 16 heads of 128, 512 tokens in bf16: 29.6 in 8 segments, 35.5 in 4; 2048 tokens: 42 in 16,
// 51 in 32.
constexpr long kSmallState = 64 * 128, kFewSegments = 8;
constexpr int kChunk = 32;         // tokens that the matrix cores take at once
constexpr int kChunkRows = 128;    // rows of a state that their kernel holds

// The recurrence.  A workgroup holds some columns of a head's state in registers: COLS threads side by side with 4 columns each, as
// many deep as there are, with ROWS rows each.  A token costs two barriers: its q and k lie in LDS for all, its answer is summed over
// the rows in the wavefront and then over the four wavefronts.
// Bound by the state, which is read and written once a call, 8 bytes an element against 4 operations a token.  32 columns a workgroup
// spread one sequence's heads over the chip; 128, whole rows, read longer pieces and sum over fewer lanes.
// One token of 16 heads of 128 in bf16: 5.4 us, the time of a launch that waits for its state and then for the sums; of 64 sequences in half (134 MB of states):
// 24.7 us, 5.5 TB/s.
template <int DT, int ROWS, int COLS>
__global__ __launch_bounds__(kThreads) void fc_linear_attention_step_kernel(const fc_la_run r) {
    typedef typename fc_elem<DT>::type E;
    constexpr int DEEP = kThreads / COLS, WIDTH = 4 * COLS;
    __shared__ float qs[2][kMaxDim], ks[2][kMaxDim], part[2][4][WIDTH];
    const int tid = threadIdx.x, col = tid % COLS, row = tid / COLS;
    const int slices = (r.Dv + WIDTH - 1) / WIDTH;
    const long bh = blockIdx.x / slices, b = bh / r.H;
    const int h = (int)(bh - b * r.H), c0 = (int)(blockIdx.x - bh * slices) * WIDTH + 4 * col;
    const long len = fc_la_length(r, b);
    const float log_decay = r.log_decay[h];
    const bool wide = r.state_col == 1 && (r.Dv & 3) == 0 &&
                      (((uintptr_t)r.state_in | (uintptr_t)r.state_out) & 15) == 0;      // four columns an access

    const E *q = (const E *)r.q.p + b * r.q.batch + (h / r.q.share) * r.q.head;
    const E *k = (const E *)r.k.p + b * r.k.batch + (h / r.k.share) * r.k.head;
    const E *v = (const E *)r.v.p + b * r.v.batch + (h / r.v.share) * r.v.head;
    const long o = b * r.o_batch + h * r.o_head;

    // a token's values are read while the one before it is taken in
    E q_in = (E)0.f, k_in = (E)0.f, v_in[4] = {(E)0.f, (E)0.f, (E)0.f, (E)0.f};
    auto load = [&](long n) __attribute__((always_inline)) {
        const long t = r.reverse ? len - 1 - n : n;
        if (tid < r.Dk) {
            q_in = q[t * r.q.token + tid];
            k_in = k[t * r.k.token + tid];
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (c0 + j < r.Dv) v_in[j] = v[t * r.v.token + c0 + j];
    };
    if (len > 0) load(0);
    float s[ROWS][4];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int rr = row + DEEP * i;
#pragma unroll
        for (int j = 0; j < 4; j++) s[i][j] = 0.f;
        if (!r.state_in || rr >= r.Dk || c0 >= r.Dv) continue;
        const float *src = r.state_in + bh * r.state_head + rr * r.state_row + c0 * r.state_col;
        if (wide) {
            const float4 x = *(const float4 *)src;
            s[i][0] = x.x; s[i][1] = x.y; s[i][2] = x.z; s[i][3] = x.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c0 + j < r.Dv) s[i][j] = src[j * r.state_col];
        }
    }
    const fc_la_power decay(log_decay, 1);
    for (long n = 0; n < len; n++) {
        const long t = r.reverse ? len - 1 - n : n;
        const int buf = n & 1;
        if (tid < r.Dk) {
            qs[buf][tid] = (float)q_in * r.scale_out;
            ks[buf][tid] = (float)k_in * r.scale_in;
        }
        float vv[4], out[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            vv[j] = (float)v_in[j];
            out[j] = 0.f;
        }
        if (n + 1 < len) load(n + 1);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const int rr = row + DEEP * i;
            if (rr >= r.Dk) break;
            const float kr = ks[buf][rr], qr = qs[buf][rr];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float now = __builtin_fmaf(kr, vv[j], r.reverse ? s[i][j] : decay.times(s[i][j]));
                out[j] = __builtin_fmaf(qr, now, out[j]);
                s[i][j] = r.reverse ? decay.times(now) : now;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
#pragma unroll
            for (int m = COLS; m < 64; m <<= 1) out[j] += __shfl_xor(out[j], m);
        }
        if ((tid & 63) < COLS) {
#pragma unroll
            for (int j = 0; j < 4; j++) part[buf][tid >> 6][4 * col + j] = out[j];
        }
        __syncthreads();
        const int c = (int)(blockIdx.x - bh * slices) * WIDTH + tid;
        if (tid < WIDTH && c < r.Dv) {
            const float sum = (part[buf][0][tid] + part[buf][1][tid]) + (part[buf][2][tid] + part[buf][3][tid]);
            if (r.o_fp32) ((float *)r.o)[o + t * r.o_token + c] = sum;
            else ((E *)r.o)[o + t * r.o_token + c] = (E)sum;
        }
    }
    // tokens past the end of a shorter sequence
    const int c = (int)(blockIdx.x - bh * slices) * WIDTH + tid % WIDTH;
    if (c < r.Dv)
        for (long t = len + tid / WIDTH; t < r.T; t += kThreads / WIDTH) {
            if (r.o_fp32) ((float *)r.o)[o + t * r.o_token + c] = 0.f;
            else ((E *)r.o)[o + t * r.o_token + c] = (E)0.f;
        }
    if (!r.state_out) return;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int rr = row + DEEP * i;
        if (rr >= r.Dk || c0 >= r.Dv) continue;
        float *dst = r.state_out + bh * r.state_head + rr * r.state_row + c0 * r.state_col;
        if (wide) {
            *(float4 *)dst = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c0 + j < r.Dv) dst[j * r.state_col] = s[i][j];
        }
    }
}

// The states that segments begin from: parts[s] becomes what enters segment s, for each element of a head's state.  Bound by the chain of segments, eight of
// which are read at once: 16 heads of 128 in 31 segments, 65 MB read and written, 14 us; 8 heads of 64 in 62 segments, 16 MB, 12 us, and in 123
// segments 21.
__global__ __launch_bounds__(kThreads) void fc_linear_attention_scan_kernel(const fc_la_run r, int segments, long segment, float *parts) {
    constexpr int AHEAD = 8;      // segments read before the first is joined
    const int size = r.Dk * r.Dv, blocks = (size + kThreads - 1) / kThreads;
    const long bh = blockIdx.x / blocks, b = bh / r.H;
    const int i = (int)(blockIdx.x - bh * blocks) * kThreads + threadIdx.x;
    if (i >= size) return;
    const long len = fc_la_length(r, b);
    const float ld = r.log_decay[bh - b * r.H];
    const fc_la_power full(ld, segment);
    const int row = i / r.Dv, col = i - row * r.Dv;
    float s = r.state_in ? r.state_in[bh * r.state_head + row * r.state_row + col * r.state_col] : 0.f;
    float *p = parts + bh * segments * size + i;
    for (int first = 0; first < segments; first += AHEAD) {
        float add[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
            add[a] = first + a < segments - 1 && (first + a) * segment < len ? p[(long)(first + a) * size] : 0.f;
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            if (first + a >= segments) break;
            p[(long)(first + a) * size] = s;
            const long n = len - (first + a) * segment;
            if (n >= segment) s = full.times(s) + add[a];
            else if (n > 0) s = fc_la_power(ld, n).times(s) + add[a];
        }
    }
}

// Answers in fp32 that belong together, [B][T][heads][share][D], added up.
template <int DT>
__global__ __launch_bounds__(kThreads) void fc_linear_attention_sum_kernel(const float *src, void *dst, long values, long T, int heads, int share,
                                                                           int D, long batch, long token, long head) {
    typedef typename fc_elem<DT>::type E;
    for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < values; i += (long)gridDim.x * kThreads) {
        const long row = i / D, d = i - row * D, bt = row / heads, h = row - bt * heads, b = bt / T, t = bt - b * T;
        const float *p = src + row * share * D + d;
        float s = 0.f;
        for (int g = 0; g < share; g++) s += p[(long)g * D];
        ((E *)dst)[b * batch + t * token + h * head + d] = (E)s;
    }
}

int fail(fc_context *ctx, int status, const char *what) { return fc_set_error(ctx, status, what, hipSuccess); }

bool shape_ok(const fc_linear_attention_shape *s) {
    if (!s || s->B < 1 || s->T < 1 || s->H < 1 || s->Hkv < 1 || s->H % s->Hkv || s->Dk < 1 || s->Dv < 1 || !fc_dtype_ok(s->dtype)) return false;
    if (!(s->scale == s->scale) || s->scale - s->scale != 0.f) return false;
    const long strides[12] = {s->q_batch, s->q_token, s->q_head, s->k_batch, s->k_token, s->k_head,
                              s->v_batch, s->v_token, s->v_head, s->o_batch, s->o_token, s->o_head};
    for (long v : strides)
        if (v < 0) return false;
    return true;
}

bool same(const fc_linear_attention_plan &a, const fc_linear_attention_plan &b) {
    const fc_linear_attention_shape &s = a.shape, &t = b.shape;
    return s.B == t.B && s.T == t.T && s.H == t.H && s.Hkv == t.Hkv && s.Dk == t.Dk && s.Dv == t.Dv && s.dtype == t.dtype && s.scale == t.scale &&
           s.q_batch == t.q_batch && s.q_token == t.q_token && s.q_head == t.q_head && s.k_batch == t.k_batch && s.k_token == t.k_token &&
           s.k_head == t.k_head && s.v_batch == t.v_batch && s.v_token == t.v_token && s.v_head == t.v_head && s.o_batch == t.o_batch &&
           s.o_token == t.o_token && s.o_head == t.o_head && a.chunk == b.chunk && a.segments == b.segments && a.ws_bytes == b.ws_bytes &&
           a.ws_backward_bytes == b.ws_backward_bytes;
}

// Floats of the workspace that hold the segments' states; what is added up follows.
size_t states_of(const fc_linear_attention_plan *plan) {
    const fc_linear_attention_shape &s = plan->shape;
    return plan->segments > 1 ? (size_t)s.B * s.H * plan->segments * s.Dk * s.Dv : 0;
}

// The same but for where the tensors begin, which a plan does not know.
bool wide_strides(const fc_linear_attention_shape &s) {
    return ((s.Dk | s.Dv | s.q_batch | s.q_token | s.q_head | s.k_batch | s.k_token | s.k_head | s.v_batch | s.v_token | s.v_head | s.o_batch | s.o_token |
             s.o_head) & 3) == 0;
}

// Tokens of a segment: whole chunks.
long segment_of(const fc_linear_attention_shape &s, int segments) {
    const long chunks = (s.T + kChunk - 1) / kChunk;
    return (chunks + segments - 1) / segments * kChunk;
}

template <int DT, int ROWS, int COLS>
void launch_step_as(fc_context *ctx, const fc_la_run &r, long heads) {
    const unsigned blocks = (unsigned)(heads * ((r.Dv + 4 * COLS - 1) / (4 * COLS)));
    fc_linear_attention_step_kernel<DT, ROWS, COLS><<<dim3(blocks), dim3(kThreads), 0, ctx->stream>>>(r);
}

template <int DT>
void launch_step(fc_context *ctx, const fc_la_run &r, long heads) {
    if (r.Dv > 64 && r.Dk <= 128 && heads >= kWholeRows) {
        if (r.Dk <= 64) launch_step_as<DT, 8, 32>(ctx, r, heads);
        else launch_step_as<DT, 16, 32>(ctx, r, heads);
    } else if (r.Dk <= 32) launch_step_as<DT, 1, 8>(ctx, r, heads);
    else if (r.Dk <= 64) launch_step_as<DT, 2, 8>(ctx, r, heads);
    else if (r.Dk <= 128) launch_step_as<DT, 4, 8>(ctx, r, heads);
    else launch_step_as<DT, 8, 8>(ctx, r, heads);
}

int run_step(fc_context *ctx, const fc_linear_attention_shape &s, const fc_la_run &r) {
    const long heads = (long)s.B * s.H;
    if (s.dtype == FC_F32) launch_step<FC_F32>(ctx, r, heads);
    else if (s.dtype == FC_BF16) launch_step<FC_BF16>(ctx, r, heads);
    else launch_step<FC_F16>(ctx, r, heads);
    FC_LAUNCH_CHECK(ctx, "fc_linear_attention_step_kernel");
    return FC_OK;
}

// Four channels lie within one access, and a chunk's offsets within 31 bits.
bool wide(const fc_la_operand &x, int D, size_t es) {
    return ((D | x.batch | x.token | x.head) & 3) == 0 && ((uintptr_t)x.p & (4 * es - 1)) == 0 && x.token < (1l << 31) / 4 / kChunk - 1024;
}

int run_chunks(fc_context *ctx, const fc_linear_attention_plan *plan, fc_la_run &r, float *parts) {
    const fc_linear_attention_shape &s = plan->shape;
    const size_t es = fc_elem_size(s.dtype);
    r.wide = wide(r.q, r.Dk, es) && wide(r.k, r.Dk, es) && wide(r.v, r.Dv, es) &&
             wide({r.o, r.o_batch, r.o_token, r.o_head, 1}, r.Dv, r.o_fp32 ? sizeof(float) : es);
    const long heads = (long)s.B * s.H, segment = segment_of(s, plan->segments);
    if (!r.parts_ready) {
        r.part_row = r.Dv;
        r.part_col = 1;
    }
    if (plan->segments > 1 && !r.parts_ready) {
        const int rc = s.dtype == FC_F32    ? fc_la_state_f32(ctx, r, heads, plan->segments, segment, parts)
                       : s.dtype == FC_BF16 ? fc_la_state_bf16(ctx, r, heads, plan->segments, segment, parts)
                                            : fc_la_state_f16(ctx, r, heads, plan->segments, segment, parts);
        if (rc) return rc;
        const unsigned blocks = (unsigned)(heads * ((r.Dk * r.Dv + kThreads - 1) / kThreads));
        fc_linear_attention_scan_kernel<<<dim3(blocks), dim3(kThreads), 0, ctx->stream>>>(r, plan->segments, segment, parts);
        FC_LAUNCH_CHECK(ctx, "fc_linear_attention_scan_kernel");
    }
    return s.dtype == FC_F32    ? fc_la_answer_f32(ctx, r, heads, plan->segments, segment, parts)
           : s.dtype == FC_BF16 ? fc_la_answer_bf16(ctx, r, heads, plan->segments, segment, parts)
                                : fc_la_answer_f16(ctx, r, heads, plan->segments, segment, parts);
}

// One run.  Its answers go to `dst` with the strides of r, or, where several belong together, in fp32 to `sums` and from there to dst: those
// of the query heads that share a key/value head, if `share` of them do, and those of the two halves of a state with more rows than the
// matrix cores' kernel holds, which is as two states that never meet.
int run(fc_context *ctx, const fc_linear_attention_plan *plan, fc_la_run r, float *parts, float *sums, void *dst, int share) {
    const fc_linear_attention_shape &s = plan->shape;
    const int halves = plan->chunk && r.Dk > kChunkRows ? 2 : 1, together = share * halves;
    const long batch = r.o_batch, token = r.o_token, head = r.o_head;
    r.o = dst;
    if (together > 1) {
        r.o = sums;
        r.o_fp32 = true;
        r.o_head = (long)halves * r.Dv;
        r.o_token = r.H * r.o_head;
        r.o_batch = s.T * r.o_token;
    }
    const size_t es = fc_elem_size(s.dtype);
    for (int half = 0; half < halves; half++) {
        fc_la_run one = r;
        if (halves > 1) {
            const long first = half * (long)kChunkRows;
            one.q.p = (const char *)r.q.p + first * es;
            one.k.p = (const char *)r.k.p + first * es;
            one.Dk = half ? r.Dk - kChunkRows : kChunkRows;
            if (r.state_in) one.state_in = r.state_in + first * r.state_row;
            if (r.state_out) one.state_out = r.state_out + first * r.state_row;
            one.o = sums + half * r.Dv;
        }
        const int rc = plan->chunk ? run_chunks(ctx, plan, one, parts) : run_step(ctx, s, one);
        if (rc) return rc;
    }
    if (together == 1) return FC_OK;
    const int heads = r.H / share;
    const long values = (long)s.B * s.T * heads * r.Dv, want = (values + kThreads - 1) / kThreads;
    const unsigned blocks = (unsigned)(want < 65536 ? want : 65536);
    const auto sum = s.dtype == FC_F32    ? fc_linear_attention_sum_kernel<FC_F32>
                     : s.dtype == FC_BF16 ? fc_linear_attention_sum_kernel<FC_BF16>
                                          : fc_linear_attention_sum_kernel<FC_F16>;
    sum<<<dim3(blocks), dim3(kThreads), 0, ctx->stream>>>(sums, dst, values, s.T, heads, together, r.Dv, batch, token, head);
    FC_LAUNCH_CHECK(ctx, "fc_linear_attention_sum_kernel");
    return FC_OK;
}

}  // namespace

extern "C" int fc_linear_attention_make_plan(const fc_linear_attention_shape *s, fc_linear_attention_plan *plan) {
    if (!plan || !shape_ok(s)) return FC_ERR_INVALID;
    if (s->Dk > kMaxDim || s->Dv > kMaxDim || fc_count(s->B, s->H) < 0 || fc_count(s->B, s->H) >= kMostThreads / kThreads / 8) return FC_ERR_UNSUPPORTED;
    const int most = s->Dk > s->Dv ? s->Dk : s->Dv;
    const long tokens = fc_count(s->B, s->T), values = tokens < 0 ? -1 : fc_count(tokens, s->H, 8 * most);
    if (s->T >= (1l << 31) || values < 0) return FC_ERR_UNSUPPORTED;
    *plan = {};
    plan->shape = *s;
    plan->segments = 1;
    if (s->T > kMostSteps) {
        plan->chunk = kChunk;
        // of the forward run, as it is launched; the backward runs are cut where it is, since dk begins from dv's states.  More than 128 rows or
        // columns count as two states.
        const long wavefronts = fc_la_wavefronts(s->dtype, s->Dk, s->Dv, wide_strides(*s)) * ((most + 127) / 128), chunks = (s->T + kChunk - 1) / kChunk;
        long segments = kWavefronts / (s->B * (long)s->H * wavefronts);
        long worth = chunks / 2;
        if ((long)s->Dk * s->Dv > kSmallState && worth > kFewSegments) worth = chunks / 4 > kFewSegments ? chunks / 4 : kFewSegments;
        if (segments > worth) segments = worth;
        if (segments > 1) {
            const long per = (chunks + segments - 1) / segments;
            segments = (chunks + per - 1) / per;
        }
        if (segments >= kLeastSegments) plan->segments = (int)segments;
        if (plan->segments > 1) plan->ws_bytes = (size_t)s->B * s->H * plan->segments * s->Dk * s->Dv * sizeof(float);
    }
    // Answers that are added up afterwards: of the forward run, of the largest backward one.
    const size_t answers = (size_t)s->B * s->T * s->H * sizeof(float);
    const bool halves = plan->chunk && most > kChunkRows;
    plan->ws_backward_bytes = plan->ws_bytes + (halves ? 2 : s->H > s->Hkv ? 1 : 0) * answers * most;
    if (plan->chunk && s->Dk > kChunkRows) plan->ws_bytes += 2 * answers * s->Dv;
    return FC_OK;
}

static bool apart(const fc_linear_attention_shape &s, long heads, long batch, long token, long head, int row) {
    return fc_apart(s.B, batch, row) && fc_apart(s.T, token, row) && fc_apart(heads, head, row);
}

static int check_plan(fc_context *ctx, const fc_linear_attention_plan *plan, const char *what) {
    fc_linear_attention_plan own;
    if (!plan || fc_linear_attention_make_plan(&plan->shape, &own) != FC_OK || !same(*plan, own)) return fail(ctx, FC_ERR_INVALID, what);
    return FC_OK;
}

extern "C" int fc_linear_attention(fc_context *ctx, const fc_linear_attention_plan *plan, const void *q_dev, const void *k_dev,
                                   const void *v_dev, const float *log_decay_dev, void *o_dev, const float *state_in_dev,
                                   float *state_out_dev, const int32_t *lengths_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_linear_attention: not a plan of fc_linear_attention_make_plan")) return FC_ERR_INVALID;
    const fc_linear_attention_shape &s = plan->shape;
    if (!q_dev || !k_dev || !v_dev || !log_decay_dev || !o_dev || (!ws_dev && plan->ws_bytes)) return fail(ctx, FC_ERR_INVALID, "fc_linear_attention: null pointer");
    if ((((uint64_t)q_dev | (uint64_t)k_dev | (uint64_t)v_dev | (uint64_t)o_dev) & (fc_elem_size(s.dtype) - 1)) || ((uint64_t)ws_dev & 15) ||
        (((uint64_t)log_decay_dev | (uint64_t)state_in_dev | (uint64_t)state_out_dev | (uint64_t)lengths_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_linear_attention: unaligned pointer");
    if (!apart(s, s.H, s.o_batch, s.o_token, s.o_head, s.Dv)) return fail(ctx, FC_ERR_INVALID, "fc_linear_attention: heads of o overlap");
    const int share = s.H / s.Hkv;
    fc_la_run r = {};
    r.q = {q_dev, s.q_batch, s.q_token, s.q_head, 1};
    r.k = {k_dev, s.k_batch, s.k_token, s.k_head, share};
    r.v = {v_dev, s.v_batch, s.v_token, s.v_head, share};
    r.o_batch = s.o_batch; r.o_token = s.o_token; r.o_head = s.o_head;
    r.state_in = state_in_dev; r.state_out = state_out_dev; r.state_head = (long)s.Dk * s.Dv; r.state_row = s.Dv; r.state_col = 1;
    r.log_decay = log_decay_dev; r.lengths = lengths_dev;
    r.T = s.T; r.H = s.H; r.Dk = s.Dk; r.Dv = s.Dv;
    r.scale_in = 1.f; r.scale_out = s.scale;
    return run(ctx, plan, r, (float *)ws_dev, (float *)ws_dev + states_of(plan), o_dev, 1);
}

extern "C" int fc_linear_attention_backward(fc_context *ctx, const fc_linear_attention_plan *plan, const void *do_dev, const void *q_dev,
                                            const void *k_dev, const void *v_dev, const float *log_decay_dev, void *dq_dev, void *dk_dev,
                                            void *dv_dev, const float *state_in_dev, const float *dstate_out_dev, float *dstate_in_dev,
                                            const int32_t *lengths_dev, void *ws_dev) {
    if (!fc_ctx_ok(ctx)) return FC_ERR_STATE;
    if (check_plan(ctx, plan, "fc_linear_attention_backward: not a plan of fc_linear_attention_make_plan")) return FC_ERR_INVALID;
    const fc_linear_attention_shape &s = plan->shape;
    if (!do_dev || !q_dev || !k_dev || !v_dev || !log_decay_dev || !dq_dev || !dk_dev || !dv_dev || (!ws_dev && plan->ws_backward_bytes))
        return fail(ctx, FC_ERR_INVALID, "fc_linear_attention_backward: null pointer");
    const uint64_t addr = (uint64_t)do_dev | (uint64_t)q_dev | (uint64_t)k_dev | (uint64_t)v_dev | (uint64_t)dq_dev | (uint64_t)dk_dev | (uint64_t)dv_dev;
    if ((addr & (fc_elem_size(s.dtype) - 1)) || ((uint64_t)ws_dev & 15) ||
        (((uint64_t)log_decay_dev | (uint64_t)state_in_dev | (uint64_t)dstate_out_dev | (uint64_t)dstate_in_dev | (uint64_t)lengths_dev) & 3))
        return fail(ctx, FC_ERR_INVALID, "fc_linear_attention_backward: unaligned pointer");
    if (!apart(s, s.H, s.q_batch, s.q_token, s.q_head, s.Dk) || !apart(s, s.Hkv, s.k_batch, s.k_token, s.k_head, s.Dk) ||
        !apart(s, s.Hkv, s.v_batch, s.v_token, s.v_head, s.Dv))
        return fail(ctx, FC_ERR_INVALID, "fc_linear_attention_backward: heads of a gradient overlap");
    const int share = s.H / s.Hkv;
    const fc_la_operand q = {q_dev, s.q_batch, s.q_token, s.q_head, 1}, k = {k_dev, s.k_batch, s.k_token, s.k_head, share},
                        v = {v_dev, s.v_batch, s.v_token, s.v_head, share}, d = {do_dev, s.o_batch, s.o_token, s.o_head, 1};
    float *parts = (float *)ws_dev, *sums = parts + states_of(plan);
    fc_la_run r = {};
    r.log_decay = log_decay_dev; r.lengths = lengths_dev;
    r.T = s.T; r.H = s.H;
    r.state_head = (long)s.Dk * s.Dv;
    // dq, from the transposed state
    r.q = d; r.k = v; r.v = k;
    r.Dk = s.Dv; r.Dv = s.Dk;
    r.state_in = state_in_dev; r.state_row = 1; r.state_col = s.Dv;
    r.scale_in = 1.f; r.scale_out = s.scale;
    r.o_batch = s.q_batch; r.o_token = s.q_token; r.o_head = s.q_head;
    int rc = run(ctx, plan, r, parts, sums, dq_dev, 1);
    if (rc) return rc;
    // dv, from the last token to the first, and the gradient of the first state
    r.reverse = 1;
    r.scale_in = s.scale; r.scale_out = 1.f;
    r.q = k; r.k = q; r.v = d;
    r.Dk = s.Dk; r.Dv = s.Dv;
    r.state_in = dstate_out_dev; r.state_out = dstate_in_dev; r.state_row = s.Dv; r.state_col = 1;
    r.o_batch = s.v_batch; r.o_token = s.v_token; r.o_head = s.v_head;
    rc = run(ctx, plan, r, parts, sums, dv_dev, share);
    if (rc) return rc;
    // dk: its segments begin from the same states, transposed
    r.q = v; r.k = d; r.v = q;
    r.Dk = s.Dv; r.Dv = s.Dk;
    r.state_out = nullptr; r.state_row = 1; r.state_col = s.Dv;
    r.parts_ready = plan->segments > 1 && s.Dk <= kChunkRows && s.Dv <= kChunkRows;
    r.part_row = 1; r.part_col = s.Dv;
    r.o_batch = s.k_batch; r.o_token = s.k_token; r.o_head = s.k_head;
    return run(ctx, plan, r, parts, sums, dk_dev, share);
}
