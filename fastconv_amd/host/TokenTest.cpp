// A block over the patches of a short video, on the device from end to end, checked against the same chain in double on the host:
//   patch embedding (a convolution whose window is the patch: every patch an image, so its output is tokens, channels last)
//   -> group norm + SiLU over each frame -> projections to q, k, v (1x1 convolutions of one-pixel images)
//   -> rotary positions by time, row and column -> linear attention with a decay for each head:
//      all frames but the last as one prompt, the last one token by token from the state that the prompt left
//   and back from the answers' gradient through attention and rotary to the projections, checked by central differences.
//   token_test [-f frames] [-g rows cols] [-p patch] [-c channels] [-n heads] [-k kv_heads] [-d head_size] [-i iterations] [--no-check]
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <vector>

#include "utility/device.h"
#include "utility/helper.h"
#include "utility/rng.h"

using fastconv::Device;
typedef std::vector<float> Floats;
typedef std::vector<double> Doubles;

static float *Upload(const void *host, size_t bytes) {
    Device &d = Device::Get();
    float *p = (float *)d.Alloc(bytes, "upload");
    d.Check(fc_upload(d.ctx(), p, host, bytes), "fc_upload");
    return p;
}
static float *Upload(const Floats &v) { return Upload(v.data(), v.size() * sizeof(float)); }
static float *Buffer(size_t floats) { return (float *)Device::Get().Alloc(floats * sizeof(float), "buffer"); }
static Floats Download(const float *dev, size_t n) {
    Floats v(n);
    Device &d = Device::Get();
    d.Check(fc_download(d.ctx(), v.data(), dev, n * sizeof(float)), "fc_download");
    return v;
}

// A convolution whose window is the whole image: y[N][K] = x[N][C*k*k] w[K][C*k*k]^T.
class Projection {
   public:
    Projection(int n, int c, int window, int k, const Floats &w) : shape_(), plan_() {
        Device &d = Device::Get();
        shape_.N = n; shape_.C = c; shape_.H = shape_.W = window; shape_.K = k; shape_.kh = shape_.kw = window; shape_.sh = shape_.sw = 1;
        d.Check(fc_igemm_make_plan(&shape_, fc_igemm_default_config(&shape_), &plan_), "fc_igemm_make_plan");
        packed_ = Buffer((plan_.Wp_bytes + 3) / 4);
        table_ = (int32_t *)Buffer((plan_.table_bytes + 3) / 4);
        ws_ = plan_.ws_bytes ? Buffer((plan_.ws_bytes + 3) / 4) : NULL;
        y = Buffer((size_t)n * k);
        d.Check(fc_igemm_pack_filter(d.ctx(), &plan_, Upload(w), packed_, table_), "fc_igemm_pack_filter");
    }
    void Forward(const float *x) {
        Device &d = Device::Get();
        d.Check(fc_conv_implicit_gemm(d.ctx(), &plan_, x, packed_, table_, NULL, 0, ws_, y), "fc_conv_implicit_gemm");
    }
    float *y;

   private:
    fc_conv_shape shape_;
    fc_igemm_plan plan_;
    float *packed_, *ws_;
    int32_t *table_;
};

static Doubles HostProjection(const Doubles &x, const Floats &w, size_t n, size_t c, size_t k) {
    Doubles y(n * k);
    for (size_t i = 0; i < n; i++)
        for (size_t j = 0; j < k; j++) {
            double s = 0;
            for (size_t e = 0; e < c; e++) s += x[i * c + e] * w[j * c + e];
            y[i * k + j] = s;
        }
    return y;
}

static void HostRotary(Doubles *x, size_t tokens, size_t heads, size_t d, const std::vector<int32_t> &pos, const Floats &inv_freq, const int *pairs) {
    const size_t R = inv_freq.size();
    for (size_t t = 0; t < tokens; t++)
        for (size_t j = 0; j < R; j++) {
            const int axis = j < (size_t)pairs[0] ? 0 : j < (size_t)(pairs[0] + pairs[1]) ? 1 : 2;
            const double a = (double)pos[t * 3 + axis] * inv_freq[j], c = cos(a), s = sin(a);
            for (size_t h = 0; h < heads; h++) {
                double *p = &(*x)[(t * heads + h) * d];
                const double u = p[j], v = p[j + R];
                p[j] = u * c - v * s;
                p[j + R] = v * c + u * s;
            }
        }
}

// Answers of all tokens, a token at a time.
static Doubles HostAttention(const Doubles &q, const Doubles &k, const Doubles &v, const Floats &log_decay, size_t tokens, size_t heads, size_t kv,
                             size_t d, double scale) {
    Doubles o(tokens * heads * d), S(d * d);
    for (size_t h = 0; h < heads; h++) {
        const size_t hk = h / (heads / kv);
        const double decay = exp((double)log_decay[h]);
        S.assign(d * d, 0.0);
        for (size_t t = 0; t < tokens; t++)
            for (size_t c = 0; c < d; c++) {
                double s = 0;
                for (size_t r = 0; r < d; r++) {
                    S[r * d + c] = decay * S[r * d + c] + k[(t * kv + hk) * d + r] * v[(t * kv + hk) * d + c];
                    s += q[(t * heads + h) * d + r] * S[r * d + c];
                }
                o[(t * heads + h) * d + c] = scale * s;
            }
    }
    return o;
}

static double RelativeError(const Floats &got, const Doubles &want) {
    double off = 0, size = 0;
    for (size_t i = 0; i < want.size(); i++) {
        off += (got[i] - want[i]) * (got[i] - want[i]);
        size += want[i] * want[i];
    }
    return sqrt(off / size);
}

int main(int argc, char **argv) {
    int frames = 3, rows = 5, cols = 7, patch = 4, channels = 48, heads = 4, kv = 2, d = 32, iterations = 5;
    bool check = true;
    for (int i = 1; i < argc; i++) {
        if (!strcmp(argv[i], "-f") && i + 1 < argc) frames = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-g") && i + 2 < argc) { rows = atoi(argv[++i]); cols = atoi(argv[++i]); }
        else if (!strcmp(argv[i], "-p") && i + 1 < argc) patch = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-c") && i + 1 < argc) channels = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-n") && i + 1 < argc) heads = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-k") && i + 1 < argc) kv = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-d") && i + 1 < argc) d = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-i") && i + 1 < argc) iterations = atoi(argv[++i]);
        else if (!strcmp(argv[i], "--no-check")) check = false;
        else { fprintf(stderr, "Error: unknown argument '%s'\n", argv[i]); return 1; }
    }
    if (frames < 2 || rows < 1 || cols < 1 || patch < 1 || channels < 8 || channels % 8 || heads < 1 || kv < 1 || heads % kv || d < 8 || d % 8 || iterations < 1) {
        fprintf(stderr, "Error: need two frames or more, channels and head size in multiples of 8, heads a multiple of the key/value heads\n");
        return 1;
    }
    const size_t grid = (size_t)rows * cols, tokens = frames * grid, prompt = tokens - grid, window = 3 * (size_t)patch * patch;
    const size_t qk = (size_t)heads * d, kk = (size_t)kv * d;

    // weights, patches and positions
    Floats embed(channels * window), wq(qk * channels), wk(kk * channels), wv(kk * channels), gamma(channels), beta(channels), pixels(tokens * window);
    fastconv::FillNormal(1, (float)sqrt(1.0 / window), embed.data(), embed.size());
    fastconv::FillNormal(2, (float)sqrt(1.0 / channels), wq.data(), wq.size());
    fastconv::FillNormal(3, (float)sqrt(1.0 / channels), wk.data(), wk.size());
    fastconv::FillNormal(4, (float)sqrt(1.0 / channels), wv.data(), wv.size());
    fastconv::FillUniform(5, 0.5f, 1.5f, gamma.data(), gamma.size());
    fastconv::FillUniform(6, -0.2f, 0.2f, beta.data(), beta.size());
    fastconv::FillUniform(7, -1.f, 1.f, pixels.data(), pixels.size());
    const int pairs[3] = {d / 8, d / 8, d / 2 - 2 * (d / 8)};
    Floats inv_freq, log_decay(heads);
    for (int a = 0; a < 3; a++)
        for (int j = 0; j < pairs[a]; j++) inv_freq.push_back((float)pow(10000.0, -(double)j / pairs[a]));
    for (int h = 0; h < heads; h++) log_decay[h] = -(float)exp2(-1.0 - 8.0 * h / heads);
    std::vector<int32_t> pos(tokens * 3);
    for (size_t t = 0; t < tokens; t++) {
        pos[3 * t] = (int32_t)(t / grid);
        pos[3 * t + 1] = (int32_t)(t % grid / cols);
        pos[3 * t + 2] = (int32_t)(t % cols);
    }
    const float scale = (float)(1.0 / sqrt((double)d));

    Device::Configure(((size_t)64 << 20) + 64 * tokens * (window + channels + 2 * (qk + kk)) + 16 * (size_t)heads * d * d + 64 * channels * (window + qk + 2 * kk));
    Device &dev = Device::Get();
    fc_context *ctx = dev.ctx();
    Projection to_tokens((int)tokens, 3, patch, channels, embed), to_q((int)tokens, channels, 1, (int)qk, wq), to_k((int)tokens, channels, 1, (int)kk, wk),
        to_v((int)tokens, channels, 1, (int)kk, wv);
    float *x = Upload(pixels), *g = Upload(gamma), *b = Upload(beta), *freq = Upload(inv_freq), *decay = Upload(log_decay);
    int32_t *at = (int32_t *)Upload(pos.data(), pos.size() * sizeof(int32_t));

    fc_group_norm_shape ns = {frames, (long)grid, channels, 8, FC_F32, FC_ACT_SILU, 1e-5f, (long)grid * channels, channels, (long)grid * channels, channels};
    fc_group_norm_plan norm;
    dev.Check(fc_group_norm_make_plan(&ns, &norm), "fc_group_norm_make_plan");
    float *normed = Buffer(tokens * channels), *norm_ws = Buffer(norm.ws_bytes / 4 + 1);

    fc_rotary_shape rs = {};
    rs.B = 1; rs.T = (long)tokens; rs.Hq = heads; rs.Hk = kv; rs.D = d; rs.axes = 3; rs.dtype = FC_F32;
    for (int a = 0; a < 3; a++) rs.pairs[a] = pairs[a];
    rs.q_token = rs.qo_token = (long)qk; rs.k_token = rs.ko_token = (long)kk;
    rs.q_head = rs.qo_head = rs.k_head = rs.ko_head = d;

    fc_linear_attention_shape as = {1, (long)prompt, heads, kv, d, d, FC_F32, scale, 0, (long)qk, d, 0, (long)kk, d, 0, (long)kk, d, 0, (long)qk, d};
    fc_linear_attention_shape one = as, whole = as;
    one.T = 1;
    whole.T = (long)tokens;
    fc_linear_attention_plan many_plan, one_plan, whole_plan;
    dev.Check(fc_linear_attention_make_plan(&as, &many_plan), "fc_linear_attention_make_plan");
    dev.Check(fc_linear_attention_make_plan(&one, &one_plan), "fc_linear_attention_make_plan");
    dev.Check(fc_linear_attention_make_plan(&whole, &whole_plan), "fc_linear_attention_make_plan");
    float *o = Buffer(tokens * qk), *state = Buffer((size_t)heads * d * d);
    size_t ws_bytes = whole_plan.ws_backward_bytes;
    if (many_plan.ws_bytes > ws_bytes) ws_bytes = many_plan.ws_bytes;
    float *attention_ws = Buffer(ws_bytes / 4 + 4);

    Timer timer;
    double prompt_ms = 0, token_ms = 0;
    for (int i = 0; i <= iterations; i++) {      // the first is not timed
        timer.startBench();
        to_tokens.Forward(x);
        dev.Check(fc_group_norm(ctx, &norm, to_tokens.y, g, b, normed, NULL, NULL, norm_ws), "fc_group_norm");
        to_q.Forward(normed);
        to_k.Forward(normed);
        to_v.Forward(normed);
        dev.Check(fc_rotary(ctx, &rs, to_q.y, to_k.y, at, freq, 0, to_q.y, to_k.y), "fc_rotary");
        dev.Check(fc_linear_attention(ctx, &many_plan, to_q.y, to_k.y, to_v.y, decay, o, NULL, state, NULL, attention_ws), "fc_linear_attention");
        dev.Check(fc_sync(ctx), "fc_sync");
        prompt_ms += i ? timer.endBench(1.0) : 0;
        timer.startBench();
        for (size_t t = prompt; t < tokens; t++)
            dev.Check(fc_linear_attention(ctx, &one_plan, to_q.y + t * qk, to_k.y + t * kk, to_v.y + t * kk, decay, o + t * qk, state, state, NULL, NULL),
                      "fc_linear_attention");
        dev.Check(fc_sync(ctx), "fc_sync");
        token_ms += i ? timer.endBench((double)grid) : 0;
    }
    printf("%zu tokens of %d frames: block up to the prompt of %zu %.3f ms, then %.1f us a token\n", tokens, frames, prompt, prompt_ms / iterations,
           1000.0 * token_ms / iterations);

    // back from the gradient of all answers to that of the projections: through attention, then turned back
    Floats up(tokens * qk);
    fastconv::FillNormal(8, 1.f, up.data(), up.size());
    float *dq = Buffer(tokens * qk), *dk = Buffer(tokens * kk), *dv = Buffer(tokens * kk);
    dev.Check(fc_linear_attention_backward(ctx, &whole_plan, Upload(up), to_q.y, to_k.y, to_v.y, decay, dq, dk, dv, NULL, NULL, NULL, NULL, attention_ws),
              "fc_linear_attention_backward");
    dev.Check(fc_rotary(ctx, &rs, dq, dk, at, freq, 1, dq, dk), "fc_rotary");
    if (!check) return 0;

    // the same chain in double
    Doubles tok = HostProjection(Doubles(pixels.begin(), pixels.end()), embed, tokens, window, channels);
    const size_t per = channels / 8;
    for (int f = 0; f < frames; f++)
        for (size_t c0 = 0; c0 < (size_t)channels; c0 += per) {
            double mean = 0, var = 0;
            for (size_t p = 0; p < grid; p++)
                for (size_t c = c0; c < c0 + per; c++) mean += tok[(f * grid + p) * channels + c] / (grid * per);
            for (size_t p = 0; p < grid; p++)
                for (size_t c = c0; c < c0 + per; c++) var += pow(tok[(f * grid + p) * channels + c] - mean, 2) / (grid * per);
            for (size_t p = 0; p < grid; p++)
                for (size_t c = c0; c < c0 + per; c++) {
                    double &v = tok[(f * grid + p) * channels + c];
                    const double z = (v - mean) / sqrt(var + 1e-5) * gamma[c] + beta[c];
                    v = z / (1 + exp(-z));
                }
        }
    const Doubles q0 = HostProjection(tok, wq, tokens, channels, qk), k0 = HostProjection(tok, wk, tokens, channels, kk),
                  v0 = HostProjection(tok, wv, tokens, channels, kk);
    auto answers = [&](Doubles q, Doubles k, const Doubles &v) {
        HostRotary(&q, tokens, heads, d, pos, inv_freq, pairs);
        HostRotary(&k, tokens, kv, d, pos, inv_freq, pairs);
        return HostAttention(q, k, v, log_decay, tokens, heads, kv, d, scale);
    };
    const double err = RelativeError(Download(o, tokens * qk), answers(q0, k0, v0));
    printf("Relative error of the answers against the host chain: %.3e (tolerance 1e-05) %s\n", err, err <= 1e-5 ? "PASS" : "FAIL");

    // the gradients along one direction against a central difference
    const Floats gq = Download(dq, tokens * qk), gk = Download(dk, tokens * kk), gv = Download(dv, tokens * kk);
    Floats uq(q0.size()), uk(k0.size()), uv(v0.size());
    fastconv::FillNormal(9, 1.f, uq.data(), uq.size());
    fastconv::FillNormal(10, 1.f, uk.data(), uk.size());
    fastconv::FillNormal(11, 1.f, uv.data(), uv.size());
    double along = 0, size = 0, diff = 0;
    for (size_t i = 0; i < uq.size(); i++) { along += (double)gq[i] * uq[i]; size += fabs((double)gq[i] * uq[i]); }
    for (size_t i = 0; i < uk.size(); i++) { along += (double)gk[i] * uk[i] + (double)gv[i] * uv[i]; size += fabs((double)gk[i] * uk[i]) + fabs((double)gv[i] * uv[i]); }
    // the answers are of third order in the projections, which differences over two steps take in exactly
    const double e = 1e-2;
    const int steps[4] = {-2, -1, 1, 2};
    const double weights[4] = {1.0 / 12, -8.0 / 12, 8.0 / 12, -1.0 / 12};
    for (int n = 0; n < 4; n++) {
        Doubles q = q0, k = k0, v = v0;
        for (size_t i = 0; i < q.size(); i++) q[i] += steps[n] * e * uq[i];
        for (size_t i = 0; i < k.size(); i++) { k[i] += steps[n] * e * uk[i]; v[i] += steps[n] * e * uv[i]; }
        const Doubles a = answers(q, k, v);
        for (size_t i = 0; i < a.size(); i++) diff += weights[n] * a[i] * up[i] / e;
    }
    const double off = fabs(along - diff) / size;
    printf("Gradient along a direction %.6e, central difference %.6e: off %.3e of its terms (tolerance 1e-05) %s\n", along, diff, off, off <= 1e-5 ? "PASS" : "FAIL");
    return err <= 1e-5 && off <= 1e-5 ? 0 : 2;
}
