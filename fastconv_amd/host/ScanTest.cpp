// A state-space block over the patches of a short video, on the device from end to end, checked against the same chain in double on the host:
//   patch embedding (a convolution whose window is the patch: every patch an image, so its output is tokens, channels last)
//   -> RMS norm in 8 bits -> 8-bit projection to the inner channels and their gate -> short causal convolution + SiLU of each channel
//   -> 8-bit projection to steps, B and C -> selective scan with the gate -> RMS norm in 8 bits -> 8-bit projection back -> RMS norm with the residual:
//      all frames but the last as one prompt, the last one token by token from the rows and states that the prompt left
// and back from a gradient of the normed answers through norm, scan and convolution to all that goes into them, checked by central differences.
//   scan_test [-f frames] [-g rows cols] [-p patch] [-c channels] [-e inner_channels] [-s states] [-k taps] [-i iterations] [--no-check]
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <vector>

#include "utility/device.h"
#include "utility/helper.h"
#include "utility/rng.h"

using fastconv::Device;
typedef std::vector<float> Floats;
typedef std::vector<double> Doubles;

static float *Buffer(size_t floats) { return (float *)Device::Get().Alloc(floats * sizeof(float), "buffer"); }
static float *Upload(const Floats &v) {
    Device &d = Device::Get();
    float *p = Buffer(v.size());
    d.Check(fc_upload(d.ctx(), p, v.data(), v.size() * sizeof(float)), "fc_upload");
    return p;
}
static Floats Download(const float *dev, size_t n) {
    Floats v(n);
    Device &d = Device::Get();
    d.Check(fc_download(d.ctx(), v.data(), dev, n * sizeof(float)), "fc_download");
    return v;
}

// Tokens from the patches of a video: y[N][K] = x[N][C*k*k] w[K][C*k*k]^T.
class Embedding {
   public:
    Embedding(int n, int c, int window, int k, const Floats &w) : shape_(), plan_() {
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

// A matrix in 8 bits, quantised once, and what its products need.
class Matrix8 {
   public:
    Matrix8(const Floats &w, int outputs, int inputs, size_t most_tokens) : outputs_(outputs), inputs_(inputs) {
        Device &d = Device::Get();
        w_ = (int8_t *)Buffer((w.size() + 3) / 4);
        scale_ = Buffer(outputs);
        d.Check(fc_quantize_rows(d.ctx(), outputs, inputs, FC_F32, Upload(w), inputs, w_, inputs, scale_), "fc_quantize_rows");
        for (size_t rows : {most_tokens, (size_t)1}) {
            fc_int8_product_plan plan = Plan(rows);
            if (plan.ws_bytes > ws_bytes_) ws_bytes_ = plan.ws_bytes;
        }
        ws_ = ws_bytes_ ? Buffer((ws_bytes_ + 3) / 4) : NULL;
    }
    void Forward(size_t tokens, const int8_t *x, const float *x_scale, float *y) {
        Device &d = Device::Get();
        const fc_int8_product_plan plan = Plan(tokens);
        if (plan.ws_bytes > ws_bytes_) { fprintf(stderr, "Error: workspace of a product\n"); exit(1); }
        d.Check(fc_int8_product(d.ctx(), &plan, x, x_scale, w_, scale_, NULL, y, ws_), "fc_int8_product");
    }

   private:
    fc_int8_product_plan Plan(size_t tokens) const {
        fc_int8_product_shape s = {(long)tokens, outputs_, inputs_, FC_F32, inputs_, inputs_, outputs_};
        fc_int8_product_plan plan;
        Device::Get().Check(fc_int8_product_make_plan(&s, &plan), "fc_int8_product_make_plan");
        return plan;
    }
    int outputs_, inputs_;
    int8_t *w_;
    float *scale_, *ws_;
    size_t ws_bytes_ = 0;
};

struct Sizes {
    size_t channels, inner, states, taps;
    size_t shared() const { return inner + 2 * states; }      // steps, B and C of a token
};

// Device buffers of all tokens, and the plans of calls that take some of them.
struct Block {
    Sizes s;
    Matrix8 *in, *mid, *out;
    float *gamma, *gamma_inner, *w, *bias, *A, *D, *step_bias;
    float *tokens, *xz, *u, *shared, *y, *back, *sum, *result;
    int8_t *q, *qi;
    float *scale;
    float *rows, *state, *scan_ws;

    fc_causal_conv_plan Conv(size_t n) const {
        fc_causal_conv_shape c = {1, (long)n, (int)s.inner, (int)s.taps, FC_F32, FC_ACT_SILU, 0, (long)(2 * s.inner), 0, (long)s.inner};
        fc_causal_conv_plan p;
        Device::Get().Check(fc_causal_conv_make_plan(&c, &p), "fc_causal_conv_make_plan");
        return p;
    }
    fc_selective_scan_plan Scan(size_t n) const {
        const long d = (long)s.inner, m = (long)s.shared();
        fc_selective_scan_shape c = {1, (long)n, (int)s.inner, (int)s.states, 1, FC_F32, 1, 0, d, 0, m, 0, 2 * d, 0, m, 0, 0, m, 0, 0, d};
        fc_selective_scan_plan p;
        Device::Get().Check(fc_selective_scan_make_plan(&c, &p), "fc_selective_scan_make_plan");
        return p;
    }
    fc_rms_norm_plan Norm(size_t n, size_t c) const {
        fc_rms_norm_shape r = {(long)n, (int)c, FC_F32, 1e-5f, (long)c, (long)c, (long)c, (long)c};
        fc_rms_norm_plan p;
        Device::Get().Check(fc_rms_norm_make_plan(&r, &p), "fc_rms_norm_make_plan");
        return p;
    }
    // tokens from t on, n of them; the first call begins from nothing
    void Forward(size_t t, size_t n) {
        Device &d = Device::Get();
        fc_context *ctx = d.ctx();
        const size_t D = s.inner, C = s.channels, M = s.shared();
        const fc_rms_norm_plan norm = Norm(n, C), inner_norm = Norm(n, D);
        const fc_causal_conv_plan conv = Conv(n);
        const fc_selective_scan_plan scan = Scan(n);
        d.Check(fc_rms_norm_int8(ctx, &norm, tokens + t * C, NULL, gamma, NULL, q, scale), "fc_rms_norm_int8");
        in->Forward(n, q, scale, xz + t * 2 * D);
        d.Check(fc_causal_conv(ctx, &conv, xz + t * 2 * D, w, bias, u + t * D, t ? rows : NULL, rows, NULL), "fc_causal_conv");
        d.Check(fc_quantize_rows(ctx, (long)n, (int)D, FC_F32, u + t * D, (long)D, qi, (long)D, scale), "fc_quantize_rows");
        mid->Forward(n, qi, scale, shared + t * M);
        const float *m = shared + t * M;
        d.Check(fc_selective_scan(ctx, &scan, u + t * D, m, A, m + D, m + D + s.states, this->D, xz + t * 2 * D + D, step_bias, y + t * D, t ? state : NULL, state, NULL,
                                  scan_ws), "fc_selective_scan");
        d.Check(fc_rms_norm_int8(ctx, &inner_norm, y + t * D, NULL, gamma_inner, NULL, qi, scale), "fc_rms_norm_int8");
        out->Forward(n, qi, scale, back + t * C);
        d.Check(fc_rms_norm(ctx, &norm, back + t * C, tokens + t * C, gamma, sum + t * C, result + t * C, NULL), "fc_rms_norm");
    }
};

// ---- the same in double

static Doubles HostNorm(const Doubles &x, const Floats &gamma, size_t c) {
    Doubles y(x.size());
    for (size_t t = 0; t < x.size() / c; t++) {
        double squares = 0;
        for (size_t i = 0; i < c; i++) squares += x[t * c + i] * x[t * c + i] / c;
        for (size_t i = 0; i < c; i++) y[t * c + i] = x[t * c + i] / sqrt(squares + (double)1e-5f) * gamma[i];
    }
    return y;
}

// Rows as 8 bits hold them: whole multiples of a 127th of their largest value.
static Doubles Held(const Doubles &x, size_t c) {
    Doubles y(x.size());
    for (size_t t = 0; t < x.size() / c; t++) {
        double top = 0;
        for (size_t i = 0; i < c; i++) top = fmax(top, fabs(x[t * c + i]));
        for (size_t i = 0; i < c; i++) y[t * c + i] = top > 0 ? nearbyint(x[t * c + i] * 127 / top) * top / 127 : 0.0;
    }
    return y;
}

static Doubles HostProduct(const Doubles &x, const Doubles &w, size_t c, size_t k) {
    const size_t n = x.size() / c;
    Doubles y(n * k);
#pragma omp parallel for
    for (size_t i = 0; i < n; i++)
        for (size_t j = 0; j < k; j++) {
            double s = 0;
            for (size_t e = 0; e < c; e++) s += x[i * c + e] * w[j * c + e];
            y[i * k + j] = s;
        }
    return y;
}

static double Silu(double z) { return z / (1 + exp(-z)); }

// x: the first D of 2D channels of a row
static Doubles HostConv(const Doubles &x, size_t pitch, const Doubles &w, const Floats &bias, size_t n, const Sizes &s) {
    Doubles u(n * s.inner);
    for (size_t t = 0; t < n; t++)
        for (size_t d = 0; d < s.inner; d++) {
            double z = bias[d];
            for (size_t j = 0; j < s.taps; j++)
                if (t + j + 1 >= s.taps) z += w[d * s.taps + j] * x[(t + j + 1 - s.taps) * pitch + d];
            u[t * s.inner + d] = Silu(z);
        }
    return u;
}

static Doubles HostScan(const Doubles &u, const Doubles &shared, const Doubles &xz, const Doubles &A, const Doubles &D, const Floats &bias, size_t n, const Sizes &s) {
    Doubles y(n * s.inner);
    const size_t M = s.shared();
#pragma omp parallel for
    for (size_t d = 0; d < s.inner; d++) {
        Doubles h(s.states, 0.0);
        for (size_t t = 0; t < n; t++) {
            const double raw = shared[t * M + d] + bias[d], dt = (raw > 0 ? raw : 0) + log1p(exp(-fabs(raw))), x = u[t * s.inner + d];
            double sum = D[d] * x;
            for (size_t k = 0; k < s.states; k++) {
                h[k] = exp(dt * A[d * s.states + k]) * h[k] + dt * x * shared[t * M + s.inner + k];
                sum += shared[t * M + s.inner + s.states + k] * h[k];
            }
            y[t * s.inner + d] = sum * Silu(xz[t * 2 * s.inner + s.inner + d]);
        }
    }
    return y;
}

static Doubles Wide(const Floats &v) { return Doubles(v.begin(), v.end()); }

static double RelativeError(const Floats &got, const Doubles &want) {
    double off = 0, size = 0;
    for (size_t i = 0; i < want.size(); i++) {
        off += (got[i] - want[i]) * (got[i] - want[i]);
        size += want[i] * want[i];
    }
    return sqrt(off / size);
}

static Floats Normal(uint64_t seed, size_t n, double sigma) {
    Floats v(n);
    fastconv::FillNormal(seed, (float)sigma, v.data(), n);
    return v;
}

int main(int argc, char **argv) {
    int frames = 3, rows = 5, cols = 7, patch = 4, channels = 48, inner = 96, states = 16, taps = 4, iterations = 5;
    bool check = true;
    for (int i = 1; i < argc; i++) {
        if (!strcmp(argv[i], "-f") && i + 1 < argc) frames = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-g") && i + 2 < argc) { rows = atoi(argv[++i]); cols = atoi(argv[++i]); }
        else if (!strcmp(argv[i], "-p") && i + 1 < argc) patch = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-c") && i + 1 < argc) channels = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-e") && i + 1 < argc) inner = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-s") && i + 1 < argc) states = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-k") && i + 1 < argc) taps = atoi(argv[++i]);
        else if (!strcmp(argv[i], "-i") && i + 1 < argc) iterations = atoi(argv[++i]);
        else if (!strcmp(argv[i], "--no-check")) check = false;
        else { fprintf(stderr, "Error: unknown argument '%s'\n", argv[i]); return 1; }
    }
    if (frames < 2 || rows < 1 || cols < 1 || patch < 1 || channels < 1 || inner < 1 || states < 1 || states > 64 || taps < 2 || taps > 8 || iterations < 1) {
        fprintf(stderr, "Error: need two frames or more, 1 to 64 states and 2 to 8 taps\n");
        return 1;
    }
    const Sizes s = {(size_t)channels, (size_t)inner, (size_t)states, (size_t)taps};
    const size_t grid = (size_t)rows * cols, tokens = frames * grid, prompt = tokens - grid, window = 3 * (size_t)patch * patch, C = s.channels, D = s.inner, M = s.shared();

    // weights and patches; steps from 0.001 to 0.1, rates from 1 to the number of states
    const Floats embed = Normal(1, C * window, sqrt(1.0 / window)), w_in = Normal(2, 2 * D * C, sqrt(1.0 / C)), w_mid = Normal(3, M * D, sqrt(1.0 / D)),
                 w_out = Normal(4, C * D, sqrt(1.0 / D)), conv_w = Normal(5, D * s.taps, sqrt(1.0 / s.taps)), conv_b = Normal(6, D, 0.2);
    Floats gamma(C), gamma_inner(D), skip(D), A(D * s.states), step_bias(D), pixels(tokens * window);
    fastconv::FillUniform(7, 0.5f, 1.5f, gamma.data(), C);
    fastconv::FillUniform(8, 0.5f, 1.5f, gamma_inner.data(), D);
    fastconv::FillUniform(9, 0.5f, 1.5f, skip.data(), D);
    fastconv::FillUniform(10, 0.f, 1.f, step_bias.data(), D);
    fastconv::FillUniform(11, -1.f, 1.f, pixels.data(), pixels.size());
    for (size_t d = 0; d < D; d++) {
        step_bias[d] = (float)log(expm1(exp(log(1e-3) + log(100.0) * step_bias[d])));
        for (size_t k = 0; k < s.states; k++) A[d * s.states + k] = -(float)(k + 1);
    }

    Block b;
    b.s = s;
    const fc_selective_scan_plan whole = b.Scan(tokens), many = b.Scan(prompt);
    const fc_causal_conv_plan conv_all = b.Conv(tokens);
    const fc_rms_norm_plan norm_all = b.Norm(tokens, D);
    const size_t scan_ws = std::max(std::max(whole.ws_bytes, whole.ws_backward_bytes), many.ws_bytes);
    Device::Configure(((size_t)64 << 20) + 64 * tokens * (window + 4 * C + 12 * D + 4 * M) + 64 * (C * window + 4 * D * C + M * D + D * (s.states + 8)) + 2 * scan_ws +
                      conv_all.ws_backward_bytes + norm_all.ws_backward_bytes);
    Device &dev = Device::Get();
    fc_context *ctx = dev.ctx();
    Embedding embedding((int)tokens, 3, patch, channels, embed);
    Matrix8 in(w_in, 2 * inner, channels, prompt), mid(w_mid, (int)M, inner, prompt), out(w_out, channels, inner, prompt);
    b.in = &in; b.mid = &mid; b.out = &out;
    b.gamma = Upload(gamma); b.gamma_inner = Upload(gamma_inner); b.w = Upload(conv_w); b.bias = Upload(conv_b);
    b.A = Upload(A); b.D = Upload(skip); b.step_bias = Upload(step_bias);
    b.tokens = embedding.y;
    b.xz = Buffer(tokens * 2 * D); b.u = Buffer(tokens * D); b.shared = Buffer(tokens * M); b.y = Buffer(tokens * D);
    b.back = Buffer(tokens * C); b.sum = Buffer(tokens * C); b.result = Buffer(tokens * C);
    b.q = (int8_t *)Buffer(tokens * C / 4 + 1); b.qi = (int8_t *)Buffer(tokens * D / 4 + 1); b.scale = Buffer(tokens);
    b.rows = Buffer((s.taps - 1) * D); b.state = Buffer(D * s.states); b.scan_ws = Buffer(scan_ws / 4 + 4);
    float *x = Upload(pixels);

    Timer timer;
    double prompt_ms = 0, token_ms = 0;
    for (int i = 0; i <= iterations; i++) {      // the first is not timed
        timer.startBench();
        embedding.Forward(x);
        b.Forward(0, prompt);
        dev.Check(fc_sync(ctx), "fc_sync");
        prompt_ms += i ? timer.endBench(1.0) : 0;
        timer.startBench();
        for (size_t t = prompt; t < tokens; t++) b.Forward(t, 1);
        dev.Check(fc_sync(ctx), "fc_sync");
        token_ms += i ? timer.endBench((double)grid) : 0;
    }
    printf("%zu tokens of %d frames: block up to the prompt of %zu %.3f ms, then %.1f us a token\n", tokens, frames, prompt, prompt_ms / iterations,
           1000.0 * token_ms / iterations);

    // back from a gradient of the normed answers to what goes into norm, scan and convolution
    float *normed = Buffer(tokens * D), *rstd = Buffer(tokens), *dy = Buffer(tokens * D), *du = Buffer(tokens * D), *dshared = Buffer(tokens * M), *dxz = Buffer(tokens * 2 * D);
    float *dA = Buffer(A.size()), *dD = Buffer(D), *dw = Buffer(conv_w.size()), *dgamma = Buffer(D);
    float *conv_ws = Buffer(conv_all.ws_backward_bytes / 4 + 4), *norm_ws = Buffer(norm_all.ws_backward_bytes / 4 + 4);
    const Floats up = Normal(12, tokens * D, 1.0);
    dev.Check(fc_rms_norm(ctx, &norm_all, b.y, NULL, b.gamma_inner, NULL, normed, rstd), "fc_rms_norm");
    dev.Check(fc_rms_norm_backward(ctx, &norm_all, Upload(up), b.y, b.gamma_inner, rstd, NULL, dy, dgamma, norm_ws), "fc_rms_norm_backward");
    dev.Check(fc_selective_scan_backward(ctx, &whole, dy, b.u, b.shared, b.A, b.shared + D, b.shared + D + s.states, b.D, b.xz + D, b.step_bias, du, dshared, dA, dshared + D,
                                         dshared + D + s.states, dD, dxz + D, NULL, NULL, NULL, NULL, NULL, b.scan_ws), "fc_selective_scan_backward");
    dev.Check(fc_causal_conv_backward(ctx, &conv_all, du, b.xz, b.w, b.bias, dxz, dw, NULL, NULL, NULL, NULL, NULL, conv_ws), "fc_causal_conv_backward");
    if (!check) return 0;

    // the same chain in double; each of its 8-bit stages from what the one before left on the device, so that a value on the border between two steps is counted once
    const Doubles tok = Wide(Download(b.tokens, tokens * C)), xz = Wide(Download(b.xz, tokens * 2 * D)), u = Wide(Download(b.u, tokens * D)),
                  shared = Wide(Download(b.shared, tokens * M)), y = Wide(Download(b.y, tokens * D)), back = Wide(Download(b.back, tokens * C));
    const Doubles cw = Wide(conv_w), wide_A = Wide(A), wide_D = Wide(skip);
    Doubles sum(tokens * C);
    for (size_t i = 0; i < sum.size(); i++) sum[i] = (double)(float)(tok[i] + back[i]);
    struct { const char *name; double error, most; } steps[] = {
        // a value in 8 bits that lies on a border goes either way, by a 127th of its row's largest, about 0.024 of the row's root mean square:
        // with one such value in a thousand, and the others exact, 0.024 / sqrt(1000) = 8e-4
        {"tokens", RelativeError(Download(b.tokens, tokens * C), HostProduct(Wide(pixels), Wide(embed), window, C)), 1e-5},
        {"inner channels", RelativeError(Download(b.xz, tokens * 2 * D), HostProduct(Held(HostNorm(tok, gamma, C), C), Held(Wide(w_in), C), C, 2 * D)), 1e-3},
        {"convolution", RelativeError(Download(b.u, tokens * D), HostConv(xz, 2 * D, cw, conv_b, tokens, s)), 1e-5},
        {"steps, B and C", RelativeError(Download(b.shared, tokens * M), HostProduct(Held(u, D), Held(Wide(w_mid), D), D, M)), 1e-3},
        {"scan", RelativeError(Download(b.y, tokens * D), HostScan(u, shared, xz, wide_A, wide_D, step_bias, tokens, s)), 1e-5},
        {"answers", RelativeError(Download(b.back, tokens * C), HostProduct(Held(HostNorm(y, gamma_inner, D), D), Held(Wide(w_out), D), D, C)), 1e-3},
        {"block", RelativeError(Download(b.result, tokens * C), HostNorm(sum, gamma, C)), 1e-5},
    };
    bool good = true;
    for (const auto &step : steps) {
        printf("Relative error of %s against the host: %.3e (tolerance %.0e) %s\n", step.name, step.error, step.most, step.error <= step.most ? "PASS" : "FAIL");
        good = good && step.error <= step.most;
    }

    // the gradients along one direction against a central difference over two steps
    struct Input {
        Doubles at, along;
        Floats gradient;
    } inputs[6] = {{xz, {}, Download(dxz, tokens * 2 * D)}, {shared, {}, Download(dshared, tokens * M)}, {wide_A, {}, Download(dA, A.size())}, {wide_D, {}, Download(dD, D)},
                   {cw, {}, Download(dw, cw.size())}, {Wide(gamma_inner), {}, Download(dgamma, D)}};
    double along = 0, size = 0, diff = 0;
    for (int i = 0; i < 6; i++) {
        // rates of a tenth the size of the others' steps: they are multiplied by up to the length of a memory
        inputs[i].along = Wide(Normal(20 + i, inputs[i].at.size(), i == 2 ? 0.1 : 1.0));
        for (size_t k = 0; k < inputs[i].at.size(); k++) {
            const double term = (double)inputs[i].gradient[k] * inputs[i].along[k];
            along += term;
            size += fabs(term);
        }
    }
    const double e = 1e-4, weights[4] = {1.0 / 12, -8.0 / 12, 8.0 / 12, -1.0 / 12};
    const int at[4] = {-2, -1, 1, 2};
    for (int n = 0; n < 4; n++) {
        Doubles v[6];
        for (int i = 0; i < 6; i++) {
            v[i] = inputs[i].at;
            for (size_t k = 0; k < v[i].size(); k++) v[i][k] += at[n] * e * inputs[i].along[k];
        }
        const Doubles conv = HostConv(v[0], 2 * D, v[4], conv_b, tokens, s), scanned = HostScan(conv, v[1], v[0], v[2], v[3], step_bias, tokens, s);
        const Floats ones(D, 1.f);
        const Doubles answers = HostNorm(scanned, ones, D);
        for (size_t i = 0; i < answers.size(); i++) diff += weights[n] * answers[i] * v[5][i % D] * up[i] / e;
    }
    const double off = fabs(along - diff) / size;
    printf("Gradient along a direction %.6e, central difference %.6e: off %.3e of its terms (tolerance 1e-05) %s\n", along, diff, off, off <= 1e-5 ? "PASS" : "FAIL");
    return good && off <= 1e-5 ? 0 : 2;
}
