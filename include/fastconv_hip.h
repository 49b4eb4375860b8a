/*
 * fastconv_hip.h -- C ABI of the MI355X (gfx950) convolution kernels.
 *
 * This is the boundary the C++ host layers (ConvWinoF63ZCLayer, ConvWinoF63Layer,
 * ConvIm2colLayer) call; it is also what any other binding (ctypes, cgo, JNI)
 * would load.  Plain pointers and sizes only.  Every function returns 0
 * (FC_OK) or a negative fc_status; nothing throws across the boundary.  A
 * context owns one HIP stream; calls on one context are ordered on that stream
 * and must come from one thread at a time.
 *
 * Each entry point names the reference interface it stands in for (paths
 * relative to the reference checkout).
 */
#ifndef FASTCONV_HIP_H_
#define FASTCONV_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    FC_OK = 0,
    FC_ERR_INVALID = -1,      /* bad argument / unsupported shape for this entry point */
    FC_ERR_NO_DEVICE = -2,    /* no usable gfx950 device */
    FC_ERR_HIP = -3,          /* a HIP runtime call failed; see fc_last_error() */
    FC_ERR_OOM = -4,          /* pool exhausted or hipMalloc failed */
    FC_ERR_STATE = -5,        /* call made in the wrong order (e.g. after destroy) */
    FC_ERR_UNSUPPORTED = -6   /* size beyond a stated limit of the kernel */
} fc_status;

typedef struct fc_context fc_context;
typedef struct fc_pool fc_pool;

/* Convolution geometry, fp32 NCHW, group 1.  Field meaning follows the
 * ConvLayer constructor arguments (conv_layer.h:27) plus a batch count. */
typedef struct {
    int N, C, H, W;
    int K, kh, kw;
    int sh, sw;
    int pt, pb, pl, pr;
} fc_conv_shape;

/* Stages whose device time can be read back, labelled as the reference prints
 * them (convLayer/winoF63ConvZC.cpp:249-253, convLayer/im2colConv.cpp:254-256). */
typedef enum {
    FC_STAGE_KERNEL_TRAN = 0,
    FC_STAGE_INPUT_TRAN = 1,
    FC_STAGE_TENSOR_GEMM = 2,
    FC_STAGE_OUTPUT_TRAN = 3,
    FC_STAGE_IMPLICIT_GEMM = 4,
    FC_STAGE_FILTER_PACK = 5,
    FC_STAGE_FUSED_GEMM_OUT = 6,
    FC_STAGE_ONEPASS = 7,
    FC_STAGE_COUNT = 8
} fc_stage;

typedef struct {
    char name[128];
    char arch[32];
    int compute_units;
    int clock_mhz;
    int mem_clock_mhz;
    int mem_bus_bits;
    size_t total_mem;
    int lds_per_block;
} fc_device_info;

/* ---- context ---------------------------------------------------------- */

/* Replaces the implicit process-wide state of the reference (one process,
 * OpenMP threads set in conv_layer.h:31).  Fails with FC_ERR_NO_DEVICE when no
 * GPU is present: there is no CPU fallback. */
int fc_init(int device, fc_context **out);
int fc_destroy(fc_context *ctx);
int fc_get_device_info(fc_context *ctx, fc_device_info *info);
const char *fc_last_error(fc_context *ctx);
const char *fc_status_string(int status);
int fc_sync(fc_context *ctx);

/* ---- memory: one hipMalloc'd arena ------------------------------------ */

/* Stands in for the allocations behind CommonMemPool / PrivateMemPool
 * (utility/mempool.h:23-71) and _mm_malloc (utility/common.cpp:26-40): one
 * device allocation per pool, sub-allocated by bumping a 256-byte aligned
 * offset.  fc_pool_reset() rewinds to empty; fc_pool_mark/release rewind to a
 * saved offset (scratch that lives for one Tuning() candidate). */
int fc_pool_create(fc_context *ctx, size_t bytes, fc_pool **out);
int fc_pool_destroy(fc_pool *pool);
int fc_pool_alloc(fc_pool *pool, size_t bytes, void **dev_ptr);
int fc_pool_reset(fc_pool *pool);
int fc_pool_mark(fc_pool *pool, size_t *mark);
int fc_pool_release(fc_pool *pool, size_t mark);
int fc_pool_stats(fc_pool *pool, size_t *capacity, size_t *used, size_t *peak);

/* Stand in for the memcpy()s into the layer's own buffers (conv_layer.h:74-77). */
int fc_upload(fc_context *ctx, void *dst_dev, const void *src_host, size_t bytes);
int fc_download(fc_context *ctx, void *dst_host, const void *src_dev, size_t bytes);
int fc_fill_zero(fc_context *ctx, void *dst_dev, size_t bytes);
/* Device-to-device copy by a plain kernel (16 bytes per lane): the known-size
 * reference that hardware traffic counters are scaled by.  Both pointers and the
 * size must be multiples of 16. */
int fc_device_copy(fc_context *ctx, void *dst_dev, const void *src_dev, size_t bytes);

/* Synthetic inputs of the drivers, written to HOST memory: n floats uniform in [lo, hi), or
 * normal with standard deviation sigma (Box-Muller in double), from a splitmix64-seeded
 * xoshiro256** stream, so that every machine sees the same layer for a given seed.  Stand in
 * for fillTestInput / fillTestKernel (ConvTest.cpp:18-46), which draw from rand(). */
int fc_host_fill_uniform(uint64_t seed, float lo, float hi, float *dst_host, size_t n);
int fc_host_fill_normal(uint64_t seed, float sigma, float *dst_host, size_t n);

/* ---- stage timing (utility/helper.h:66-80 Timer, per stage) ----------- */

/* stage_mask has bit (1 << stage) set for every stage whose kernel launches are
 * to be bracketed by two events on the context's stream (FC_TIMING_ALL for all,
 * 0 to switch timing off).  fc_stage_time_ms() waits for the stream, folds the
 * pending event pairs into per-stage totals and returns total milliseconds and
 * launch count since the last fc_timing_reset(). */
#define FC_TIMING_ALL 0xff
int fc_timing_enable(fc_context *ctx, int stage_mask);
int fc_timing_reset(fc_context *ctx);
int fc_stage_time_ms(fc_context *ctx, int stage, double *total_ms, long *launches);

/* Shader clock under load.  The published MFMA peak is quoted at the maximum shader clock
 * (2400 MHz on MI355X); under fp32 MFMA load with real data the chip's power management runs
 * the shaders slower, and the clock it sustains is what bounds the products.
 * fc_clock_probe_begin starts a one-wavefront kernel on a stream of its own that, `samples`
 * times (1..256), waits `sample_us` microseconds (1..100000) on the constant 100 MHz counter and
 * records how far the shader-clock counter moved meanwhile; work enqueued through this context
 * afterwards runs beside it.  fc_clock_probe_end waits for the probe and returns the shader
 * clock of every sample in MHz (at most `capacity` of them; *n_samples = how many were taken).
 * One probe at a time per context; not while a graph is being recorded.  No counterpart in the
 * reference, whose Timer (utility/helper.cpp:113-148) sees wall time only. */
int fc_clock_probe_begin(fc_context *ctx, int samples, int sample_us);
int fc_clock_probe_end(fc_context *ctx, double *mhz, int capacity, int *n_samples);

/* ---- Winograd F(6x6,3x3), stride 1 ------------------------------------ */

/* Tile shapes of the batched GEMM stage.  The reference tunes
 * ocBlock/tileBlock/icBlock and a 4x4 or 4x5 register kernel
 * (convLayer/winoF63ConvZC.cpp:25-174); here a configuration is a workgroup
 * tile BM (output channels) x BN (tiles) x BK (input channels) and a wave grid
 * (waves_m x waves_n wavefronts side by side over the tile, times waves_k
 * wavefronts that each take a share of the reduction).  lds_bytes and the wave grid are
 * those of the kernel that runs on fp32 matrix instructions; where a plan's products are
 * split (fc_wino_gemm_splits_products, fc_igemm_splits_products) a tile takes
 * 192 * (bm + bn) bytes of LDS, up to 72 KB, and the 128x128 one eight wavefronts. */
typedef struct {
    int id;
    int bm, bn, bk;
    int waves_m, waves_n;
    int lds_bytes;
    int waves_k;              /* wavefronts of a workgroup that split the reduction among themselves (1: no split) */
} fc_gemm_config;

int fc_wino_gemm_num_configs(void);
int fc_wino_gemm_get_config(int id, fc_gemm_config *cfg);
/* Tile shape to use when a layer has not been tuned (the role of the defaults
 * ocBlock=140, tileBlock=52, icBlock=64 in convLayer/winoF63ConvZC.cpp:11-16):
 * the shape with the least padded work, discounted for narrow tiles and for
 * grids that leave compute units idle.  Returns a configuration id. */
int fc_wino_gemm_default_config(const fc_conv_shape *shape);

/* Buffer geometry for one layer under one GEMM configuration.  Frequencies
 * f = 8*row + col of the transformed 8x8 tile; tiles t = (n*tiles_h + th)*tiles_w + tw.
 *   U[64][C_pad][K_pad]   transformed filters, output channel fastest
 *   V[64][C_pad][T_pad]   transformed input tiles, tile fastest
 *   M[64][K_pad][T_pad]   per-frequency products, tile fastest
 * Padding (to the GEMM tile) is written as zeros by the transforms.
 * Stands in for the buffer sizing in ConvWinoF63ZCLayer::Init
 * (convLayer/winoF63ConvZC.cpp:176-213). */
typedef struct {
    fc_conv_shape shape;
    int OH, OW;
    int tiles_h, tiles_w;
    long T;
    int K_pad, C_pad;
    long T_pad;
    int gemm_config;
    size_t U_bytes, V_bytes, M_bytes;
} fc_wino_plan;

/* FC_ERR_INVALID unless the layer is 3x3 with stride 1; FC_ERR_UNSUPPORTED when the output is
 * wider than 1020 columns (170 tiles: two bands of the input transform must fit 64 KiB of LDS)
 * or a buffer would pass 2^31 elements per frequency plane.  Every later call checks the plan it
 * is given against the one this function makes for plan->shape and plan->gemm_config. */
int fc_wino_make_plan(const fc_conv_shape *shape, int gemm_config, fc_wino_plan *plan);

/* The rule behind `-a auto` for one layer (select_algorithm, ConvTest.cpp:318-331, which looks at
 * filter size and stride only): 1 when the Winograd path is expected to be faster than the
 * implicit GEMM on MI355X, 0 when not or when Winograd cannot run the layer at all (not 3x3
 * stride 1, or wider than fc_wino_make_plan admits).  The thresholds come from measured
 * per-layer times of both paths on the VGG-16 and ResNet-50 layers at batch 1 and 32. */
int fc_prefer_winograd(const fc_conv_shape *shape);

/* U = G g G^T.  Replaces the kernel transform inside winoF63_v1_single
 * (winoF63ZC/winoF63ZC.cpp:433-500) and offline_kernel_transform_v1 (:242-322).
 * w is K x C x 3 x 3. */
int fc_wino_filter_transform(fc_context *ctx, const fc_wino_plan *plan,
                             const float *w_dev, float *U_dev);

/* V = B^T d B with zero-filled borders.  Replaces the input transform inside
 * winoF63_v1_single (winoF63ZC/winoF63ZC.cpp:512-813). */
int fc_wino_input_transform(fc_context *ctx, const fc_wino_plan *plan,
                            const float *x_dev, float *V_dev);

/* Both transforms above in one launch (the filter transform of a layer is a short kernel;
 * launched by itself it costs a launch and a drain of the chip per layer).  What the online
 * strategy of winoF63_v1_single does back to back (winoF63ZC/winoF63ZC.cpp:433-813).  Its
 * time is booked under FC_STAGE_INPUT_TRAN. */
int fc_wino_filter_input_transform(fc_context *ctx, const fc_wino_plan *plan,
                                   const float *w_dev, float *U_dev,
                                   const float *x_dev, float *V_dev);

/* M[f] = U[f]^T-layout product over input channels for all 64 frequencies in
 * one launch, at fp32 accuracy: on fp32 MFMA, or, where that is faster, as six products
 * of three bf16 parts of each operand, which add up to it exactly.  Replaces the depth x oc x tile loop nest calling
 * TensorGEMMInnerKernel4x4x4_v3 (winoF63ZC/winoF63ZC.cpp:818-860,
 * winoF63ZC/TensorGEMMZC.cpp:443-583).  M is overwritten, never accumulated. */
int fc_wino_gemm(fc_context *ctx, const fc_wino_plan *plan,
                 const float *U_dev, const float *V_dev, float *M_dev);
/* 1 when the products of this plan are formed from bf16 parts (above; fc_wino_gemm_output_fused
 * does as fc_wino_gemm, so that the two give the same bits for one plan), else 0.  The error of such a sum
 * against 64 bits is 0.3 to 0.7 of the fp32 instructions', 1.03 where a single term is not zero;
 * one plan always rounds alike, but plans of one layer with other batches or tiles may not.
 * Values that are not finite, and sums from 2^80 on, are formed on fp32 MFMA in a second pass. */
int fc_wino_gemm_splits_products(const fc_wino_plan *plan);

/* The same stage fed by the untransformed filter w[K][C][3][3]: U = G g G^T is formed
 * in registers, lane by lane in the layout the MFMA takes its first operand in, and never
 * exists in memory.  For layers with few tiles (batch 1 on 7x7 to 28x28 images), where
 * the stage above is one pass over U, 64/9 times the size of w.  Like the reference's
 * online strategy (kernel transform inside Forward, ConvTest.cpp:230-243) without its
 * kernelBuf.  Needs plan->T <= 64 and C a multiple of 16
 * (fc_wino_raw_filter_gemm_applies); freqs_per_wave = 0 lets the library choose how many
 * of the 64 frequencies a wavefront multiplies (1, 2 or 4) and channel_split = 0 over how
 * many groups of wavefronts a workgroup spreads the input channels (1, 2 or 4): tuning
 * parameters like the tile shape of fc_wino_gemm.  M is overwritten: rows K up to K rounded
 * up to 16 are written as zeros and columns T up to T rounded up to 16, 32 or 64 hold the
 * products of V's (zero) padding; rows and columns beyond that, up to K_pad and T_pad, are
 * left as they were.  The output transform reads none of the padding. */
int fc_wino_gemm_raw_filter(fc_context *ctx, const fc_wino_plan *plan,
                            const float *w_dev, const float *V_dev, float *M_dev,
                            int freqs_per_wave, int channel_split);
int fc_wino_raw_filter_gemm_applies(const fc_wino_plan *plan);
/* 1 when fc_wino_gemm_raw_filter is expected to beat filter transform + fc_wino_gemm
 * (measured on MI355X: at most 32 tiles and C*K >= 32768).  Against fc_wino_gemm alone,
 * with the filter transformed beforehand, the two are level. */
int fc_wino_prefer_raw_filter_gemm(const fc_wino_plan *plan);

/* Y = A^T m A clipped to the image, written NCHW, with an optional per-channel
 * bias (K floats) and optional ReLU.  Replaces the output transform inside
 * winoF63_v1_single (winoF63ZC/winoF63ZC.cpp:869-973). */
int fc_wino_output_transform(fc_context *ctx, const fc_wino_plan *plan,
                             const float *M_dev, const float *bias_dev, int relu,
                             float *y_dev);

/* GEMM and output transform in one kernel: the 64 per-frequency products of a
 * block of (32 output channels x 32 tiles) stay in registers and LDS, M is never
 * written (M_dev is not needed).  The counterpart of the reference's blocked
 * pipeline, where the GEMM result of one block is consumed by the output
 * transform out of block-local scratch (winoF63/winoF63.cpp:1574-1737).  Pays
 * when the transformed filter fits in L2 (C*K up to about 8192); any plan whose
 * C_pad is a multiple of 8 is accepted. */
int fc_wino_gemm_output_fused(fc_context *ctx, const fc_wino_plan *plan,
                              const float *U_dev, const float *V_dev,
                              const float *bias_dev, int relu, float *y_dev);

/* 1 when the fused kernel is expected to beat fc_wino_gemm + fc_wino_output_transform
 * for this layer (measured on MI355X: when the transformed filter, 256*C*K bytes,
 * stays L2-resident, C*K <= 8192, and the layer brings at least 512 blocks of 32 tiles x 32
 * output channels or has at most 8 input channels), else 0. */
int fc_wino_prefer_fused(const fc_conv_shape *shape);

/* Filter transform (unless filter_ready), input transform, fused GEMM + output
 * transform: the whole layer without an M buffer. */
int fc_wino_forward_fused(fc_context *ctx, const fc_wino_plan *plan, const float *x_dev,
                          const float *w_dev, const float *bias_dev, int relu, int filter_ready,
                          float *U_dev, float *V_dev, float *y_dev);

/* ---- the whole layer in one kernel ------------------------------------ */

/* gemm_config value of a plan made by fc_wino_make_onepass_plan. */
#define FC_WINO_ONEPASS (-1)

/* Plan for the single-kernel path: input transform, the 64 products and the output
 * transform inside one workgroup per (16 tiles x 64 output channels), so neither V nor M
 * exists (V_bytes = M_bytes = 0).  K_pad is K rounded up to 64, C_pad is C rounded up to 8.
 * The transformed filter uses its own layout, U4[64][C_pad/4][K_pad/64][4][16][4] (channel
 * 4q + c, output channel 64kb + 16sb + k at [f][q][kb][c][k][sb]); only
 * fc_wino_onepass_filter_transform writes it and
 * only fc_wino_conv_onepass reads it.  The stage calls above reject such a plan.
 * Images narrower than 8 columns are not supported (FC_ERR_UNSUPPORTED): use the staged calls.
 * Layers with at most four input channels (and an input of at most 2 GiB) run through a kernel
 * of their own on the vector ALUs behind the same three calls (the products are too few for the
 * matrix cores to matter and the layer is bound by the stores of y); their transformed filter
 * is laid out [K_pad][8][8][4] in the same buffer.
 * The GPU reading of the reference's blocked pipeline taken to its end: there one block of
 * tiles goes through input transform, TensorGEMM and output transform out of block-local
 * scratch (winoF63/winoF63.cpp:1574-1737); here the block-local scratch is LDS and registers. */
int fc_wino_make_onepass_plan(const fc_conv_shape *shape, fc_wino_plan *plan);

/* U4 = G g G^T in the layout above (offlineKernelTransform, winoF63/winoF63.cpp:846-973). */
int fc_wino_onepass_filter_transform(fc_context *ctx, const fc_wino_plan *plan,
                                     const float *w_dev, float *U_dev);

/* y = conv(x) (+bias, ReLU) from x and U4 in one launch. */
int fc_wino_conv_onepass(fc_context *ctx, const fc_wino_plan *plan, const float *x_dev,
                         const float *U_dev, const float *bias_dev, int relu, float *y_dev);

/* Filter transform (unless filter_ready) + fc_wino_conv_onepass.  U_dev holds the transformed filter
 * afterwards either way; for a layer with at most four input channels and few tiles the two run as one
 * launch (the convolution kernel transforms the filter itself and writes U_dev as a by-product, equal to
 * fc_wino_onepass_filter_transform's to the last bit or two). */
int fc_wino_forward_onepass(fc_context *ctx, const fc_wino_plan *plan, const float *x_dev,
                            const float *w_dev, const float *bias_dev, int relu, int filter_ready,
                            float *U_dev, float *y_dev);

/* 1 when the single-kernel path is expected to be the fastest Winograd pipeline for this
 * layer (measured on MI355X: 16 to 64 input channels, where the products are cheap next to
 * moving V and M through HBM, the image at least 8 columns wide, and at least 512 blocks of
 * 16 tiles x 64 output channels -- 192 when one block covers all output channels -- i.e. not
 * at batch 1, and V and M too large for the staged pipeline to be faster, from 3.5 MB per input
 * channel on, 10 MB where C*K > 8192; layers that the staged pipeline does not take; and every
 * layer with at most four input channels, at any batch), else 0.  A layer for which it is 0
 * runs fastest with V and, unless fc_wino_prefer_fused is 1, M in memory: up to 640 MB for the
 * two (fc_wino_make_plan gives the sizes).  Where there is no room for them the single kernel
 * still takes the layer if fc_wino_make_onepass_plan does. */
int fc_wino_prefer_onepass(const fc_conv_shape *shape);

/* 1 when the single-kernel path is expected to be faster than fc_wino_forward_fused, the choice
 * of a caller with these two ways only (the blocked layer class, which has no M), else 0. */
int fc_wino_prefer_onepass_to_fused(const fc_conv_shape *shape);

/* All stages back to back: what winoF63_v1_single (winoF63ZC/winoF63ZC.h:5-6)
 * does in one call.  filter_ready != 0 skips the filter transform (U already
 * holds it: the "offline" strategy, ConvTest.cpp:230-243).  With filter_ready == 0
 * the contents of U after the call are unspecified: a layer with few tiles
 * (fc_wino_prefer_raw_filter_gemm) multiplies straight from w and leaves U alone. */
int fc_wino_forward(fc_context *ctx, const fc_wino_plan *plan, const float *x_dev,
                    const float *w_dev, const float *bias_dev, int relu, int filter_ready,
                    float *U_dev, float *V_dev, float *M_dev, float *y_dev);

/* ---- implicit GEMM (replaces im2col + pack + GEMM) -------------------- */

int fc_igemm_num_configs(void);
int fc_igemm_get_config(int id, fc_gemm_config *cfg);
/* Where products are split (fc_igemm_splits_products) the tiles of 256x128, 128x256 and 64x256 run as
 * 128x128, 128x128 and 64x128, and plans are made for those. */
/* Untuned choice, as above (the role of mc=8, nc=256, kc=384 in
 * convLayer/im2colConv.h:17-18). */
int fc_igemm_default_config(const fc_conv_shape *shape);

/* Filter re-layout done once at Init: Wp[Kred_pad][K_pad], output channel
 * fastest, plus the per-row gather table; where products are split the filter
 * follows a second time as operand words of its three bf16 parts, 10 bytes an
 * element together (Wp_bytes says how many there are).  The order of the
 * reduction rows and the rows added to it are the library's business and depend
 * on plan->config: the column matrix's (c, r, s) (convLayer/im2colConv.cpp:285-309)
 * or tap-major (r, s, c) on fp32 instructions, blocks of 16 channels or window
 * rows in runs of 8 or 4 columns, both padded to whole ones, on split products.
 * Treat Wp and the table as opaque, hand them only to calls made with the same
 * plan, and pack them again when the configuration changes. */
typedef struct {
    fc_conv_shape shape;
    int OH, OW;
    int Kred, Kred_pad, K_pad;
    long Npix;
    int config;
    size_t Wp_bytes, table_bytes;
    int split_k;              /* > 1: the reduction is split over this many workgroups per tile */
    size_t ws_bytes;          /* workspace for the partial sums ([split_k][K][Npix] floats), 0 if unsplit */
} fc_igemm_plan;

int fc_igemm_make_plan(const fc_conv_shape *shape, int config, fc_igemm_plan *plan);
/* As fc_wino_gemm_splits_products: 1 where fc_igemm_pack_filter splits the filter.  (Some layers of short
 * reductions, and pointwise ones of 33 to 64 output channels, keep their filter in fp32 and split it in the kernel;
 * their results are no less exact.)  Without room for the filter of split products, the configurations for which
 * this is 0 (32x64, and those with waves_k above 1) keep it in fp32 alone. */
int fc_igemm_splits_products(const fc_igemm_plan *plan);
/* 1 when the products of this plan are formed on the bf16 matrix cores, whether its filter is split when it is packed or in
 * the kernel: the peak that a measured rate is a fraction of. */
int fc_igemm_on_bf16(const fc_igemm_plan *plan);
/* Name of the kernel that runs this plan, as a profiler shows it; "" for a plan that was not made. */
const char *fc_igemm_kernel_name(const fc_igemm_plan *plan);

/* Replaces pack_a_v2 (im2col/gemm_pack.cpp:192-260) as a one-time step. */
int fc_igemm_pack_filter(fc_context *ctx, const fc_igemm_plan *plan, const float *w_dev,
                         float *Wp_dev, int32_t *table_dev);

/* y[n][k][oh][ow] = sum_{c,r,s} w[k][c][r][s] * x[n][c][oh*sh+r-pt][ow*sw+s-pl].
 * Replaces ConvIm2colLayer::im2col_v1 + sgemm (convLayer/im2colConv.cpp:311-398,
 * 434-565) and the register kernels of im2col/gemm_kernel.cpp; the column matrix
 * is never materialised and y is overwritten (not accumulated).  Layers too small
 * to fill the GPU have plan->split_k > 1: the reduction is cut into parts whose
 * partial sums go to ws_dev (plan->ws_bytes) and are added in a fixed order by a
 * second small kernel; ws_dev may be NULL when plan->ws_bytes is 0. */
int fc_conv_implicit_gemm(fc_context *ctx, const fc_igemm_plan *plan, const float *x_dev,
                          const float *Wp_dev, const int32_t *table_dev,
                          const float *bias_dev, int relu, float *ws_dev, float *y_dev);

/* The same layer for callers that cannot allocate device memory (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc): no counterpart in the reference.  The
 * partial sums of a split reduction go to a static device array of FC_IGEMM_STATIC_WS_BYTES
 * inside the library instead of a workspace of the caller's (each GPU the library runs on holds
 * that array until the process ends); the call allocates nothing and is never bracketed by
 * timing events.  A plan whose ws_bytes exceeds FC_IGEMM_STATIC_WS_BYTES is refused with
 * FC_ERR_UNSUPPORTED, but for the plan of fc_igemm_default_config, which then runs in as many
 * parts as the array holds (one if need be): its result is that of fc_conv_implicit_gemm up to
 * the order of the sums.  All calls on one GPU share the array and calls that overlapped in time
 * would race, so one context per GPU uses it at a time: the first context to make this call on a
 * GPU owns the array until fc_destroy, and the call is refused for any other context meanwhile
 * (FC_ERR_STATE); calls of one context are ordered on its stream and safe.  Other processes have
 * their own copy of the array. */
#define FC_IGEMM_STATIC_WS_BYTES (32 << 20)
int fc_conv_implicit_gemm_static(fc_context *ctx, const fc_igemm_plan *plan, const float *x_dev,
                                 const float *Wp_dev, const int32_t *table_dev,
                                 const float *bias_dev, int relu, float *y_dev);

/* ---- recorded launch sequences ----------------------------------------- */

/* Records every launch made on the context between fc_graph_begin and fc_graph_end into a
 * graph that fc_graph_launch replays with one call: for stacks of layers whose kernels are
 * so short that launching them one by one is what takes the time (batch 1).  No counterpart
 * in the reference.  While recording, nothing runs; fc_upload, fc_download, fc_sync and
 * stage timing are refused (FC_ERR_STATE), and the fused and single-kernel Winograd calls
 * must have run once on the context before.  The replay reads and writes the same device
 * buffers as the recorded calls.  fc_graph_destroy waits for the stream first. */
typedef struct fc_graph fc_graph;
int fc_graph_begin(fc_context *ctx);
int fc_graph_end(fc_context *ctx, fc_graph **graph);
int fc_graph_launch(fc_context *ctx, fc_graph *graph);
int fc_graph_destroy(fc_graph *graph);

/* ---- glue for running layers back to back ---------------------------- */

/* 2x2 max pooling, stride 2, NCHW, floor((H)/2) x floor((W)/2) output: the step between
 * the convolution blocks of a VGG-style stack.  No counterpart in the reference (it has
 * no layer but convolution); it exists so that a whole conv trunk can run on the device
 * without host round trips (the layer graph of layer.h:29-84). */
int fc_maxpool2x2(fc_context *ctx, const float *x_dev, float *y_dev, int N, int C, int H, int W);

/* ---- operators on tokens, channels last -------------------------------- */

/* What a network runs on the pixels of a convolution trunk, or on the patches of a patch embedding, once they are tokens:
 * channels last, so that a token's channels are neighbours.  No counterpart in the reference, which ends at the
 * convolution.  The convolutions' fp32 NCHW output has this layout as it is where images have one pixel (N tokens of
 * C x 1 x 1: a patch embedding, the projections of tokens); larger images, and 16-bit tensors, are the caller's to lay out.
 *
 * Tensors hold fp32, bf16 or IEEE half (fc_dtype); every sum, statistic, state and angle is held in fp32 or wider, and a
 * result is rounded once to the tensor's type.  Two things have fewer bits on their way into a result of 16 bits: GELU's erf is
 * good to 1.5e-7, and linear attention of more than six tokens multiplies q k^T and the state as 16 bits of each (bf16 products, added up in
 * fp32; fp32 tensors have 24 bits of everything there, and every state takes in 24 bits of what is added to it).  Parameters (gamma, beta, log_decay, inv_freq), statistics and states are fp32 always.
 * Strides are in elements; channels of one token (one head) are neighbours.  Pointers need the alignment of their type only:
 * rows that begin on 16 bytes and have sizes that are multiples of 16 bytes are read fastest.  Buffers must not overlap, but
 * where a call says so.  An input may be shared along an axis (stride 0); the rows of an output may not, and a gradient has the strides of
 * what it is the gradient of: FC_ERR_INVALID.  All calls run on the context's stream, allocate nothing and can be recorded into a graph; they are not
 * stages and are never bracketed by timing events.  Sizes that are refused: FC_ERR_INVALID for what no such operator has,
 * FC_ERR_UNSUPPORTED beyond the limits stated here. */
typedef enum { FC_F32 = 0, FC_BF16 = 1, FC_F16 = 2 } fc_dtype;
typedef enum { FC_ACT_NONE = 0, FC_ACT_RELU = 1, FC_ACT_SILU = 2, FC_ACT_GELU = 3 /* with erf */ } fc_activation;

/* Group norm with an activation.  x is N images of P pixels with C channels in G groups of C/G neighbours:
 *   xhat = (x - mean) * rstd over the P*C/G values of a group,  rstd = 1/sqrt(variance + eps)
 *   y = act(gamma * xhat + beta)
 * Pixel p of image n begins at n*x_image + p*x_pixel; y (and dy) likewise, dx as x.  G == 1 is a layer norm over whole images,
 * G == C an instance norm.  Limits: C/G <= 4096, N*C < 2^31, and fewer than 2^24 - C/8 workgroups, of which an image has one for every
 * `span` channels (of the plan: up to 4096, whole groups): about 2^24 images of up to 4096 channels, half as many of 8192. */
typedef struct {
    int N;
    long P;
    int C, G;
    int dtype, act;
    float eps;
    long x_image, x_pixel, y_image, y_pixel;
} fc_group_norm_shape;

typedef struct {
    fc_group_norm_shape shape;
    int span;                 /* channels that one workgroup reads of a pixel: whole groups */
    int chunks;               /* parts that the pixels of an image are cut into */
    int resident;             /* channels whose groups stay in a workgroup's registers, so that x is read once; 0: they do */
    int resident_backward;    /* not fit, and x is read twice, as it is by a call whose tensors do not begin on 16 bytes */
    size_t ws_bytes;          /* workspace of the forward call, 0 if none */
    size_t ws_backward_bytes; /* and of the backward call */
} fc_group_norm_plan;

int fc_group_norm_make_plan(const fc_group_norm_shape *shape, fc_group_norm_plan *plan);

/* gamma and beta: C floats, or NULL for ones and zeros.  mean and rstd: N*G floats for the backward pass, or both NULL.
 * y may be x where their strides are equal.  The variance is formed from differences to running means, so that a mean many
 * times the deviation costs no accuracy. */
int fc_group_norm(fc_context *ctx, const fc_group_norm_plan *plan, const void *x_dev, const float *gamma_dev,
                  const float *beta_dev, void *y_dev, float *mean_dev, float *rstd_dev, void *ws_dev);

/* Gradients of x (in the tensor's type), gamma and beta (fp32, overwritten; each may be NULL) from that of y.  mean and rstd are the
 * forward call's.  Sums run in a fixed order: the same call gives the same bits.  ReLU's slope at 0 is 0. */
int fc_group_norm_backward(fc_context *ctx, const fc_group_norm_plan *plan, const void *dy_dev, const void *x_dev,
                           const float *gamma_dev, const float *beta_dev, const float *mean_dev, const float *rstd_dev,
                           void *dx_dev, float *dgamma_dev, float *dbeta_dev, void *ws_dev);

/* Rotary positions with up to FC_ROTARY_AXES axes (time, height, width): pair j of a head is turned by the angle
 * position[axis of j] * inv_freq[j]:  (a, b) -> (a cos - b sin, b cos + a sin).  The first pairs[0] pairs belong to axis 0, the
 * next pairs[1] to axis 1, and so on; with R pairs in all, pair j is channels j and j + R, or 2j and 2j + 1 if `interleaved`.
 * Channels from 2R on pass unchanged.  positions: int32 [B][T][axes], those of sequence b at b*positions_batch (0: the same
 * ones for all); any int32 is a position, and the angle is reduced in 64 bits.  q has Hq heads and k Hk (0: no k).
 * Token t of sequence b and head h begins at b*q_batch + t*q_token + h*q_head, and so for k and both outputs.
 * Limits: D <= 1024, Hq + Hk <= 65536, at most 2^25 - 2 tokens in all. */
#define FC_ROTARY_AXES 4
typedef struct {
    int B;
    long T;
    int Hq, Hk, D;
    int axes;
    int pairs[FC_ROTARY_AXES];
    int interleaved;
    int dtype;
    long positions_batch;
    long q_batch, q_token, q_head;
    long k_batch, k_token, k_head;
    long qo_batch, qo_token, qo_head;
    long ko_batch, ko_token, ko_head;
} fc_rotary_shape;

/* inverse != 0 turns the other way: the backward pass (gradients in, gradients out).  q_out may be q and k_out may be k where
 * the strides are equal.  One launch for both, one token or many. */
int fc_rotary(fc_context *ctx, const fc_rotary_shape *shape, const void *q_dev, const void *k_dev, const int32_t *positions_dev,
              const float *inv_freq_dev, int inverse, void *q_out_dev, void *k_out_dev);

/* Linear attention with a decay for each head.  Head h has a state S of Dk x Dv floats that takes in a token at a time:
 *   S_t = decay S_(t-1) + k_t v_t^T,   o_t = scale * S_t^T q_t,   decay = exp(log_decay[h]) in [0, 1]
 * H query heads share Hkv key/value heads (H a multiple of Hkv; head h reads key/value head h / (H/Hkv)); every query head has
 * its own decay and state.  Token t of sequence b and head h begins at b*q_batch + t*q_token + h*q_head, and so for k, v and o
 * (gradients: as what they are gradients of).  States are packed [B][H][Dk][Dv].  log_decay above 0 is not checked for (the state
 * grows); minus infinity is a decay of 0, a token that sees itself alone.
 * lengths: B int32, or NULL when every sequence has T tokens; sequence b then ends after min(max(lengths[b], 0), T) of them: its later
 * tokens are not read, their outputs and gradients are zeros, and a state passes an empty sequence unchanged.
 * A value that is not finite reaches no token before its own; in v it makes its channel of the state NaN from then on.
 * Limits: Dk, Dv <= 256, B*H < 2^21, T < 2^31. */
typedef struct {
    int B;
    long T;
    int H, Hkv, Dk, Dv;
    int dtype;
    float scale;
    long q_batch, q_token, q_head;
    long k_batch, k_token, k_head;
    long v_batch, v_token, v_head;
    long o_batch, o_token, o_head;
} fc_linear_attention_shape;

typedef struct {
    fc_linear_attention_shape shape;
    int chunk;                /* tokens that are taken in together; 0: the recurrence, a token at a time */
    int segments;             /* parts of a sequence that run side by side, joined by their states */
    size_t ws_bytes;          /* workspace of the forward call, 0 if none */
    size_t ws_backward_bytes; /* and of the backward call */
} fc_linear_attention_plan;

int fc_linear_attention_make_plan(const fc_linear_attention_shape *shape, fc_linear_attention_plan *plan);

/* state_in: the state before the first token (NULL: zeros).  state_out: the state after the last one (NULL: not wanted); may be
 * state_in.  A prompt runs in chunks on the matrix cores, a few tokens through the recurrence: the same call serves both. */
int fc_linear_attention(fc_context *ctx, const fc_linear_attention_plan *plan, const void *q_dev, const void *k_dev,
                        const void *v_dev, const float *log_decay_dev, void *o_dev, const float *state_in_dev,
                        float *state_out_dev, const int32_t *lengths_dev, void *ws_dev);

/* Gradients of q, k, v and state_in (dstate_in; NULL: not wanted) from those of o and state_out (dstate_out; NULL: none).  The
 * decays are constants of the model and have no gradient.  Gradients of a shared key/value head are summed over its query
 * heads in a fixed order. */
int fc_linear_attention_backward(fc_context *ctx, const fc_linear_attention_plan *plan, const void *do_dev, const void *q_dev,
                                 const void *k_dev, const void *v_dev, const float *log_decay_dev, void *dq_dev, void *dk_dev,
                                 void *dv_dev, const float *state_in_dev, const float *dstate_out_dev, float *dstate_in_dev,
                                 const int32_t *lengths_dev, void *ws_dev);

/* RMS norm over rows of channels, after the addition of a residual:
 *   h = x + residual, rounded to the tensors' type;   rstd = 1/sqrt(mean of h^2 + eps);   y = h * rstd * gamma
 * Row i of x begins at i*x_row, and so for the residual, the sum h and y (in 8 bits: strides of bytes); dy as y, dsum as the sum, dx as x.  A row whose
 * squares overflow fp32 is normed like any other.  One whose root is below 2^-128 (subnormal rows, no eps) is too, but its rstd is infinite and its gradients are
 * no numbers.  Limits: C <= 2^20, rows <= 2^40. */
typedef struct {
    long rows;
    int C;
    int dtype;
    float eps;
    long x_row, residual_row, sum_row, y_row;
} fc_rms_norm_shape;

typedef struct {
    fc_rms_norm_shape shape;
    int parts;                /* sums of dgamma that are formed side by side */
    size_t ws_backward_bytes; /* workspace of the backward call, for dgamma */
} fc_rms_norm_plan;

int fc_rms_norm_make_plan(const fc_rms_norm_shape *shape, fc_rms_norm_plan *plan);

/* residual and gamma (C floats): or NULL for none and ones.  sum: h, or NULL if not wanted; may be x or the residual where their strides are equal.
 * y may be x or the residual likewise, if the sum is another.  rstd: a float a row for the backward pass, or NULL. */
int fc_rms_norm(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x_dev, const void *residual_dev, const float *gamma_dev,
                void *sum_dev, void *y_dev, float *rstd_dev);

/* The same in 8 bits with a scale for each row: scale = max |y| / 127, q = y / scale rounded to nearest, ties to even.  y is in fp32 here, whatever the
 * tensors' type, and every product and quotient is one fp32 operation: fc_quantize_rows makes the same bits of the same rows of y.  A row whose largest value
 * is below 2^-110 is zeros with a scale of 0; one with a value that is not finite is zeros with a scale of NaN, so that a product of it is NaN. */
int fc_rms_norm_int8(fc_context *ctx, const fc_rms_norm_plan *plan, const void *x_dev, const void *residual_dev, const float *gamma_dev,
                     void *sum_dev, int8_t *q_dev, float *scale_dev);

/* Gradient of x, which is that of the residual too (dx), and of gamma (fp32, overwritten; NULL: not wanted, and no workspace) from that of y and, where h
 * is read elsewhere as well, of the sum (dsum; NULL: none).  sum: h of the forward call (x itself if there was no residual, with sum_row == x_row).
 * dx may be dsum where sum_row == x_row, or dy where y_row == x_row.  Sums run in a fixed order. */
int fc_rms_norm_backward(fc_context *ctx, const fc_rms_norm_plan *plan, const void *dy_dev, const void *sum_dev, const float *gamma_dev,
                         const float *rstd_dev, const void *dsum_dev, void *dx_dev, float *dgamma_dev, void *ws_dev);

/* Rows in 8 bits as above, without a norm: activations on their way into a product, or its matrix (a row for each output channel) once. */
int fc_quantize_rows(fc_context *ctx, long rows, int C, int dtype, const void *x_dev, long x_row, int8_t *q_dev, long q_row, float *scale_dev);

/* Product of 8-bit rows with scales for each token and channel:
 *   y[m][n] = (sum over k of x[m][k] w[n][k]) * x_scale[m] * w_scale[n] + bias[n]
 * Rows of x, w (bytes) and y (of `dtype`) begin x_row, w_row and y_row apart; w holds a row for each output channel.  Sums are exact, in 32-bit integers.
 * Rows of x and w that begin on 16 bytes and have sizes that are multiples of 16 are read fastest.  Limits: K <= 131071, M < 2^31, M*N < 2^36,
 * and fewer than 2^24 tiles of 64 or 128 tokens and channels (2^23 of 256; 2^23 workgroups of up to 32 channels where tokens are few). */
typedef struct {
    long M;
    int N, K;
    int dtype;
    long x_row, w_row, y_row;
} fc_int8_product_shape;

typedef struct {
    fc_int8_product_shape shape;
    int tile;                 /* tokens and channels that a workgroup takes; 0: few tokens, w read straight into registers */
    int parts;                /* of the reduction, summed up afterwards */
    size_t ws_bytes;          /* workspace, 0 if none */
} fc_int8_product_plan;

int fc_int8_product_make_plan(const fc_int8_product_shape *shape, fc_int8_product_plan *plan);

/* bias: N floats or NULL. */
int fc_int8_product(fc_context *ctx, const fc_int8_product_plan *plan, const int8_t *x_dev, const float *x_scale_dev, const int8_t *w_dev,
                    const float *w_scale_dev, const float *bias_dev, void *y_dev, void *ws_dev);

/* What the calls below write shares nothing: answers or gradients of which two tokens, sequences or groups have an element in common are refused.  Inputs may lie
 * anyhow.
 *
 * Short causal convolution of each channel over the tokens of a sequence, with its activation (FC_ACT_NONE or FC_ACT_SILU):
 *   y_t = act(bias + sum over j < taps of w[c][j] x_(t - taps + 1 + j))
 * Token t of sequence b begins at b*x_batch + t*x_token, and so for y; dy as y, dx as x.  w is fp32 [C][taps], the last tap the token's own.  The inputs before
 * the first token are a state of taps - 1 rows, packed [B][taps - 1][C] in the tensors' type, the oldest first.
 * lengths as above: later tokens are not read, their outputs and gradients are zeros, and the state after a sequence holds its own last rows.
 * Limits: 2 <= taps <= 8, C <= 2^23, B*C < 2^30, T <= 2^30. */
typedef struct {
    int B;
    long T;
    int C, taps;
    int dtype, act;
    long x_batch, x_token, y_batch, y_token;
} fc_causal_conv_shape;

typedef struct {
    fc_causal_conv_shape shape;
    int walks, walks_backward; /* parts of a sequence that threads walk over side by side */
    size_t ws_backward_bytes;  /* workspace of the backward call, for dw and dbias */
} fc_causal_conv_plan;

int fc_causal_conv_make_plan(const fc_causal_conv_shape *shape, fc_causal_conv_plan *plan);

/* bias: C floats or NULL.  state_in: NULL for zeros.  state_out: NULL if not wanted; may be state_in.  One token or many. */
int fc_causal_conv(fc_context *ctx, const fc_causal_conv_plan *plan, const void *x_dev, const float *w_dev, const float *bias_dev, void *y_dev,
                   const void *state_in_dev, void *state_out_dev, const int32_t *lengths_dev);

/* Gradients of x, w and bias (fp32, overwritten; each may be NULL) and state_in (dstate_in; NULL: not wanted) from those of y and state_out (dstate_out;
 * NULL: none).  Without dw and dbias no workspace is needed.  Sums run in a fixed order. */
int fc_causal_conv_backward(fc_context *ctx, const fc_causal_conv_plan *plan, const void *dy_dev, const void *x_dev, const float *w_dev,
                            const float *bias_dev, void *dx_dev, float *dw_dev, float *dbias_dev, const void *state_in_dev,
                            const void *dstate_out_dev, void *dstate_in_dev, const int32_t *lengths_dev, void *ws_dev);

/* Selective scan: every channel d has N states that decay and take in by what the token says:
 *   dt = delta_t + delta_bias[d], through log(1 + e^dt) if `softplus`
 *   h_t[n] = exp(dt * A[d][n]) h_(t-1)[n] + dt * x_t * B_t[n],   y_t = (sum over n of C_t[n] h_t[n] + D[d] x_t) * z_t / (1 + e^-z_t)
 * x, delta, z and y: token t of sequence b begins at b*x_batch + t*x_token and so on, D channels side by side.  B and C are shared by the D/G channels of a
 * group: N values from b*b_batch + t*b_token + group*b_group on.  A is fp32 [D][N], not its logarithm; a rate above 0 is not checked for (the state
 * grows), one of minus infinity is a decay of 0 after a step above 0.  States are packed fp32 [B][D][N].
 * lengths as above: later tokens are not read, their outputs and gradients are zeros, and a state passes an empty sequence unchanged.
 * Limits: N <= 64, B*D < 2^26, D*(N+2) < 2^27 - 2^19, fewer than 2^24 workgroups, of which 32 tokens of 64 channels (N > 16: 32; N > 32: 16) are one; more
 * than one token: distances of tokens below 2^24 values. */
typedef struct {
    int B;
    long T;
    int D, N, G;
    int dtype;
    int softplus;
    long x_batch, x_token;
    long delta_batch, delta_token;
    long z_batch, z_token;
    long b_batch, b_token, b_group;
    long c_batch, c_token, c_group;
    long y_batch, y_token;
} fc_selective_scan_shape;

typedef struct {
    fc_selective_scan_shape shape;
    int tiles;                /* tokens are taken in tiles of 32, so many; 0: one by one */
    int segments;             /* parts of a sequence that run side by side, joined by their states */
    int walks_backward;       /* parts of a sequence, in whole tiles, of the backward call */
    size_t ws_bytes;          /* workspace of the forward call, 0 if none */
    size_t ws_backward_bytes; /* and of the backward call */
} fc_selective_scan_plan;

int fc_selective_scan_make_plan(const fc_selective_scan_shape *shape, fc_selective_scan_plan *plan);

/* D, delta_bias: D floats each, or NULL for zeros.  z: NULL for no gate.  state_in: NULL for zeros.  state_out: NULL if not wanted; may be state_in.
 * One token or many. */
int fc_selective_scan(fc_context *ctx, const fc_selective_scan_plan *plan, const void *x_dev, const void *delta_dev, const float *A_dev,
                      const void *B_dev, const void *C_dev, const float *D_dev, const void *z_dev, const float *delta_bias_dev, void *y_dev,
                      const float *state_in_dev, float *state_out_dev, const int32_t *lengths_dev, void *ws_dev);

/* Gradients of x, delta, B, C and, with a gate, z in the tensors' type and with the strides of what they are gradients of, of A, D and delta_bias (fp32,
 * overwritten; each may be NULL) and of state_in (dstate_in; NULL: not wanted) from those of y and state_out (dstate_out; NULL: none; may be dstate_in).
 * States are formed again from the inputs.  Gradients of shared values are summed in a fixed order. */
int fc_selective_scan_backward(fc_context *ctx, const fc_selective_scan_plan *plan, const void *dy_dev, const void *x_dev, const void *delta_dev,
                               const float *A_dev, const void *B_dev, const void *C_dev, const float *D_dev, const void *z_dev,
                               const float *delta_bias_dev, void *dx_dev, void *ddelta_dev, float *dA_dev, void *dB_dev, void *dC_dev, float *dD_dev,
                               void *dz_dev, float *ddelta_bias_dev, const float *state_in_dev, const float *dstate_out_dev, float *dstate_in_dev,
                               const int32_t *lengths_dev, void *ws_dev);

#ifdef __cplusplus
}
#endif
#endif
