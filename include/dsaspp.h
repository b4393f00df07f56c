/*
 * dsaspp.h -- C ABI of libdsaspp.so, the MI355X (gfx950) kernels behind the DenseASPP
 * forward/backward path.
 *
 * The reference implements this path with PyTorch built-ins called from Python
 * (there is no FFI in the reference); each entry point below names the reference
 * call site whose arithmetic it takes over.  All tensors are device pointers borrowed
 * for the duration of the call; nothing is retained or freed.  Every call enqueues on
 * the given HIP stream and returns without synchronising.  Return value: 0 on success,
 * non-zero on error (message via dsaspp_last_error(), thread-local).  No C++ exception
 * crosses this boundary.
 *
 * Layouts: activations are NHWC with an explicit pixel stride ("ld", in elements) so a
 * layer can read or write a channel slice of a wider feature slab; bf16 unless stated.
 * Descriptors with a `dtype` field also have an fp32 form (dtype = 1): activations AND the
 * weights they are multiplied with are then fp32 (weights straight from the fp32 master
 * arena, same [cout][taps][cin] layout), arithmetic is fp32 throughout.  That form exists so that
 * the network can be checked against an fp32 reference (logits to 1e-4, gradients to 1e-3): it
 * covers the forward pass of both trunks and the training pass (statistics, gradient epilogues,
 * weight gradients, BatchNorm backward) of the DenseNet trunks at output stride 8, with plain
 * untuned kernels.
 * Convolution weights are bf16 [cout][taps][cin] (K contiguous).  Channel counts, channel
 * offsets and strides must be multiples of 8 (16-byte chunks).
 */
#ifndef DSASPP_H
#define DSASPP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef void* dsaspp_stream_t; /* hipStream_t */

#define DSASPP_STAT_REPLICAS 16 /* per-channel sums are spread over this many replica rows */

int dsaspp_version(void);
/* Hash (16 hex digits) of the source files this library was built from, as semantic-segmentation_amd/build.py computes it
 * for the tree: lets a prebuilt library be matched to a checkout (measurement records carry it). */
const char* dsaspp_source_hash(void);
const char* dsaspp_last_error(void);

/* ------------------------------------------------------------------------------------
 * Fused [BN scale/shift -> ReLU -> (per-image channel mask)] -> convolution (1x1 or 3x3
 * dilated, stride 1, 'same' zero padding applied AFTER the prologue) -> epilogue.
 * Replaces nn.BatchNorm2d + nn.ReLU + nn.Conv2d of a dense layer / transition / ASPP
 * branch and the torch.cat that follows (reference call sites graph_seg_main.py:237,
 * graph_seg_test.py:144; cousin op models/bfp_net.py:60-62), and, with transposed
 * weights, their data-gradient in loss.backward() (graph_seg_main.py:239).
 *
 * Epilogue, per output element v (fp32 accumulator), pixel m of image n, channel c:
 *   v += bias[c]; v *= out_mask[n*out_mask_ld + c];
 *   if (epi_relu) { pre = ref[m*ldref+c] * e_scale[c] + e_shift[c] (ref itself when
 *                   e_scale is NULL); if (pre <= 0) v = 0; }
 *   if (s_acc)   { s_acc[rep][c] += v;  s_acc[rep][cout+c] += v * (ref - e_mean[c]) * e_rstd[c]; }
 *   if (g)       { t = v * (e_scale ? e_scale[c] : 1);  g[m*ldg+c] = (g_accumulate ? g + t : t); }   (fp32 or bf16 slab)
 *   else         { y[m*ldy+c] = v (bf16, or fp32 when y_f32);
 *                  if (stat_acc) { stat_acc[rep][c] += v_stored; stat_acc[rep][cout+c] += v_stored^2; } }
 * where rep = blockIdx % DSASPP_STAT_REPLICAS and the stat buffers are fp32
 * [DSASPP_STAT_REPLICAS][2*cout]: the sum over all rows counts (the fp32 form adds
 * 64-bit sums to stat_acc as a value and its rest in two rows).
 */
typedef struct dsaspp_conv_desc {
    int32_t n_img, H, W;      /* feature-map geometry (input == output) */
    int32_t cin, cout;        /* GEMM K per tap, GEMM N */
    int32_t taps, dil;        /* 1 (1x1) or 9 (3x3 with dilation dil) */
    const void* x;            /* bf16 NHWC input, channel offset already applied */
    int32_t ldx;
    const void* w;            /* bf16 [cout][taps*cin] */
    const float* in_scale;    /* [cin] or NULL (identity) */
    const float* in_shift;    /* [cin] or NULL */
    int32_t in_relu;          /* 0 none, 1 ReLU, 2 ReLU6 (1x1 forward form only) */
    const float* in_mask;     /* [n_img][in_mask_ld] per-image channel multiplier or NULL */
    int32_t in_mask_ld;
    const float* bias;        /* [cout] or NULL */
    const float* out_mask;    /* [n_img][out_mask_ld] or NULL */
    int32_t out_mask_ld;
    void* y;                  /* output (bf16, or fp32 if y_f32) ; unused when g != NULL */
    int32_t ldy;
    int32_t y_f32;
    float* stat_acc;          /* [R][2*cout] sum / sum of squares of the stored output, or NULL */
    int32_t epi_relu;         /* mask by the reference pre-activation: 1 = ReLU (pre > 0), 2 = ReLU6 (0 < pre < 6; single-source forms) */
    const void* ref;          /* bf16 [M][ldref] */
    int32_t ldref;
    const float* e_scale;     /* [cout] or NULL */
    const float* e_shift;
    const float* e_mean;
    const float* e_rstd;
    float* s_acc;             /* [R][2*cout] sum(v), sum(v*xhat) or NULL */
    void* g;                  /* gradient slab [M][ldg] (fp32, or bf16 when g_bf16) or NULL */
    int32_t ldg;
    int32_t g_accumulate;
    int32_t g_bf16;
    int32_t s_ld;             /* row half-width of s_acc when it is a slice of a wider accumulator (0: cout) */
    /* Extra sources (gradient-slab epilogue only, taps == 1): n_src in 2..4 sums the masked, scaled
     * data gradients of several consumer layers of the same slab prefix in one pass,
     *   g += sum_s e_scale_s * relu_mask_s(ref) * (x_s . w_s),
     * so the slab is read and written once per group of layers instead of once per layer.  Source 0 is
     * (x, w, e_scale, e_shift, s_acc, s_ld); sources 1..3 follow.  All sources share cin and ldx. */
    int32_t n_src;
    const void* x1; const void* w1; const float* es1; const float* eh1; float* sa1; int32_t sl1;
    const void* x2; const void* w2; const float* es2; const float* eh2; float* sa2; int32_t sl2;
    const void* x3; const void* w3; const float* es3; const float* eh3; float* sa3; int32_t sl3;
    int32_t dtype;            /* storage type of the activation tensors: 0 = bf16 (default), 1 = fp32 (eval-mode forward only) */
    /* Gradient read-out prologue (3x3 data gradient of a dense layer).  When gx_corr1 != NULL, x is a channel
     * slice of a bf16 gradient slab and the operand of the convolution is what dsaspp_grad_extract computes from it,
     *   v[m][c] = x[m][c] - gx_corr1[c] - ((gx_xs[m][c] - gx_mean[c]) * gx_rstd[c]) * gx_corr2[c]   (rounded to bf16),
     * gx_xs being the same channel slice of the activation slab (bf16 [M][gx_ldxs]); v is also stored to
     * gx_dz (bf16 [M][gx_lddz]) when that is non-NULL, for the weight gradient of the same layer.  Form: taps 9,
     * dil 1, 2 or 4, (cin, cout) = (48, 192) or (32, 128), epi_relu 1 with s_acc, bf16 output y, no other prologue. */
    const float* gx_corr1; const float* gx_corr2;
    const void* gx_xs; int32_t gx_ldxs;
    const float* gx_mean; const float* gx_rstd;
    void* gx_dz; int32_t gx_lddz;
} dsaspp_conv_desc;

int dsaspp_conv_fwd(const dsaspp_conv_desc* d, dsaspp_stream_t stream);
/* Name of the kernel family the calling thread's most recent dsaspp_conv_fwd or dsaspp_conv_wgrad was routed to
 * ("dgrad_wide", "dgrad_group", "conv3x3_halo", "conv_tile", "wgrad_wide", "wgrad_tile", ...; "" before the first call).  No counterpart in the reference: a
 * diagnostic, so that a test of one kernel can tell that its case did not quietly take another route. */
const char* dsaspp_conv_last_route(void);

/* Compute units to leave free for a collective that runs beside the backward pass.  The bucketed gradient all-reduce
 * (the reference's implicit nn.DataParallel reduce-add, graph_seg_main.py:173-174,239) is launched while later buckets are
 * still being computed; the slab data-gradient, wide forward and weight-gradient kernels are persistent, one block per
 * compute unit, and would otherwise leave the collective's kernels nowhere to run until they finish.  n in [0, 128]
 * (0 = use every compute unit; the default).  Process-wide; read at every launch.  dsaspp_get_comm_cus returns it. */
int dsaspp_set_comm_cus(int32_t n);
int dsaspp_get_comm_cus(void);

/* ------------------------------------------------------------------------------------
 * Weight gradient of the same convolution: dw[cout][taps][cin] (fp32) += sum over pixels
 * of dz[m][cout] * A[m + tap offset][cin], with A = prologue(x) recomputed on the fly
 * (never stored).  Replaces the weight-gradient half of loss.backward()
 * (reference graph_seg_main.py:239).  dw must be zeroed by the caller before the first
 * accumulation of a step; accumulation is by fp32 atomics (split over pixel ranges).
 */
typedef struct dsaspp_wgrad_desc {
    int32_t n_img, H, W;
    int32_t cin, cout;
    int32_t taps, dil;
    const void* x;            /* bf16 NHWC forward input */
    int32_t ldx;
    const float* in_scale;
    const float* in_shift;
    int32_t in_relu;
    const float* in_mask;
    int32_t in_mask_ld;
    const void* dz;           /* bf16 [M][lddz] gradient w.r.t. the conv output */
    int32_t lddz;
    float* dw;                /* fp32 [cout][taps*cin] */
    int32_t ksplit;           /* pixel-range splits (<=0: library picks) */
    /* Extra sources (taps == 1, in_mask == NULL, cout <= 192): n_src in 2..4 computes the weight gradients of
     * several 1x1 layers that read the SAME input tensor x (the dense layers of one block: each normalises the
     * shared slab prefix with its own BatchNorm) in one pass, so that x is fetched once per group instead of once
     * per layer:   dw_s[q][c] += sum_m dz_s[m][q] * relu(x[m][c] * sc_s[c] + sh_s[c])   for c < cin_s.
     * Source 0 is (dz, dw, in_scale, in_shift, cin); sources 1..3 follow.  All sources share x, ldx, cout, lddz and
     * in_relu; every source needs its scale/shift tables. */
    int32_t n_src;
    const void* dz1; float* dw1; const float* sc1; const float* sh1; int32_t cin1;
    const void* dz2; float* dw2; const float* sc2; const float* sh2; int32_t cin2;
    const void* dz3; float* dw3; const float* sc3; const float* sh3; int32_t cin3;
    int32_t dtype;            /* storage type of x and dz: 0 = bf16 (default), 1 = fp32 */
} dsaspp_wgrad_desc;

int dsaspp_conv_wgrad(const dsaspp_wgrad_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * BatchNorm bookkeeping (replaces the statistics side of nn.BatchNorm2d in train()/eval(),
 * reference graph_seg_main.py:162,312; graph_seg_test.py:136).
 *
 * For channel c in [0,C):
 *   if use_running:      mean = running_mean[c], var = running_var[c]
 *   else if c in [acc_c0, acc_c0+acc_cn): mean/var from acc (replica sums of x and x^2 over
 *                        `count` elements; acc is indexed by c-acc_c0 with width acc_cn and is
 *                        zeroed afterwards), stored to mean[c]/var[c]/rstd[c]
 *   else                 mean/var read from mean[c]/var[c]
 *   scale[c] = gamma[c]*rsqrt(var+eps); shift[c] = beta[c]-mean*scale[c]
 *   training (!use_running) and running_mean != NULL: running stats updated with `momentum`
 *   (unbiased variance), *num_batches_tracked += 1.
 */
typedef struct dsaspp_bn_desc {
    int32_t C;
    float* acc;               /* [R][2*acc_cn] or NULL */
    int32_t acc_c0, acc_cn;
    float count;              /* elements per channel (N*H*W) */
    float* mean;              /* [C] slab-level batch statistics (in/out) */
    float* var;
    float* rstd;
    const float* gamma;       /* [C] or NULL (identity affine) */
    const float* beta;
    float* running_mean;      /* [C] or NULL */
    float* running_var;
    int64_t* num_batches_tracked;
    float momentum, eps;
    int32_t use_running;
    float* scale;             /* [C] out (may be NULL) */
    float* shift;
    int32_t dtype;            /* form of the sums in acc: 0 = bf16 (default), added up in fp32; 1 = fp32, added up in 64 bits */
} dsaspp_bn_desc;

int dsaspp_bn_finalize(const dsaspp_bn_desc* d, dsaspp_stream_t stream);

/* BatchNorm backward bookkeeping (training mode).  acc holds replica sums S1 = sum(dy),
 * S2 = sum(dy*xhat) for C channels and is zeroed afterwards.
 *   dbeta[c] += S1, dgamma[c] += S2   (when non-NULL)
 *   mode 0 (private input): coefficient tables for dsaspp_bn_bwd_apply:
 *        A = scale, B = -scale*rstd*S2/count, Cc = -scale*S1/count - B*mean
 *   mode 1 (input is a shared feature slab): corr1[c] += scale*S1/count, corr2[c] += scale*S2/count
 */
typedef struct dsaspp_bn_bwd_desc {
    int32_t C;
    float* acc;               /* [R][2*acc_ld], this call's channels at [r][c] and [r][acc_ld+c] */
    int32_t acc_ld;           /* 0: C */
    float count;
    const float* scale;       /* forward scale (gamma*rstd) */
    const float* mean;
    const float* rstd;
    float* dgamma;
    float* dbeta;
    int32_t mode;
    float* coefA;
    float* coefB;
    float* coefC;
    float* corr1;
    float* corr2;
} dsaspp_bn_bwd_desc;

int dsaspp_bn_bwd_finalize(const dsaspp_bn_bwd_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Row-wise (pixel x channel) streaming kernels, NHWC, 8 channels per lane.
 */

/* y = act(x*scale+shift + res) -> bf16, optional statistics of the stored values
 * (features.norm5 + the in-place ReLU heading ASPP_3; the BatchNorm closing a MobileNetV2
 * inverted-residual block and its skip connection).  relu: 0 none, 1 ReLU, 2 ReLU6. */
typedef struct dsaspp_bnact_desc {
    int64_t M; int32_t C;
    const void* x; int32_t ldx;
    const float* scale; const float* shift; int32_t relu;
    void* y; int32_t ldy;
    float* stat_acc;          /* [R][2*C] or NULL */
    const void* res; int32_t ldres;   /* bf16 [M][ldres] added after the affine map, or NULL */
    int32_t dtype;            /* storage type of the activation tensors: 0 = bf16 (default), 1 = fp32 (eval-mode forward only) */
} dsaspp_bnact_desc;
int dsaspp_bn_act(const dsaspp_bnact_desc* d, dsaspp_stream_t stream);

/* Gradient read-out from a slab:
 *   v = g[m][c] - corr1[c] - ((xs[m][c]-s_mean[c])*s_rstd[c])*corr2[c]   (corr terms when corr1 != NULL)
 *   v *= mask[n][c]                                                       (when mask != NULL)
 *   if relu: pre = yref*r_scale+r_shift (yref itself if r_scale NULL); if pre<=0: v = 0
 *   dz[m][c] = bf16(v);  s_acc += {v, v*((yref-r_mean)*r_rstd)} (when s_acc != NULL)
 *   colsum[c] += v (when non-NULL; plain fp32 atomics) */
typedef struct dsaspp_gradx_desc {
    int64_t M; int32_t C; int32_t hw;       /* hw = pixels per image (for mask row lookup) */
    const void* g; int32_t ldg; int32_t g_bf16;   /* gradient slab: fp32, or bf16 when g_bf16 */
    const float* corr1; const float* corr2;
    const void* xs; int32_t ldxs; const float* s_mean; const float* s_rstd;
    const float* mask; int32_t mask_ld;
    int32_t relu;
    const void* yref; int32_t ldyref;
    const float* r_scale; const float* r_shift; const float* r_mean; const float* r_rstd;
    void* dz; int32_t lddz;
    int32_t dz_f32;           /* store dz as fp32 (when it feeds a BatchNorm backward: see bn_bwd_apply) */
    float* s_acc;
    float* colsum;
    int32_t dtype;            /* 0 = bf16 activations (default); 1 = fp32: g, xs, yref and dz are all fp32 */
} dsaspp_gradx_desc;
int dsaspp_grad_extract(const dsaspp_gradx_desc* d, dsaspp_stream_t stream);

/* dy = A[c]*dr + B[c]*y + Cc[c] -> bf16 ; colsum[c] += dy when non-NULL.
 * dr is normally fp32 (dr_f32): the BatchNorm backward removes the mean and xhat components of
 * dr, which can dominate it, so rounding dr to bf16 first would swamp what is left. */
typedef struct dsaspp_bnapply_desc {
    int64_t M; int32_t C;
    const void* dr; int32_t lddr; int32_t dr_f32;
    const void* y; int32_t ldy;
    const float* coefA; const float* coefB; const float* coefC;
    void* dy; int32_t lddy;
    float* colsum;
    int32_t dtype;            /* 0 = bf16 activations (default); 1 = fp32: dr, y and dy are all fp32 */
} dsaspp_bnapply_desc;
int dsaspp_bn_bwd_apply(const dsaspp_bnapply_desc* d, dsaspp_stream_t stream);

/* 2x2 average pooling (transition1) forward (+ statistics) and backward. */
typedef struct dsaspp_pool_desc {
    int32_t n_img, H, W, C;   /* input geometry (H, W even) */
    const void* x; int32_t ldx;
    void* y; int32_t ldy;     /* output geometry H/2 x W/2 */
    float* stat_acc;
    int32_t dtype;            /* storage type of the activation tensors: 0 = bf16 (default), 1 = fp32 (eval-mode forward only) */
} dsaspp_pool_desc;
int dsaspp_avgpool2_fwd(const dsaspp_pool_desc* d, dsaspp_stream_t stream);
/* dx[n][h][w][c] = dy[n][h/2][w/2][c] / 4 ; here x is the gradient OUTPUT (full size), y the INPUT */
int dsaspp_avgpool2_bwd(const dsaspp_pool_desc* d, dsaspp_stream_t stream);

/* Bilinear x2 upsample (align_corners=False) of an NHWC feature map, the `upsample` stage that follows
 * features.norm5 when output_stride = 16 (upstream DenseASPP(model_cfg, n_class, output_stride) constructor;
 * reference call site graph_seg_test.py:129), fused with that BatchNorm and the ReLU heading ASPP_3:
 *   fwd: y[n][Y][X][c] = act(scale[c] * interp2(x)[n][Y][X][c] + shift[c])   (interpolation weights sum to 1, so the
 *        affine map commutes with it); optional statistics of the stored values
 *   bwd: dx[n][y][x][c] = sum over the <= 3x3 outputs that read (y, x) of weight * dy ; optional BatchNorm-backward
 *        sums s_acc += {dx, dx * (yref - mean) * rstd}, yref being the low-resolution forward input
 * x / dx are [N*h*w][ld], y / dy are [N*2h*2w][ld]. */
typedef struct dsaspp_up2_desc {
    int32_t n_img, h, w, C;   /* low-resolution geometry */
    const void* x; int32_t ldx;           /* fwd: input ; bwd: yref (may be NULL when s_acc is NULL) */
    const float* scale; const float* shift; int32_t relu;   /* fwd only */
    void* y; int32_t ldy;                 /* fwd: output ; bwd: dy (input) */
    float* stat_acc;                      /* fwd: [R][2*C] or NULL */
    void* dx; int32_t lddx; int32_t dx_f32;   /* bwd output (bf16, or fp32 when dx_f32) */
    const float* mean; const float* rstd; float* s_acc;     /* bwd: BatchNorm-backward sums [R][2*C] or NULL */
    int32_t dtype;            /* fwd: 0 = bf16, 1 = fp32 storage (eval-mode forward only) */
} dsaspp_up2_desc;
int dsaspp_upsample2_fwd(const dsaspp_up2_desc* d, dsaspp_stream_t stream);
int dsaspp_upsample2_bwd(const dsaspp_up2_desc* d, dsaspp_stream_t stream);

/* Stem: 7x7/2 im2col of the NCHW fp32 network input to bf16 rows [N*Ho*Wo][ldcol]
 * (K order (ky,kx,ci), zero padded), so conv0 runs as a 1x1 GEMM; and the
 * BN+ReLU -> 3x3/2 max pooling that follows, with its backward. */
typedef struct dsaspp_im2col_desc {
    int32_t n_img, H, W;      /* input image size; output Ho = H/2, Wo = W/2 */
    const float* x;           /* NCHW fp32, 3 channels */
    void* col; int32_t ldcol; /* >= 152 and multiple of 8; columns >= 147 zero filled */
    int32_t dtype;            /* storage type of the activation tensors: 0 = bf16 (default), 1 = fp32 (eval-mode forward only) */
} dsaspp_im2col_desc;
int dsaspp_stem_im2col(const dsaspp_im2col_desc* d, dsaspp_stream_t stream);

/* The same stem without a column matrix in memory (bf16 storage): a block builds the column tile of one output-row
 * segment in LDS from the input rows it draws from.  dsaspp_stem7_fwd replaces dsaspp_stem_im2col + the 1x1 dsaspp_conv_fwd
 * over its rows (conv0 of model(image), reference graph_seg_main.py:237): y = bf16(col . w^T) with the batch-statistics sums
 * of the rounded values in stat_acc.  dsaspp_stem7_wgrad replaces dsaspp_bn_bwd_apply + dsaspp_conv_wgrad of the same layer
 * (the conv0 part of loss.backward(), graph_seg_main.py:239): dw[q][k] += sum over pixels of dy[p][q] * col[p][k] with
 * dy = bf16(coefA*dr + coefB*yref + coefC) formed on the fly, k < 147; the blocks' partial sums pass through the workspace
 * ws (dsaspp_stem7_wgrad_workspace_floats(cout) floats) and are added in a fixed order: no atomics. */
typedef struct dsaspp_stem7_desc {
    int32_t n_img, H, W;      /* input image size (even); outputs at Ho = H/2, Wo = W/2 */
    const float* x;           /* NCHW fp32, 3 channels */
    int32_t cout;             /* 64 or 96 */
    const void* w; int32_t ldw;           /* fwd: bf16 [cout][ldw], columns (ky, kx, ci), ldw >= 160, columns >= 147 zero */
    void* y; int32_t ldy;                 /* fwd: bf16 [N*Ho*Wo][ldy] */
    float* stat_acc;                      /* fwd: [R][2*cout] or NULL */
    const void* dr; int32_t lddr; int32_t dr_f32;     /* wgrad: masked gradient entering norm0's backward, bf16 or fp32 */
    const void* yref; int32_t ldyref;     /* wgrad: the forward output y */
    const float* coefA; const float* coefB; const float* coefC;   /* wgrad: [cout] each (dsaspp_bn_bwd_finalize, mode 0) */
    float* dw; int32_t lddw;              /* wgrad: fp32 [cout][lddw], lddw >= 147, accumulated */
    float* ws; int64_t ws_floats;         /* wgrad: workspace */
} dsaspp_stem7_desc;
int dsaspp_stem7_fwd(const dsaspp_stem7_desc* d, dsaspp_stream_t stream);
int dsaspp_stem7_wgrad(const dsaspp_stem7_desc* d, dsaspp_stream_t stream);
int64_t dsaspp_stem7_wgrad_workspace_floats(int32_t cout);

typedef struct dsaspp_maxpool_desc {
    int32_t n_img, H, W, C;   /* input (conv0 output) geometry; output ceil(H/2) x ceil(W/2), H, W even */
    const void* x; int32_t ldx;       /* raw conv0 output bf16 */
    const float* scale; const float* shift; /* norm0 */
    void* y; int32_t ldy;             /* pooled relu(bn(x)) bf16 */
    uint8_t* argmax;                  /* [N*Ho*Wo][C] window position 0..8, or NULL */
    float* stat_acc;
    /* backward only */
    const void* dy; int32_t lddy;     /* bf16 gradient w.r.t. pooled output */
    void* dr; int32_t lddr;           /* masked gradient w.r.t. norm0 output (bf16, or fp32 if dr_f32) */
    int32_t dr_f32;
    const float* mean; const float* rstd;
    float* s_acc;
    int32_t dtype;            /* storage type of the activation tensors: 0 = bf16 (default), 1 = fp32 (eval-mode forward only) */
} dsaspp_maxpool_desc;
int dsaspp_maxpool3s2_fwd(const dsaspp_maxpool_desc* d, dsaspp_stream_t stream);
int dsaspp_maxpool3s2_bwd(const dsaspp_maxpool_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * MobileNetV2 trunk of MobileNetDenseASPP (reference: cfgs/MobileNetDenseASPP.py:1-8 configures
 * it; constructor call site graph_seg_test.py:129).  Pointwise convolutions run through
 * dsaspp_conv_fwd; these two cover the layers that are not GEMM shaped.
 */

/* Stem: 3x3 stride-2 pad-1 convolution of the NCHW fp32 network input (3 channels) to raw
 * (pre-BatchNorm) bf16 NHWC rows [N*(H/2)*(W/2)][ldy]; H and W even.
 * w: bf16 [cout][27], K order (ky, kx, ci); cout a multiple of 8, at most 64. */
typedef struct dsaspp_stem3_desc {
    int32_t n_img, H, W;      /* input image size */
    const float* x;
    const void* w;
    int32_t cout;
    void* y; int32_t ldy;
    int32_t dtype;            /* storage type of the activation tensors: 0 = bf16 (default), 1 = fp32 (eval-mode forward only) */
} dsaspp_stem3_desc;
int dsaspp_stem3x3s2(const dsaspp_stem3_desc* d, dsaspp_stream_t stream);

/* Depthwise 3x3 convolution, stride 1 or 2, dilation dil, zero padding dil (applied AFTER the
 * prologue), with the producer's BatchNorm + activation fused in front:
 *   a = act(x*in_scale + in_shift)   (in_relu: 0 none, 1 ReLU, 2 ReLU6; identity affine when NULL)
 *   y[n][ho][wo][c] = sum_{ky,kx} w[c][ky*3+kx] * a[n][ho*stride+(ky-1)*dil][wo*stride+(kx-1)*dil][c]
 * Output geometry ((H-1)/stride+1) x ((W-1)/stride+1); raw (pre-BatchNorm) bf16 NHWC. */
typedef struct dsaspp_dw_desc {
    int32_t n_img, H, W, C;   /* input geometry; C a multiple of 8 */
    int32_t stride, dil;
    const void* x; int32_t ldx;
    const float* in_scale; const float* in_shift; int32_t in_relu;
    const void* w;            /* bf16 [C][9] */
    void* y; int32_t ldy;
    int32_t dtype;            /* storage type of the activation tensors: 0 = bf16 (default), 1 = fp32 (eval-mode forward only) */
} dsaspp_dw_desc;
int dsaspp_dwconv3x3(const dsaspp_dw_desc* d, dsaspp_stream_t stream);

/* Backward of the depthwise 3x3 convolution above (training of the MobileNetV2 trunk; the reference
 * trains it through autograd: graph_seg_test.py:129 builds the model, train.py-style loops call
 * loss.backward()).  Geometry, prologue and weights are those of the forward call.
 *   bwd_data:  da[n][h][w][c] = sum_{ky,kx} w[c][ky*3+kx] * dy[n][ho][wo][c]  over the output pixels with
 *              ho*stride + (ky-1)*dil == h, wo*stride + (kx-1)*dil == w;
 *              dx = da where the prologue's activation passes gradient (pre = x*in_scale+in_shift;
 *              in_relu 1: pre > 0, 2: 0 < pre < 6, 0: everywhere), else 0 -- the gradient w.r.t. the
 *              producer's BatchNorm output; with s_acc the BatchNorm-backward sums of that BatchNorm,
 *              sum(dx) and sum(dx * (x - e_mean) * e_rstd), go to replica rows [R][2*C].
 *   wgrad:     dw[c][ky*3+kx] += sum_{n,ho,wo} dy[n][ho][wo][c] * a[n][ho*stride+(ky-1)*dil][wo*stride+(kx-1)*dil][c]
 *              (a = the prologue output rounded to bf16, zero outside the image), fp32 [C][9]. */
typedef struct dsaspp_dwbwd_desc {
    int32_t n_img, H, W, C;   /* forward input geometry; C a multiple of 8 */
    int32_t stride, dil;
    const void* x; int32_t ldx;       /* forward raw input, bf16 */
    const float* in_scale; const float* in_shift; int32_t in_relu;
    const void* w;                    /* bf16 [C][9] (bwd_data) */
    const void* dy; int32_t lddy;     /* gradient w.r.t. the forward output, bf16 [N*Ho*Wo][lddy] */
    void* dx; int32_t lddx;           /* bwd_data result, bf16 or fp32 [N*H*W][lddx] */
    int32_t dx_f32;
    const float* e_mean; const float* e_rstd; float* s_acc;   /* optional BatchNorm-backward sums */
    float* dw;                        /* wgrad result, accumulated */
} dsaspp_dwbwd_desc;
int dsaspp_dwconv3x3_bwd_data(const dsaspp_dwbwd_desc* d, dsaspp_stream_t stream);
int dsaspp_dwconv3x3_wgrad(const dsaspp_dwbwd_desc* d, dsaspp_stream_t stream);

/* 3x3/2 pad-1 im2col of the NCHW fp32 network input to bf16 rows [N*(H/2)*(W/2)][ldcol], K order
 * (ky, kx, ci), columns >= 27 zero: the MobileNetV2 stem's weight gradient is then a 1x1
 * dsaspp_conv_wgrad with cin = ldcol (uses dsaspp_im2col_desc; ldcol >= 32, a multiple of 8). */
int dsaspp_stem3_im2col(const dsaspp_im2col_desc* d, dsaspp_stream_t stream);

/* Adjoint of the two stem im2col forms: the gradient with respect to the network input,
 *   dx[n][ci][hi][wi] (fp32 NCHW) = sum over output positions (ho, wo) and taps (ky, kx) with 2*ho - pad + ky == hi and
 *   2*wo - pad + kx == wi of dcol[(n*Ho + ho)*Wo + wo][(ky*ks + kx)*3 + ci],
 * ks = 7 (pad 3: conv0 of the DenseNet trunks) or 3 (pad 1: the MobileNetV2 stem), Ho = H/2, Wo = W/2.  With the column
 * gradient dcol = dy . W0 (a 1x1 dsaspp_conv_fwd over the stem's output gradient) this is what autograd delivers to an image
 * tensor that requires grad when loss.backward() runs (reference graph_seg_main.py:237-239).  Each input pixel gathers its at
 * most 4 x 4 (2 x 2) contributions in a fixed order: no atomics.  accumulate != 0 adds to dx. */
typedef struct dsaspp_col2im_desc {
    int32_t n_img, H, W;      /* image size (even) */
    int32_t ks;               /* 7 or 3 */
    const void* dcol; int32_t ldcol;   /* bf16 (fp32 when dtype == 1) [N*Ho*Wo][ldcol], ldcol >= ks*ks*3 */
    float* dx;                /* NCHW fp32, 3 channels */
    int32_t accumulate;
    int32_t dtype;
} dsaspp_col2im_desc;
int dsaspp_stem_col2im(const dsaspp_col2im_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Bilinear x8 upsample (align_corners=False) fused with softmax cross-entropy
 * (replaces nn.Upsample(scale_factor=8, mode='bilinear') + CrossEntropyLoss(ignore_index)
 * + their backward; reference graph_seg_main.py:216,238-239).
 *   logits: fp32 NHWC [N][h][w][ldl] low-resolution class scores (n_class <= 32 used)
 *   labels: int64 [N][8h][8w]
 *   dlogits: fp32 same shape as logits; must be zero on entry, receives the UNNORMALISED
 *            gradient (sum over pixels of softmax - onehot)
 *   accum:  fp32[DSASPP_CE_ACCUM_FLOATS] zero on entry: DSASPP_CE_ACCUM_SLOTS partial {sum of per-pixel losses,
 *            number of non-ignored pixels} pairs, pair s at accum[s*DSASPP_CE_ACCUM_STRIDE] (one per 128-byte line:
 *            atomics on a single address are executed one after the other); their sums are the totals
 * dsaspp_ce_finalize then divides: loss[0] = sum/count, dlogits /= count
 * (times grad_scale), writes a bf16 copy for the classifier backward and the per-class
 * column sums (the classifier bias gradient, += into dbias when non-NULL).
 */
#define DSASPP_CE_ACCUM_SLOTS 32
#define DSASPP_CE_ACCUM_STRIDE 32
#define DSASPP_CE_ACCUM_FLOATS (DSASPP_CE_ACCUM_SLOTS * DSASPP_CE_ACCUM_STRIDE)
typedef struct dsaspp_ce_desc {
    int32_t n_img, h, w;      /* low-res geometry */
    int32_t n_class; int32_t ldl;
    const float* logits;
    const int64_t* labels;
    int32_t ignore_index;
    float* dlogits;
    float* accum;
    /* finalize */
    float grad_scale;
    float* loss;
    void* dlogits_bf16; int32_t lddb;
    float* dbias;
} dsaspp_ce_desc;
int dsaspp_upsample8_ce(const dsaspp_ce_desc* d, dsaspp_stream_t stream);
int dsaspp_ce_finalize(const dsaspp_ce_desc* d, dsaspp_stream_t stream);

/* The two calls above in one, without any device allocation by caller or library.  It has no counterpart
 * in the reference; it is for callers that cannot allocate device memory around the loss: code under HIP
 * graph capture, tight serving / evaluation loops, harnesses that forbid hipMalloc.  The fp32 gradient
 * staging (`dlogits`) and the loss accumulators (`accum`) live in a built-in per-GPU array instead of
 * caller buffers: d->dlogits and d->accum are ignored (may be NULL).  Inputs logits/labels and outputs
 * loss (required), dlogits_bf16 and dbias (optional, dbias is added to) are the caller's, with the
 * meaning they have in dsaspp_upsample8_ce + dsaspp_ce_finalize.
 * Limit: n_img*h*w <= DSASPP_NOALLOC_MAX_PIXELS low-resolution pixels and ldl <= 32; larger calls fail
 * with an error and touch nothing.  The built-in array (16 MiB) stays resident on every GPU the library
 * runs on until the process ends.  All calls on one GPU share it: calls that overlap on one GPU (two
 * streams, two threads) race; serialise them.  The first call on a GPU looks the array's device address
 * up (hipGetSymbolAddress), so make that first call outside a graph capture. */
#define DSASPP_NOALLOC_MAX_PIXELS 131072
int dsaspp_upsample8_ce_loss_noalloc(const dsaspp_ce_desc* d, dsaspp_stream_t stream);

/* Materialised x8 upsample for the plain forward() API: fp32 NHWC low-res -> fp32 NCHW
 * [N][n_class][8h][8w]; its adjoint; and the inference variant that writes only the arg-max
 * class per pixel (replaces Upsample + F.softmax + argmax, reference graph_seg_test.py:144-146,62). */
typedef struct dsaspp_up_desc {
    int32_t n_img, h, w, n_class, ldl;
    const float* logits;      /* low-res NHWC fp32 (fwd/argmax: input ; bwd: OUTPUT, zero on entry) */
    float* out;               /* NCHW fp32 full-res (fwd: output ; bwd: input gradient) */
    int64_t* argmax;          /* [N][8h][8w] */
} dsaspp_up_desc;
int dsaspp_upsample8_fwd(const dsaspp_up_desc* d, dsaspp_stream_t stream);
int dsaspp_upsample8_bwd(const dsaspp_up_desc* d, dsaspp_stream_t stream);
int dsaspp_upsample8_argmax(const dsaspp_up_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Evaluation metric next to the path: bilinear x8 upsample + arg-max + confusion-matrix counts in one
 * pass (replaces F.softmax + torch.argmax + the per-class Python loop with .item() syncs of
 * evaluate_model, reference graph_seg_main.py:85-103, and get_iou, graph_seg_test.py:61-78).
 *   conf: int64 [(n_class+1)][n_class], conf[r][p] += 1 for every full-resolution pixel with arg-max p and
 *         label r; labels outside [0, n_class) (the ignore label 255) count in row n_class, because the
 *         reference's union term counts predictions on ignored pixels too.
 *   argmax: optional int64 [N][8h][8w] map of the arg-max classes.
 */
typedef struct dsaspp_conf_desc {
    int32_t n_img, h, w, n_class, ldl;
    const float* logits;      /* low-res NHWC fp32 class scores */
    const int64_t* labels;    /* [N][8h][8w] */
    int64_t* conf;
    int64_t* argmax;
} dsaspp_conf_desc;
int dsaspp_upsample8_confusion(const dsaspp_conf_desc* d, dsaspp_stream_t stream);

/* Input pre-processing in front of the path (replaces the numpy/torchvision steps of the data loader,
 * reference graph_seg_dataloader.py:111-116,129-131 labelId -> trainId table, :136 /255, :177-180
 * horizontal flip, :213-214 mean/std normalisation, :226-227 HWC -> CHW float / int64 labels):
 *   x[n][c][y][x'] = (img[n][y][x][c] / 255 - mean_c) / std_c   with x' = W-1-x when hflip
 *   labels[n][y][x'] = lut[label_ids[n][y][x]]                   (when label_ids != NULL)
 * so that the host-to-device copy can be the 3 B/pixel image and 1 B/pixel label map. */
typedef struct dsaspp_prep_desc {
    int32_t n_img, H, W;
    const uint8_t* img;       /* [N][H][W][3] bytes */
    float* x;                 /* [N][3][H][W] fp32 */
    float mean0, mean1, mean2;
    float std0, std1, std2;
    int32_t hflip;
    const uint8_t* label_ids; /* [N][H][W] or NULL */
    const uint8_t* lut;       /* [256] */
    int64_t* labels;          /* [N][H][W] */
} dsaspp_prep_desc;
int dsaspp_preprocess(const dsaspp_prep_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Class scores: log probability of a given label, entropy and the most probable classes of every row (a pixel, a token) of a
 * tensor of logits, and their gradient.  It sits next to dsaspp_upsample8_argmax / _ce: the reference only has the arg-max and
 * the mean loss of the same logits (graph_seg_test.py:62, graph_seg_main.py:238).
 *   log_p[c] = z[c] - logsumexp(z),  p = exp(log_p)
 *   logp = log_p[label]; 0 for a row without a label: label == ignore_index or outside [0, n_class)
 *   entropy = -sum p log_p, top_class / top_logp: the top_k largest logits, descending, the lowest class first among equal ones
 * Classes at -inf are masked out: p = 0, never an alternative; alternatives a row does not have are -1 with log probability -inf.
 * A row with nothing but -inf: logp -inf (if labelled), entropy 0, gradient 0.  A row with a NaN or +inf: logp (if labelled), entropy
 * and top_logp NaN, top_class -1.  The gradient of a row whose upstream gradients are all 0 is 0 whatever its logits hold.
 * Backward, a = g_logp (0 without a label), b = g_entropy, t_j = g_top[j] (0 at -1), A = a + sum t_j:
 *   dz[c] = a [c == label] + sum_j t_j [c == top_class[j]] - p[c] A - b p[c] (log_p[c] + entropy)
 *
 * Rows are numbered (i0, i1, i2) row-major over [d0][d1][d2]; logits of row (i0, i1, i2), class c at
 * logits[i0*s0 + i1*s1 + i2*s2 + c*sc] (strides in elements, >= 0).  labels, logp and entropy are dense [rows];
 * top_logp and top_class are [d0][top_k][d1][d2].  dlogits is dense: [rows][n_class] when sc == 1, else [d0][n_class][d1][d2].
 * With sc != 1 a lane walks the classes of a row, which is made for many rows of few classes (few rows of many: milliseconds; copy them first).
 * Arithmetic is fp32 on logits of any dtype; dlogits has the logits' dtype (0 = bf16, 1 = fp32, 2 = fp16), rounded once, and must not
 * overlap the logits. */
#define DSASPP_SCORES_MAX_TOP 8
typedef struct dsaspp_scores_desc {
    int32_t dtype, n_class, top_k;
    int64_t d0, d1, d2;
    int64_t s0, s1, s2, sc;
    const void* logits;
    const int64_t* labels;    /* may be NULL: then logp must be NULL too */
    int64_t ignore_index;
    float* logp;              /* outputs of the forward call, each may be NULL; inputs of the backward call: stats, entropy */
    float* entropy;           /* (only when g_entropy is given) and top_class (only when g_top is given) */
    float* stats;             /* [rows][2] for the backward call: largest logit, log of the sum of exponentials relative to it */
    float* top_logp; int64_t* top_class;
    /* backward: upstream gradients, each may be NULL (counts as 0); *_one != 0: one value for all rows / entries */
    const float* g_logp; const float* g_entropy; const float* g_top;
    int32_t g_logp_one, g_entropy_one, g_top_one;
    void* dlogits;
    float* ws; int64_t ws_len; /* forward, few long rows: dsaspp_scores_workspace floats, contents need not be initialised */
} dsaspp_scores_desc;
int64_t dsaspp_scores_workspace(const dsaspp_scores_desc* d); /* floats for the forward call, often 0; -1 on a bad descriptor */
int dsaspp_scores_fwd(const dsaspp_scores_desc* d, dsaspp_stream_t stream);
int dsaspp_scores_bwd(const dsaspp_scores_desc* d, dsaspp_stream_t stream);

/* The same on logits at 1/8 resolution, with the bilinear x8 upsample (align_corners=False) fused in: the full-resolution logits
 * are never written.  z = hy*r0 + ly*r1, r_i = hx*L[yi][x0] + lx*L[yi][x1], every product and sum rounded to fp32 by itself, so the
 * order of the classes is that of those values to the bit.  What is computed from them has the errors of an fp32 log-softmax, and in pixels
 * whose largest logit is M < 64 in magnitude up to 4 M + 92 + 5 (|log p| + entropy) half-steps (2^-24) more in a log probability.  A NaN or
 * infinity counts in every pixel whose four source pixels hold it, at weight 0 too, as in torch's upsample.
 * n_class <= 32, fewer than 2^24 tiles of 64 x 32 pixels.  Logits of image n, pixel (y, x), class c at
 * logits[n*sn + y*sy + x*sx + c*sc]; labels, logp, entropy [n_img][8h][8w]; top_* [n_img][top_k][8h][8w]; upstream gradients
 * likewise.  Backward reads logits, labels, stats and (with g_entropy) entropy and (with g_top) top_class; dlogits at dlogits[n*gn + y*gy + x*gx + c*gc], dtype g_dtype;
 * ws: dsaspp_scores8_workspace floats, contents need not be initialised. */
typedef struct dsaspp_scores8_desc {
    int32_t n_img, h, w, n_class, top_k;
    int32_t dtype, g_dtype;
    int64_t sn, sy, sx, sc;
    const void* logits;
    const int64_t* labels;
    int64_t ignore_index;
    float* logp; float* entropy; float* top_logp; int64_t* top_class;
    float* stats;             /* [n_img][8h][8w] for the backward call: sum of exponentials relative to a reference that it forms again */
    const float* g_logp; const float* g_entropy; const float* g_top;
    int32_t g_logp_one, g_entropy_one, g_top_one;
    void* dlogits;
    int64_t gn, gy, gx, gc;
    float* ws; int64_t ws_len;
} dsaspp_scores8_desc;
int64_t dsaspp_scores8_workspace(const dsaspp_scores8_desc* d); /* floats for the backward call; -1 on a bad descriptor */
int dsaspp_scores8_fwd(const dsaspp_scores8_desc* d, dsaspp_stream_t stream);
int dsaspp_scores8_bwd(const dsaspp_scores8_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Parameter-side kernels over the flat parameter arena (adjacent to the path:
 * torch.optim.Adam(weight_decay) + poly learning rate, reference graph_seg_main.py:186,241-245).
 */
/* p, g, m, v fp32[n]; Adam with coupled L2 (g += wd*p), bias correction from `step`
 * (1-based); also refreshes the bf16 shadow copy w16[n]. */
typedef struct dsaspp_adam_desc {
    int64_t n;
    float* p; const float* g; float* m; float* v;
    void* w16;
    float lr, beta1, beta2, eps, weight_decay;
    int32_t step;
    float grad_scale;         /* multiply g first (e.g. 1/world_size) */
} dsaspp_adam_desc;
int dsaspp_adam_step(const dsaspp_adam_desc* d, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Global gradient norm over many tensors, clipping by it, and the Adam update with the clip coefficient applied on the fly
 * (what torch.nn.utils.clip_grad_norm_ + torch.optim.Adam do between backward and the next step).
 *   norm = scale * sqrt(sum over all ranges of g^2)   (norm_type 2)      scale * max |g|   (norm_type 0)
 *   coef = min(1, max_norm / (norm + 1e-6))           a NaN norm gives a NaN coefficient
 * The gradients are a HOST array of dense device ranges; it is read during the call only and may be freed after it.  A range
 * needs no more alignment than its element type.  Sums are fp64 (the square of an fp32 value is exact there and cannot overflow) and
 * taken in an order that depends on the list alone -- sizes, types, addresses (ranges that follow one another in memory are one) and their
 * order: the same list gives the same bits each time.  Equal values elsewhere in memory may be added up in another order: their norm may be
 * another last bit away.
 *   1. dsaspp_grad_norm_partials: one fp64 partial per block into ws (dsaspp_grad_norm_workspace doubles, contents need not be
 *      initialised).  n_ranges == 0 is allowed: the norm is 0.
 *   2. dsaspp_grad_norm_finish: norm[0] from the partials; or
 *      dsaspp_clip_scale: every range times coef in place, rounded once to its type (ranges are left untouched where coef is 1),
 *      norm[0] too; or dsaspp_adam_step_clipped: the Adam update with g * scale * coef; g itself is not written.
 * The three read the partials and nothing but the partials: call 1 with the same ranges first, on the same stream.
 * dsaspp_clip_grads is 1 and dsaspp_clip_scale in one call (in one kernel where the gradients are few).
 * Ranges that are written must not overlap: dsaspp_grad_ranges_overlap tells (0 = disjoint, 1 = two of them share memory).
 * dtype of a range: 0 = bf16, 1 = fp32, 2 = fp16. */
typedef struct dsaspp_grad_range {
    void* p;
    int64_t n;                /* elements, > 0 */
    int32_t dtype, pad;
} dsaspp_grad_range;
typedef struct dsaspp_clip_desc {
    const dsaspp_grad_range* ranges; /* host */
    int32_t n_ranges;
    int32_t norm_type;        /* 2 = Euclidean, 0 = largest magnitude */
    float scale;              /* the gradients count as scale * g (> 0); dsaspp_clip_scale takes 1 only */
    float max_norm;           /* >= 0, may be +inf */
    double* ws; int64_t ws_len; /* device, in doubles */
    float* norm;              /* device, 1 float */
} dsaspp_clip_desc;
int64_t dsaspp_grad_norm_workspace(const dsaspp_clip_desc* d); /* doubles; -1 on a bad descriptor */
int dsaspp_grad_norm_partials(const dsaspp_clip_desc* d, dsaspp_stream_t stream);
int dsaspp_grad_norm_finish(const dsaspp_clip_desc* d, dsaspp_stream_t stream);
int dsaspp_clip_scale(const dsaspp_clip_desc* d, dsaspp_stream_t stream);
int dsaspp_clip_grads(const dsaspp_clip_desc* d, dsaspp_stream_t stream);
int dsaspp_grad_ranges_overlap(const dsaspp_clip_desc* d);
/* The update of dsaspp_adam_step with g * c->scale * coef, on any n > 0 elements with no more alignment than their type.  The factors
 * come in double, as an optimizer's host code holds them: 1 - beta2 of a beta2 rounded to fp32 is 1.3e-5 off at 0.999. */
typedef struct dsaspp_adam_clip_desc {
    int64_t n;
    float* p; const float* g; float* m; float* v;
    void* w16;                /* bf16 copy of p, may be NULL */
    double lr, beta1, beta2, eps, weight_decay;
    int64_t step;             /* 1-based */
} dsaspp_adam_clip_desc;
int dsaspp_adam_step_clipped(const dsaspp_adam_clip_desc* a, const dsaspp_clip_desc* c, dsaspp_stream_t stream);

/* fp32 -> bf16 cast of the flat arena */
int dsaspp_cast_bf16(const float* src, void* dst, int64_t n, dsaspp_stream_t stream);

/* Transposed weight copies for the data-gradient kernels, batched:
 * dst[c][taps-1-t][n] = src[n][t][c] for each table entry. */
typedef struct dsaspp_wt_entry {
    int64_t src_off, dst_off; /* element offsets into src / dst arenas (bf16) */
    int32_t cout, cin, taps, pad;
} dsaspp_wt_entry;
int dsaspp_weight_transpose(const void* src, void* dst, const dsaspp_wt_entry* table_dev,
                            int32_t n_entries, int64_t max_elems, dsaspp_stream_t stream);
/* same for fp32 arenas (the fp32 form of the data-gradient convolutions) */
int dsaspp_weight_transpose_f32(const float* src, float* dst, const dsaspp_wt_entry* table_dev,
                                int32_t n_entries, int64_t max_elems, dsaspp_stream_t stream);

/* fp32 2-D strided copy (row pad / unpad of the stem weight and its gradient);
 * dst[r][c] = src[r][c] (+= when accumulate) for c < cols; dst columns [cols, dst_cols) are zeroed. */
int dsaspp_copy2d_f32(const float* src, int32_t lds, float* dst, int32_t ldd,
                      int32_t rows, int32_t cols, int32_t dst_cols, int32_t accumulate,
                      dsaspp_stream_t stream);
/* same, fp32 source rows -> bf16 destination rows */
int dsaspp_copy2d_f32_bf16(const float* src, int32_t lds, void* dst, int32_t ldd,
                           int32_t rows, int32_t cols, int32_t dst_cols, dsaspp_stream_t stream);

int dsaspp_memset_async(void* p, int32_t value, int64_t bytes, dsaspp_stream_t stream);

/* ------------------------------------------------------------------------------------
 * Programs: a recorded sequence of the calls above, replayed with one host call
 * (and optionally as one captured HIP graph).  Descriptors are copied at record time.
 */
typedef struct dsaspp_program dsaspp_program;
enum {
    DSASPP_OP_CONV = 1, DSASPP_OP_WGRAD, DSASPP_OP_BN_FINALIZE, DSASPP_OP_BN_BWD_FINALIZE,
    DSASPP_OP_BN_ACT, DSASPP_OP_GRAD_EXTRACT, DSASPP_OP_BN_BWD_APPLY, DSASPP_OP_AVGPOOL_FWD,
    DSASPP_OP_AVGPOOL_BWD, DSASPP_OP_IM2COL, DSASPP_OP_MAXPOOL_FWD, DSASPP_OP_MAXPOOL_BWD,
    DSASPP_OP_UPCE, DSASPP_OP_CE_FINALIZE, DSASPP_OP_UP_FWD, DSASPP_OP_UP_BWD, DSASPP_OP_UP_ARGMAX,
    DSASPP_OP_MEMSET, DSASPP_OP_COPY2D, DSASPP_OP_COPY2D_BF16, DSASPP_OP_STEM3, DSASPP_OP_DWCONV,
    DSASPP_OP_UP2_FWD, DSASPP_OP_UP2_BWD, DSASPP_OP_DW_BWD_DATA, DSASPP_OP_DW_WGRAD, DSASPP_OP_STEM3_COL,
    DSASPP_OP_COL2IM, DSASPP_OP_STEM7_FWD, DSASPP_OP_STEM7_WGRAD
};
dsaspp_program* dsaspp_program_create(void);
void dsaspp_program_destroy(dsaspp_program* p);
/* desc points at the descriptor struct of that op; for MEMSET / COPY2D see dsaspp_generic_desc */
typedef struct dsaspp_generic_desc {
    const void* src; void* dst;
    int64_t n;                /* bytes (memset) */
    int32_t value;
    int32_t lds, ldd, rows, cols, dst_cols, accumulate;
} dsaspp_generic_desc;
int dsaspp_program_add(dsaspp_program* p, int32_t op, const void* desc, int64_t desc_bytes);
int dsaspp_program_size(const dsaspp_program* p);
/* run ops [first, last) ; last < 0 means to the end */
int dsaspp_program_run(dsaspp_program* p, int32_t first, int32_t last, dsaspp_stream_t stream);
/* Ops marked with side != 0 are enqueued on a second HIP stream that the program owns: before each of them the
 * side stream waits for everything the run has enqueued on the caller's stream so far, and the caller's stream waits
 * for the side stream at the end of every dsaspp_program_run call.  The recorder must make sure that nothing enqueued
 * later in the same run overwrites what a side op reads or reads what it writes (the engine marks the dense-layer
 * weight gradients, whose inputs live in per-layer buffers and whose outputs only the optimizer reads): two MFMA
 * kernels that are each latency bound overlap to 1.17-1.23x of their sequential time. */
/* side = 2 marks an op that stays on the caller's stream but must not start before the side stream has finished what
 * it was given so far (it overwrites a buffer a side op reads): the caller's stream waits for the side stream there. */
int dsaspp_program_set_side(dsaspp_program* p, int32_t op_index, int32_t side);
/* Per-kernel timing with HIP events on the launch stream (measurement only): ops given a
 * non-zero tag are bracketed by two events on every run until the timing is read.
 * dsaspp_program_read_timing synchronises the recorded events, adds the elapsed milliseconds
 * and launch counts of tag t to ms[t] / launches[t] (t < n_tags) and clears the recordings. */
int dsaspp_program_set_tag(dsaspp_program* p, int32_t op_index, int32_t tag);
int dsaspp_program_read_timing(dsaspp_program* p, int32_t n_tags, double* ms, int64_t* launches);

#ifdef __cplusplus
}
#endif
#endif /* DSASPP_H */
