/*
 * kdec.h — C ABI of the MI355X (gfx950) Kokoro-82M iSTFTNet decoder kernels.
 *
 * The reference (wlejon/brosoundml) drives the decoder back half through
 * brotensor ops from src/kokoro_decoder_backward.cpp. Each entry point below
 * replaces one such op or a fused group of them; the comment on each names
 * the reference call sites it stands in for (paths relative to the reference
 * repository). The C++ drop-in layer (kokoro_decoder_backward.h in this
 * project) calls these; so do the ctypes tests and the benchmark.
 *
 * Conventions
 *  - Every pointer argument named like a tensor is a DEVICE pointer to FP32
 *    data. Activations are batched NCL: utterance n, channel c, sample l at
 *    n * bs + c * L + l, where `bs` is the batch stride in elements (bs >= C*L;
 *    a larger stride addresses a channel slice of a wider tensor, which is how
 *    channel concatenation and slicing are expressed without copies).
 *  - Weight layouts are the reference's (include/brosoundml/modules.h:14-21,
 *    kokoro_modules.h): Conv1d W (C_out, C_in*k) index [co][ci*k+t];
 *    ConvTranspose1d W (C_in, C_out*k) index [ci][co*k+t]; depthwise pool
 *    W (C, 3); biases (C_out).
 *  - Per-utterance affines: gamma/beta hold N rows of C values at row stride
 *    `gb_bs` (0 broadcasts one row to every utterance).
 *  - Every call is asynchronous on the context's stream and returns 0 on
 *    success or a negative KDEC_E* code; kdec_last_error() gives the message.
 *    Output buffers are caller-allocated; the library allocates only its own
 *    workspace (split-K partials, packed weights, statistics).
 *  - Grad outputs documented as "accumulated" are added to (caller zeroes
 *    them); all others are overwritten.
 */
#ifndef KDEC_H
#define KDEC_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KDEC_OK 0
#define KDEC_EINVAL -1   /* bad argument / shape */
#define KDEC_EHIP -2     /* HIP runtime error */
#define KDEC_ENOMEM -3   /* device allocation failed */

typedef struct kdec_ctx kdec_ctx;

/* Activation applied after an AdaIN affine. */
#define KDEC_ACT_NONE 0
#define KDEC_ACT_LEAKY 1 /* leaky_relu(slope)             (bt::leaky_relu_*) */
#define KDEC_ACT_SNAKE 2 /* x + sin^2(alpha_c x)/alpha_c  (bt::snake_*)      */

/* ─── context ─────────────────────────────────────────────────────────── */

/* Creates a context on HIP device `device` with a default-priority stream of
 * its own. No reference counterpart (brotensor's runtime is implicit). */
int kdec_ctx_create(int device, kdec_ctx** out);
int kdec_ctx_destroy(kdec_ctx* ctx);
/* Last error message of this context ("" if none). */
const char* kdec_last_error(const kdec_ctx* ctx);
/* Runs subsequent work on `stream` (a hipStream_t; NULL = the HIP null
 * stream). Until the first call the context uses a stream of its own. */
int kdec_set_stream(kdec_ctx* ctx, void* stream);
void* kdec_get_stream(const kdec_ctx* ctx);
int kdec_synchronize(kdec_ctx* ctx);
/* Device memory from the context's stream-ordered caching allocator. */
int kdec_malloc(kdec_ctx* ctx, size_t bytes, void** out);
int kdec_free(kdec_ctx* ctx, void* ptr);
/* Per-kernel-family timing with HIP events on the context stream (0 = off).
 * Calls that are captured into a graph are not timed. */
int kdec_profile_enable(kdec_ctx* ctx, int on);
/* Fills names / ms / launches / algorithmic FLOP / algorithmic HBM bytes
 * (any may be NULL) for up to `cap` families; returns the count. */
int kdec_profile_read(kdec_ctx* ctx, const char** names, double* ms,
                      long* launches, double* flops, double* bytes, int cap);
int kdec_profile_reset(kdec_ctx* ctx);

/* ─── convolutions (implicit GEMM on FP32 MFMA) ───────────────────────── */

/* Y = scale * (conv1d(X, W) + bias + R) + beta * Y
 * Replaces bt::conv1d via Conv1d::forward (src/modules.cpp:103-108) at
 * kokoro_decoder_backward.cpp:185,193,199,307,316,389,502-504,617, with the
 * residual add / scale that follow it (:204-205, :319, :642, :654-656) fused.
 * bias, R may be NULL. L_out = (L + 2p - d(k-1) - 1)/s + 1. groups = 1. */
int kdec_conv1d_fwd(kdec_ctx* ctx, const float* X, long x_bs, const float* W,
                    const float* bias, float* Y, long y_bs, int N, int C_in,
                    int L, int C_out, int k, int stride, int pad, int dil,
                    const float* R, long r_bs, float scale, float beta);

/* kdec_conv1d_fwd (beta = 0) that also writes the instance-norm statistics
 * of its output rows, stats[n*C_out + c] = (mean, 1/sqrt(var + eps)) as
 * kdec_instnorm_stats computes them. Where the GEMM runs the quad-packed
 * kernel, its epilogue records each tile's per-row count, mean and squared
 * deviations and a wave per row merges them (in double), so Y is not read
 * again; elsewhere it is the two calls. For the conv outputs that feed an
 * AdaIN (kokoro_decoder_backward.cpp:307-313, the ResBlock1 convs whose
 * output the next adain_affine_forward normalises, :100-120). */
int kdec_conv1d_fwd_stats(kdec_ctx* ctx, const float* X, long x_bs,
                          const float* W, const float* bias, float* Y,
                          long y_bs, int N, int C_in, int L, int C_out, int k,
                          int stride, int pad, int dil, const float* R,
                          long r_bs, float scale, float eps, float* stats);
/* 1 where kdec_conv1d_fwd_stats takes the fused path for this geometry, else
 * 0 (a caller may then prefer the one-pass kdec_adain_act_fwd_stats). */
int kdec_conv1d_fwd_stats_fused(kdec_ctx* ctx, int N, int C_in, int L,
                                int C_out, int k, int stride, int pad,
                                int dil);

/* dX = scale * conv1d_backward_input(W, dY) + beta * dX   (stride 1)
 * Replaces bt::conv1d_backward_input at kokoro_decoder_backward.cpp:230-234,
 * 244-248, 271-275, 347-350, 360-363, 453-456. L is the input length. */
int kdec_conv1d_dgrad(kdec_ctx* ctx, const float* W, const float* dY,
                      long dy_bs, float* dX, long dx_bs, int N, int C_in,
                      int L, int C_out, int k, int stride, int pad, int dil,
                      float scale, float beta);

/* The input grad of a stride-1 conv1d followed by the backward of the
 * AdaIN + activation whose output feeds that conv:
 *   dX = kdec_adain_act_bwd(X, ..., dY' = conv1d_dgrad(W, dY)) (+ R)
 * with dgamma / dbeta overwritten and dalpha accumulated, as the two calls
 * kdec_conv1d_dgrad + kdec_adain_act_bwd (same arguments). On grids of four
 * output tiles per CU or more, the GEMM's epilogue applies the activation
 * derivative and forms the AdaIN's per-row partial sums, so dY' is never
 * written separately and the AdaIN pass reads it once; elsewhere it makes
 * those two calls. dX must not alias X or R.
 * Replaces bt::conv1d_backward_input followed by bt::snake_backward and
 * adain_affine_backward at kokoro_decoder_backward.cpp:347-356 and :360-369
 * (leaky: :230-241, :244-266). */
int kdec_conv1d_dgrad_adain_bwd(kdec_ctx* ctx, const float* W, const float* dY,
                                long dy_bs, int N, int C_in, int L, int C_out,
                                int k, int stride, int pad, int dil,
                                const float* X, long x_bs, const float* stats,
                                const float* gamma, const float* beta,
                                long gb_bs, int act, float slope,
                                const float* alpha, const float* R, long r_bs,
                                float* dX, long dx_bs, float* dgamma,
                                float* dbeta, long dgb_bs, float* dalpha);

/* dW (C_out, C_in*k) and db (C_out) accumulated over the batch; either may
 * be NULL.
 * Extension: the reference freezes conv weights; the signature of
 * its accumulating bt::conv1d_backward_weight/_bias is the one used in
 * src/bc_resnet.cpp:1006-1007, 1020-1025. */
int kdec_conv1d_wgrad(kdec_ctx* ctx, const float* X, long x_bs,
                      const float* dY, long dy_bs, float* dW, float* db, int N,
                      int C_in, int L, int C_out, int k, int stride, int pad,
                      int dil);

/* Y = convT(X, W) + bias (groups = 1, dilation 1, output_padding op).
 * Replaces bt::conv_transpose1d_forward at kokoro_decoder_backward.cpp:627-629
 * (ups). Polyphase implicit GEMM. */
int kdec_convt1d_fwd(kdec_ctx* ctx, const float* X, long x_bs, const float* W,
                     const float* bias, float* Y, long y_bs, int N, int C_in,
                     int L, int C_out, int k, int stride, int pad, int op);
/* The generator's last upsample stage in one pass (kokoro_decoder_backward.cpp
 * :627-642): Y = reflection_pad_left1(convT(X, W) + bias) + R, i.e. with
 * pad_left = 1 each output row is L_out + 1 long, column j + 1 holds the
 * transposed conv's column j and column 0 its column 1, and R (the noise
 * source, Y's layout and length, or NULL) is added to every column; with
 * pad_left = 0, Y = convT(X, W) + bias + R. Same polyphase GEMM as
 * kdec_convt1d_fwd, with the pad and the add in its epilogue. */
int kdec_convt1d_fwd_res(kdec_ctx* ctx, const float* X, long x_bs, const float* W, const float* bias, float* Y,
                         long y_bs, int N, int C_in, int L, int C_out, int k, int stride, int pad, int op,
                         const float* R, long r_bs, int pad_left);
/* dX = conv_transpose1d_backward_input(W, dY) (= strided conv1d of dY with W).
 * Replaces bt::conv_transpose1d_backward_input at :725-728. */
int kdec_convt1d_dgrad(kdec_ctx* ctx, const float* W, const float* dY,
                       long dy_bs, float* dX, long dx_bs, int N, int C_in,
                       int L, int C_out, int k, int stride, int pad, int op);
/* dW (C_in, C_out*k), db (C_out) accumulated. Extension of the reference. */
int kdec_convt1d_wgrad(kdec_ctx* ctx, const float* X, long x_bs,
                       const float* dY, long dy_bs, float* dW, float* db,
                       int N, int C_in, int L, int C_out, int k, int stride,
                       int pad, int op);

/* Depthwise ConvTranspose1d k3 s2 p1 op1 (the upsampling block's pool):
 * replaces bt::conv_transpose1d_forward / _backward_input with groups = C at
 * kokoro_decoder_backward.cpp:176-180, 252-256. L_out = 2L. */
int kdec_pool_fwd(kdec_ctx* ctx, const float* X, long x_bs, const float* W,
                  const float* bias, float* Y, long y_bs, int N, int C, int L);
int kdec_pool_dgrad(kdec_ctx* ctx, const float* W, const float* dY,
                    long dy_bs, float* dX, long dx_bs, int N, int C, int L);
/* dW (C,3), db (C) accumulated. Extension of the reference. */
int kdec_pool_wgrad(kdec_ctx* ctx, const float* X, long x_bs, const float* dY,
                    long dy_bs, float* dW, float* db, int N, int C, int L);

/* ─── AdaIN (instance norm + style affine) fused with its activation ───── */

/* Per-(n,c) mean and 1/sqrt(biased var + eps) over L (G = C group norm).
 * Replaces the statistics half of bt::group_norm_forward at
 * kokoro_decoder_backward.cpp:112-113. stats: N*C (mean, rstd) pairs. */
int kdec_instnorm_stats(kdec_ctx* ctx, const float* X, long x_bs, int N,
                        int C, int L, float eps, float* stats);

/* Y = act((1 + gamma) * (X - mean) * rstd + beta); Ypre (optional) gets the
 * pre-activation. Replaces adain_affine_forward (:100-120: group_norm,
 * nchw_to_sequence, modulate, sequence_to_nchw) plus the following
 * bt::leaky_relu_forward (:172, :190) or bt::snake_forward (:305-306,
 * :313-314). slope for LEAKY; alpha (C) for SNAKE. beta may be NULL (zero). */
int kdec_adain_act_fwd(kdec_ctx* ctx, const float* X, long x_bs,
                       const float* stats, const float* gamma,
                       const float* beta, long gb_bs, int act,
                       float slope, const float* alpha, float* Y, long y_bs,
                       float* Ypre, long ypre_bs, int N, int C, int L);

/* Statistics and the affine + activation in one pass: stats (N*C (mean,
 * rstd) pairs, as kdec_instnorm_stats) are written and used at once. Short
 * rows are held in registers, so x is read once (the two-call sequence reads
 * it twice); longer rows take the two passes. Replaces the
 * group_norm + modulate + activation sequence of kokoro_decoder_backward.cpp
 * :100-120 with :172/:190 (leaky) or :305-306/:313-314 (snake). */
int kdec_adain_act_fwd_stats(kdec_ctx* ctx, const float* X, long x_bs,
                             float eps, float* stats, const float* gamma,
                             const float* beta, long gb_bs, int act,
                             float slope, const float* alpha, float* Y,
                             long y_bs, float* Ypre, long ypre_bs, int N,
                             int C, int L);

/* Backward of kdec_adain_act_fwd given dY (grad at the activation output):
 *   dX = adain_backward(act_backward(dY)) + (R ? R : 0)
 *   dgamma/dbeta (N*C at gb_bs rows) overwritten; dalpha (C) accumulated
 *   over the batch when non-NULL (SNAKE only).
 * Replaces bt::leaky_relu_backward / bt::snake_backward followed by
 * adain_affine_backward (:237+240-241, :262+265-266, :352-356, :365-369);
 * R carries the residual skip added at :372. beta may be NULL for ACT_NONE
 * (adain_affine_backward takes no beta). */
int kdec_adain_act_bwd(kdec_ctx* ctx, const float* X, long x_bs,
                       const float* stats, const float* gamma,
                       const float* beta, long gb_bs, int act, float slope,
                       const float* alpha, const float* dY, long dy_bs,
                       const float* R, long r_bs, float* dX, long dx_bs,
                       float* dgamma, float* dbeta, long dgb_bs,
                       float* dalpha, int N, int C, int L);

/* kdec_adain_act_bwd without any allocation: same arguments, kernels and
 * results. No counterpart in the reference; it is for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). Its scratch lives in a device array of
 * KDEC_NOALLOC_SCRATCH_BYTES per GPU: the per-row alpha-grad shares (4 B per
 * row, with dalpha when N > 1 or the rows take the chunked passes) and, for
 * rows that no one-block row kernel holds (longer than 62464, or longer than
 * 49152 when a row does not start on 16 B), the chunk partial sums and row
 * means (24 B per row and 4096-sample chunk, plus 8 B per row). The array is
 * held until the process ends; a call that needs more returns
 * KDEC_EINVAL with the sizes in kdec_last_error. It calls no hipMalloc /
 * hipFree and records no profiling events. Every call on one GPU shares
 * that GPU's array: calls that overlap on one GPU (any two streams or
 * contexts) race and must be serialised by the caller. */
#define KDEC_NOALLOC_SCRATCH_BYTES (4 << 20)
int kdec_adain_act_bwd_noalloc(kdec_ctx* ctx, const float* X, long x_bs,
                               const float* stats, const float* gamma,
                               const float* beta, long gb_bs, int act,
                               float slope, const float* alpha,
                               const float* dY, long dy_bs, const float* R,
                               long r_bs, float* dX, long dx_bs,
                               float* dgamma, float* dbeta, long dgb_bs,
                               float* dalpha, int N, int C, int L);

/* ─── elementwise ─────────────────────────────────────────────────────── */

/* Y[i] = value for i < n (a kernel, not hipMemset, so it can be captured). */
int kdec_fill(kdec_ctx* ctx, float* Y, long n, float value);

/* Y = leaky_relu(X, slope) over N rows of `len` (bt::leaky_relu_forward). */
int kdec_leaky_fwd(kdec_ctx* ctx, const float* X, long x_bs, float* Y,
                   long y_bs, int N, long len, float slope);
/* dX = (X > 0 ? 1 : slope) * dY (bt::leaky_relu_backward, :613/731 0.1). */
int kdec_leaky_bwd(kdec_ctx* ctx, const float* X, long x_bs, const float* dY,
                   long dy_bs, float* dX, long dx_bs, int N, long len,
                   float slope);
/* kdec_leaky_bwd followed by a scaling pass, in one: dX = scale * ((X > 0 ?
 * 1 : slope) * dY), the same two roundings. The generator's backward, whose
 * stage output grad is divided by the K resblocks right after a leaky
 * backward forms it (kokoro_decoder_backward.cpp:457 and :731, then
 * :689-690). */
int kdec_leaky_bwd_scaled(kdec_ctx* ctx, const float* X, long x_bs, const float* dY, long dy_bs, float* dX,
                          long dx_bs, int N, long len, float slope, float scale);
/* Y = a*A + b*B (B may be NULL) over N rows of `len` (bt::add_inplace /
 * bt::scale_inplace, copy_d2d for concat / slice). */
int kdec_axpby(kdec_ctx* ctx, float a, const float* A, long a_bs, float b,
               const float* B, long b_bs, float* Y, long y_bs, int N,
               long len);
/* Y = (A + B) + C over N rows of `len`, the float adds in that order (Y may
 * alias A). The generator stage's resblock sum (kokoro_decoder_backward.cpp:
 * 644-657, xs = x0; xs += x1; xs += x2) when the K = 3 resblocks run on
 * concurrent streams into separate buffers, each with the 1/K already applied
 * by its last conv: the same two roundings as the one-stream schedule, whose
 * last convs accumulate into one buffer in that order. */
int kdec_add3(kdec_ctx* ctx, const float* A, long a_bs, const float* B,
              long b_bs, const float* C, long c_bs, float* Y, long y_bs,
              int N, long len);
/* kdec_add3 that also writes Z = leaky_relu(Y, slope) (Y may alias A): the
 * generator stage's resblock sum (kokoro_decoder_backward.cpp:645-655) and
 * the activation the next stage's transposed conv (slope 0.1, :613) or
 * conv_post (0.01, :388) reads. */
int kdec_add3_leaky(kdec_ctx* ctx, const float* A, long a_bs, const float* B, long b_bs, const float* C, long c_bs,
                    float* Y, long y_bs, float* Z, long z_bs, int N, long len, float slope);
/* kdec_add3 over N x C rows of L + 1 that also writes the left reflect
 * pad's adjoint in the same pass (the generator's last stage backward,
 * :716-728): Y = (A + B) + C (as kdec_add3), and Z (rows of L) = the
 * gradient of the unpadded rows, Z[j] = Y[j + 1] + (j == 1 ? Y[0] : 0), the
 * bits kdec_pad_reflect_left1_bwd(Y) gives. Y may alias A; Z aliases
 * none of the others. */
int kdec_add3_unpad_left1(kdec_ctx* ctx, const float* A, long a_bs, const float* B, long b_bs, const float* C,
                          long c_bs, float* Y, long y_bs, float* Z, long z_bs, int N, int Cn, int L);
/* Left reflect pad by one sample, C rows of L -> L+1 (bt::pad1d_* mode 1 at
 * :633-634 / :720-721). */
int kdec_pad_reflect_left1_fwd(kdec_ctx* ctx, const float* X, long x_bs,
                               float* Y, long y_bs, int N, int C, int L);
int kdec_pad_reflect_left1_bwd(kdec_ctx* ctx, const float* dY, long dy_bs,
                               float* dX, long dx_bs, int N, int C, int L);
/* Nearest 2x along L (:63-96, the host round trip in the reference). */
int kdec_nearest2x_fwd(kdec_ctx* ctx, const float* X, long x_bs, float* Y,
                       long y_bs, int N, int C, int L);
/* dX = scale * (dY[2l] + dY[2l+1]) + beta * dX */
int kdec_nearest2x_bwd(kdec_ctx* ctx, const float* dY, long dy_bs, float* dX,
                       long dx_bs, int N, int C, int L, float scale,
                       float beta);

/* ─── spectral head, iSTFT, harmonic source, style projection ─────────── */

/* audio = istft(complex_from_polar(exp(post[:F]), sin(post[F:]))), center,
 * not normalized, periodic Hann of length n_fft, hop `hop`; post (N, 2F, L)
 * with F = n_fft/2+1; audio (N, (L-1)*hop). Replaces the host exp/sin, the
 * bt::complex_from_polar and bt::istft of kokoro_decoder_backward.cpp:391-409. */
int kdec_spectral_fwd(kdec_ctx* ctx, const float* post, long post_bs,
                      const float* window, float* audio, long audio_bs, int N,
                      int L, int n_fft, int hop);
/* dpost from daudio: bt::istft_backward and the host polar/exp/sin adjoint at
 * kokoro_decoder_backward.cpp:423-449. `window` (n_fft values, device) may be
 * NULL for the periodic Hann window in both calls. */
int kdec_spectral_bwd(kdec_ctx* ctx, const float* post, long post_bs,
                      const float* window, const float* daudio,
                      long daudio_bs, float* dpost, long dpost_bs, int N,
                      int L, int n_fft, int hop);

/* HarmonicSource::forward (kokoro_modules.cpp:1574-1665) for N utterances:
 * F0 (N, frame_count) -> har (N, n_fft+2, frame_count*upsample_scale/hop+1).
 * The phase recurrence runs sequentially per (utterance, harmonic) in float
 * exactly as the reference's host loop; sin / l_linear / tanh / STFT /
 * abs / atan2 run in parallel. lW (harmonic_num+1), lb (1) device pointers. */
int kdec_harmonic_source(kdec_ctx* ctx, const float* F0, long f0_bs,
                         float* har, long har_bs, int N, int frame_count,
                         const float* lW, const float* lb, int harmonic_num,
                         int sample_rate, int upsample_scale, int n_fft,
                         int hop);

/* Style projection for a group of AdaIN units stacked row-wise:
 * out[n, r] = W[r, :] . style[n, :] + b[r] for r < rows (W rows x S).
 * Replaces compute_style_affine (kokoro_modules.cpp:563-572) /
 * bt::lora_forward with the LoRA term absent (decoder_lora.cpp:184-194). */
int kdec_style_proj_fwd(kdec_ctx* ctx, const float* W, const float* b,
                        const float* style, long style_bs, float* out,
                        long out_bs, int N, int rows, int S);
/* dstyle[n, :] = beta*dstyle + sum_r W[r, :] dout[n, r]  (dstyle may be NULL);
 * dW += sum_n dout[n, r] style[n, :]; db += sum_n dout[n, r] (may be NULL).
 * The adjoint of bt::lora_backward with dX requested
 * (decoder_lora.cpp:198-207); the reference passes dX = nullptr. */
int kdec_style_proj_bwd(kdec_ctx* ctx, const float* W, const float* style,
                        long style_bs, const float* dout, long dout_bs,
                        float* dstyle, long dstyle_bs, float beta, float* dW,
                        float* db, int N, int rows, int S);

/* LoRA-adapted style projection (DecoderLora's adapter_fwd,
 * decoder_lora.cpp:184-194, over bt::lora_forward; the adapter contract of
 * decoder_lora.h:63-77): for `units` AdaIN units stacked row-wise, unit u
 * owning rows [unit_off[u], unit_off[u+1]) (unit_off: units+1 ints, device),
 *   H[n, u*rank + j] = A[u*rank + j, :] . style[n, :]
 *   out[n, r] = W[r, :] . style[n, :] + b[r]
 *               + scale * sum_j B[r, j] * g[n, j] * H[n, u(r)*rank + j]
 * A (units*rank, S), B (rows, rank), g the gate (N, rank) at batch stride
 * g_bs (0: one gate for every utterance). H (N, units*rank) is written for
 * the backward. */
int kdec_lora_proj_fwd(kdec_ctx* ctx, const float* W, const float* b,
                       const float* A, const float* B, const float* g,
                       long g_bs, float scale, const int* unit_off, int units,
                       int rank, const float* style, long style_bs, float* H,
                       float* out, long out_bs, int N, int rows, int S);
/* Its adjoint (adapter_bwd, decoder_lora.cpp:198-207, over bt::lora_backward)
 * plus the d(style) extension. With dHG[n, u*rank+j] = scale * sum_{r in u}
 * B[r, j] dout[n, r]:
 *   dB[r, j] += scale * sum_n dout[n, r] g[n, j] H[n, u(r)*rank + j]
 *   dG[n, j] += sum_u dHG[n, u*rank+j] H[n, u*rank+j]   (summed over n when g_bs = 0)
 *   dA[u*rank+j, :] += sum_n dHG[n, u*rank+j] g[n, j] style[n, :]
 *   dstyle[n, :] = beta*dstyle + W^T dout[n] + A^T (dHG g)[n]
 *   dW, db as kdec_style_proj_bwd.
 * Any of dstyle, dW, db, dA, dB, dG may be NULL. */
int kdec_lora_proj_bwd(kdec_ctx* ctx, const float* W, const float* A,
                       const float* B, const float* g, long g_bs, float scale,
                       const int* unit_off, int units, int rank,
                       const float* style, long style_bs, const float* H,
                       const float* dout, long dout_bs, float* dstyle,
                       long dstyle_bs, float beta, float* dW, float* db,
                       float* dA, float* dB, float* dG, int N, int rows, int S);

/* DecoderLora's conditioning gate g(v) = W2 tanh(W1 v), bias-free
 * (ConditioningGate::forward, decoder_lora.cpp:56-66): for N condition
 * vectors v (in_dim each, batch stride v_bs) writes act = tanh(W1 v)
 * (N, hidden; kept for the backward) and g (N, rank) at batch stride g_bs.
 * W1 (hidden, in_dim), W2 (rank, hidden). N * hidden <= 16384. */
int kdec_lora_gate_fwd(kdec_ctx* ctx, const float* W1, const float* W2,
                       const float* v, long v_bs, int N, int in_dim,
                       int hidden, int rank, float* act, float* g,
                       long g_bs);
/* Its adjoint (ConditioningGate::backward, decoder_lora.cpp:68-80): with the
 * forward's act and the gate grad dG (N, rank at batch stride dg_bs),
 * accumulates dW2 += dG^T act and dW1 += ((1 - act^2) * (dG W2))^T v. The
 * condition is an input, not a trainable: no dv. */
int kdec_lora_gate_bwd(kdec_ctx* ctx, const float* W2, const float* v,
                       long v_bs, const float* act, const float* dG,
                       long dg_bs, int N, int in_dim, int hidden, int rank,
                       float* dW1, float* dW2);
/* One Adam step over n parameters (bt::adam_step as DecoderLora::adam_step
 * calls it, decoder_lora.cpp:305-314): m = b1 m + (1-b1) g,
 * v = b2 v + (1-b2) g^2, p -= lr (m / (1 - b1^step)) /
 * (sqrt(v / (1 - b2^step)) + eps). step >= 1. */
int kdec_adam_step(kdec_ctx* ctx, float* p, const float* g, float* m,
                   float* v, long n, float lr, float beta1, float beta2,
                   float eps, int step);

/* Length regulation (the host loop of Kokoro::prepare_decode_context /
 * synthesize, kokoro.cpp:667-689): asr[n, c, t] = t_en[n, c, l] for the
 * phoneme l whose duration run covers frame t (runs in token order,
 * negative durations count as zero), zero for t >= the utterance's total.
 * t_en (N, C, L) at batch stride te_bs, dur (N, L) int32 (device) at dur_bs,
 * asr (N, C, T) at asr_bs; totals (N int32, device) receives each total
 * when not NULL. L <= 4096. */
int kdec_length_regulate(kdec_ctx* ctx, const float* t_en, long te_bs,
                         const int* dur, long dur_bs, int N, int C, int L,
                         float* asr, long asr_bs, int T, int* totals);

/* ─── token operators ─────────────────────────────────────────────────── */
/*
 * For the text networks beside the decoder and for batches whose requests
 * each have adapters of their own. They have no counterpart on the
 * reference's path. Tensors are FP32 or bf16 (`dtype`, one type for all of a
 * call's tensors unless noted), sums and softmax statistics are float, and
 * each output is rounded once. Besides, bf16 calls round to bf16 what enters a
 * matrix product: attention's probabilities (for O and dV) and dS (for dK and
 * dQ; in dQ to 16 bits where a tile is masked), and dQ takes dO . O from the
 * rounded O (dK from the exact sums); the adapters' H and dH enter Y
 * and dX to 16 bits, dA and dB to 24. Float calls round nothing on the way.
 * Rows are tokens; a row stride (`_rs`, in elements) is the distance of two
 * tokens, a head stride (`_hs`) that of two heads; the innermost axis is
 * contiguous. Inputs take any alignment and any stride; tensors whose base,
 * strides and widths are multiples of 16 bytes take the wide loads. Offsets and
 * adapter choices are int32 on the device. The rows of an output must not
 * overlap (repeated ones are refused), nor outputs inputs unless noted.
 */
#define KDEC_F32 0
#define KDEC_BF16 1

/* Y = R + drop(X) over `rows` rows of `cols` (R may be NULL): an element is
 * dropped where its 16 random bits are below thr = round(p * 65536), a kept
 * one is multiplied by 65536 / (65536 - thr). The bits are those of
 * Philox4x32-10 under key `seed` and counter (col / 8, row, offset's low and
 * high word): the same seed, offset, row and column give the same mask, so
 * the backward is this call on dY with R = NULL. Y may be X or R.
 * 0 <= p, and p and its rounding below 1. A row stride of 0 broadcasts one row
 * of X or R (a mask of its own for every row). */
int kdec_dropout(kdec_ctx* ctx, int dtype, const void* X, long x_rs,
                 const void* R, long r_rs, void* Y, long y_rs, long rows,
                 int cols, float p, long seed, long offset);

/* Attention of packed documents. Document d has the query rows
 * [q_off[d], q_off[d+1]) and, within its slot [k_off[d], k_off[d+1]) of the
 * key rows, the first k_len[d] (all where k_len is NULL). A document's last
 * query row stands at its last key. Where `causal`, a row sees the keys up to
 * its own position and the first prefix[d] (none where prefix is NULL);
 * otherwise all of its document's. The score of a row at position i and a
 * key at j is
 *   s = scale q.k;  s = cap tanh(s / cap) if cap > 0;
 *   s -= slopes[h] |i - j| if slopes (Hq floats),
 * O = softmax(s) V over the keys that the row sees, lse (Hq, Tq) = log sum
 * exp s. A row that sees nothing, or that no document holds, gets O = 0 and
 * lse = -inf. Query head h reads key head h / (Hq / Hkv). Offsets must not
 * decrease; they are clamped to the Tq and Tk rows. Key and value rows that
 * a row does not see do not reach it, whatever they hold. A value row that it
 * sees and that is not finite makes its O and lse NaN; a key row that is not
 * finite enters its score by the formula (a score of -inf has probability 0,
 * one of +inf or NaN makes the row NaN).
 * D <= 128, Hq a multiple of Hkv, scale > 0. */
int kdec_attn_fwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs,
                  long q_hs, const void* K, long k_rs, long k_hs,
                  const void* V, long v_rs, long v_hs, const int* q_off,
                  const int* k_off, const int* k_len, const int* prefix,
                  int docs, int causal, const float* slopes, float scale,
                  float cap, int Tq, int Tk, int Hq, int Hkv, int D, void* O,
                  long o_rs, long o_hs, float* lse);
/* Its backward from dO, with the forward's O and lse: dQ, dK and dV are
 * overwritten (zeros in rows that nothing sees), dK and dV summed over the
 * query heads of a key head in a fixed order. Scores are formed again; the
 * slopes are constants. A row whose Q, O or dO is not finite, or that sees a
 * key row that is not, has a dQ of NaN, and so have dK and dV of the keys
 * that it sees. */
int kdec_attn_bwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs,
                  long q_hs, const void* K, long k_rs, long k_hs,
                  const void* V, long v_rs, long v_hs, const void* O,
                  long o_rs, long o_hs, const float* lse, const void* dO,
                  long do_rs, long do_hs, const int* q_off, const int* k_off,
                  const int* k_len, const int* prefix, int docs, int causal,
                  const float* slopes, float scale, float cap, int Tq, int Tk,
                  int Hq, int Hkv, int D, void* dQ, long dq_rs, long dq_hs,
                  void* dK, long dk_rs, long dk_hs, void* dV, long dv_rs,
                  long dv_hs);

/* A projection shared by all rows and the low-rank adapters that each row
 * chooses beside it: row t takes adapter a = idx[t], none where idx[t] is
 * outside [0, adapters);
 *   H[t, u*rank + j] = scale[a] sum_i A[a][u*rank + j, i] drop(X)[t, i]
 *   Y[t, r] = W[r, :] . X[t, :] + bias[r] + sum_j B[a][r, j] H[t, u(r)*rank + j]
 * with the output rows cut into `units` units, unit u owning
 * [unit_off[u], unit_off[u+1]) (units+1 ints on the device, from 0 to out:
 * one unit for a plain projection, three for a fused query / key / value,
 * one per AdaIN unit for the stacked style projection). X (T, in) at row
 * stride x_rs, W (out, in), bias (out) or NULL, A (adapters, units*rank, in),
 * B (adapters, out, rank), scale (adapters floats), Y (T, out) at y_rs.
 * p > 0 drops inputs of the adapters (not of W) as kdec_dropout does with
 * this seed and offset. H (T, units*rank floats; zero rows where no adapter
 * is chosen) is written when not NULL, for the backward.
 * An adapter's values reach the rows that choose it and their unit's outputs,
 * whatever they hold; an infinity comes out infinite.
 * More than 64 rows are sorted by adapter, by one block per adapter that looks
 * at all of them.
 * rank <= 128, units <= 4096, in and out <= 2^24, adapters <= 2^20. */
int kdec_adapter_fwd(kdec_ctx* ctx, int dtype, const void* X, long x_rs,
                     const void* W, const void* bias, const void* A,
                     const void* B, const float* scale, const int* idx,
                     const int* unit_off, int T, int in, int out,
                     int adapters, int units, int rank, float p, long seed,
                     long offset, float* H, void* Y, long y_rs);
/* Its backward from dY (T, out) and the forward's H, W and bias frozen:
 *   dH[t, u*rank+j] = scale[a] sum_{r in u} B[a][r, j] dY[t, r]
 *   dX = dY W + drop(A[a]^T dH)
 *   dA[a] = beta dA[a] + sum_{t of a} dH[t]^T drop(X)[t]
 *   dB[a][r, j] = beta dB[a][r, j]
 *                 + sum_{t of a} dY[t, r] H[t, u(r)*rank + j]
 * dA and dB are floats of A's and B's shapes; adapters that no row chooses
 * get zeros (beta = 0: overwritten, what they held is not read). dX (T, in)
 * at dx_rs. dX, or dA and dB together, may be NULL. The rows' shares of dA and
 * dB (more than 256 rows) take the room of up to 513 adapters' gradients beside
 * that of dA and dB themselves. */
int kdec_adapter_bwd(kdec_ctx* ctx, int dtype, const void* X, long x_rs,
                     const void* W, const void* A, const void* B,
                     const float* scale, const int* idx, const int* unit_off,
                     int T, int in, int out, int adapters, int units,
                     int rank, float p, long seed, long offset,
                     const float* H, const void* dY, long dy_rs, void* dX,
                     long dx_rs, float* dA, float* dB, float beta);

/* The calls from here on can be captured into a graph once they were made with
 * the same sizes before (their workspaces are then the context's, which keeps
 * them until it is destroyed). Graphs that were captured on one stream share these
 * with each other and with the context's calls on it, so they are replayed on that
 * stream, and the context outlives them. Memory from kdec_malloc (the drop-in
 * layer's tensors among it) and calls on another stream get none of them. */

/* Embedding: Y[t] = scale * table[ids[t]] (table (vocab, cols) at row stride
 * t_rs, Y (T, cols) at y_rs); an id outside [0, vocab) gives a row of zeros. */
int kdec_embed_fwd(kdec_ctx* ctx, int dtype, const void* table, long t_rs,
                   const int* ids, int T, int vocab, int cols, float scale,
                   void* Y, long y_rs);
/* Its table's gradient, dtable (vocab, cols) floats:
 *   dtable[v] = beta dtable[v] + scale sum_{t: ids[t] = v} dY[t]
 * (beta = 0: overwritten, what it held is not read). Every sum has one order,
 * the tokens sorted by id and cut into pieces: the same bits every time. */
int kdec_embed_bwd(kdec_ctx* ctx, int dtype, const void* dY, long dy_rs,
                   const int* ids, int T, int vocab, int cols, float scale,
                   float* dtable, float beta);

/* The norms before and after a block with its gate and residual, rows of C:
 *   u = N_post(Z) if `post`, else Z;  R = x_scale X + scale gate u
 *   Y = N_pre(R) if `pre`
 * N(v) = v / sqrt(mean(v^2) + eps) * w + b, or where `layer` that of v less
 * its mean; w1, b1 are N_post's (NULL: ones, zeros), w2, b2 N_pre's. gate is
 * NULL (ones), a row for all (gate_rs 0) or a row each. Z may be NULL: then
 * Y = N_pre(X) alone, without post, gate and R. stats (T, 4 floats, aligned to
 * 16 bytes) is written when not NULL, for the backward. R enters N_pre before
 * its rounding. R may be X or Z, and Y either of them. Sums are floats: squares
 * past 2^127 overflow. C <= 8192, eps > 0; up to 2^26 - 4 rows of up
 * to 512 columns, fewer of more. */
int kdec_resnorm_fwd(kdec_ctx* ctx, int dtype, int layer, const void* X,
                     long x_rs, const void* Z, long z_rs, const void* gate,
                     long gate_rs, int post, const void* w1, const void* b1,
                     int pre, const void* w2, const void* b2, float eps,
                     float scale, float x_scale, int T, int C, void* R,
                     long r_rs, void* Y, long y_rs, float* stats);
/* Its backward from dR (NULL: none) and dY (with `pre`) and the forward's
 * inputs and stats. dX, dZ (with Z) and, where each row has a gate of its own,
 * dgate are (T, C) without gaps, of the tensors' type; the gradient of one row
 * of gates for all, dw1, db1, dw2 and db2 (each may be NULL) are C floats,
 * overwritten, their sums over the rows in one order. R is formed again from X
 * and Z, so these must hold what the forward read. */
int kdec_resnorm_bwd(kdec_ctx* ctx, int dtype, int layer, const void* X,
                     long x_rs, const void* Z, long z_rs, const void* gate,
                     long gate_rs, int post, const void* w1, const void* b1,
                     int pre, const void* w2, const void* b2, float eps,
                     float scale, float x_scale, int T, int C,
                     const float* stats, const void* dR, long dr_rs,
                     const void* dY, long dy_rs, void* dX, void* dZ,
                     void* dgate, float* dw1, float* db1, float* dw2,
                     float* db2);

/* A key and value cache in 8 bits. A token's values in one head are held as
 * integers: scale s = max(max|x| / 127, 2^-126) in float, codes x / s to the
 * nearest, ties to even; a token with a value that is not finite has the scale
 * NaN. Codes Kc, Vc: Tk rows of H heads, strides in bytes, each row of a head
 * code_width = D rounded up to 16 bytes (those past D are written as zeros);
 * base and strides are multiples of 16, a row stride is below 2^24. k_scale and
 * v_scale: (H, Tk) floats.
 *
 * Writes the rows of K and V (Tq, H, D): document d's rows
 * [q_off[d], q_off[d+1]) are the last of its k_len[d] filled keys in the slot
 * [k_off[d], k_off[d+1]), as kdec_attn_fwd sees them. Rows that no document
 * holds, or that lie before the slot's first key, are not written. */
int kdec_cache_write(kdec_ctx* ctx, int dtype, const void* K, long k_rs,
                     long k_hs, const void* V, long v_rs, long v_hs,
                     const int* q_off, const int* k_off, const int* k_len,
                     int docs, int Tq, int Tk, int H, int D, void* Kc,
                     long kc_rs, long kc_hs, void* Vc, long vc_rs, long vc_hs,
                     float* k_scale, float* v_scale);
/* Reads them back: the rows that the same arguments wrote, scale times code,
 * into K and V (Tq, H, D); zeros in rows that it would not have written. */
int kdec_cache_read(kdec_ctx* ctx, int dtype, const void* Kc, long kc_rs,
                    long kc_hs, const void* Vc, long vc_rs, long vc_hs,
                    const float* k_scale, const float* v_scale,
                    const int* q_off, const int* k_off, const int* k_len,
                    int docs, int Tq, int Tk, int H, int D, void* K, long k_rs,
                    long k_hs, void* V, long v_rs, long v_hs);
/* kdec_attn_fwd over such a cache: the same documents, masks, scores and
 * outputs, keys and values scale times code (Q, O of `dtype`). A row that sees
 * a token whose key or value scale is not finite becomes NaN. Weights up to 2^8
 * are summed before the division: values past 2^119 over the number of keys may
 * overflow, and make their row NaN. */
int kdec_attn_cache_fwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs,
                        long q_hs, const void* Kc, long kc_rs, long kc_hs,
                        const void* Vc, long vc_rs, long vc_hs,
                        const float* k_scale, const float* v_scale,
                        const int* q_off, const int* k_off, const int* k_len,
                        const int* prefix, int docs, int causal,
                        const float* slopes, float scale, float cap, int Tq,
                        int Tk, int Hq, int Hkv, int D, void* O, long o_rs,
                        long o_hs, float* lse);

#ifdef __cplusplus
}
#endif

#endif /* KDEC_H */
