/*
 * rnnt_mi355x.h -- C ABI of librnnt_mi355x.so, a from-scratch RNN-Transducer
 * loss (forward-backward + gradient) for AMD MI355X (gfx950).
 *
 * The boundary this library replaces is the one call the reference makes into
 * its un-vendored dependency:
 *
 *     from warprnnt_tensorflow import rnnt_loss
 *     rnnt_loss(acts, labels, input_length, label_length, blank_label=39)
 *         reference rnnt/base/util.py:70-72   (Util.rnnt_lambda_func_v2)
 *         reference rnnt/base/util.py:113-115 (Util.rnnt_lambda_func)
 *
 * together with the tf.nn.log_softmax the reference applies just before it
 * (util.py:66, util.py:109) and the gradient TensorFlow chains back through
 * both during training (rnnt/train.py:151-157), including the per-utterance
 * upstream factor of the Keras batch mean (rnnt/keras_model.py:215-217).
 *
 * Conventions
 *   - every pointer except `host_flags` and `out_bytes` is a DEVICE pointer;
 *   - logits: float32 [B, maxT, maxU1, V], contiguous, V fastest
 *     (acts of util.py:63 / :109 -- raw joint logits or log-probabilities:
 *     log-softmax is idempotent so both give the same costs and gradients);
 *   - labels: int32 [B, maxU1-1]; in_len, lab_len: int32 [B]
 *     (dtypes of reference rnnt/keras_model.py:125-127);
 *   - blank: any index in [0, V) (util.py:72 hard-codes 39);
 *   - costs: float32 [B], cost_b = -log P(labels_b | logits_b);
 *   - the gradient is d(sum_b grad_scale[b]*cost_b)/d(logits), i.e. it already
 *     contains the log-softmax backward; cells with t >= in_len[b] or
 *     u > lab_len[b] receive exact zeros;
 *   - the caller owns every buffer including the workspace; no entry point
 *     allocates or frees device memory, all work is enqueued on `hip_stream`
 *     (a hipStream_t, NULL = default stream; its device must be the current
 *     one) and, except rnnt_mi355x_read_status / rnnt_mi355x_read_stats, none
 *     synchronises; the only state the library keeps between calls is the
 *     default pruning threshold of rnnt_mi355x_set_prune_log2 (used only by
 *     calls that pass NaN as their own) and, per device, the address of the
 *     built-in workspace of rnnt_mi355x_loss_grad_static;
 *   - prune_log2 (last argument of every entry point that writes a gradient):
 *     the gradient pass writes an element as exact zero without computing it
 *     when it can bound its magnitude by grad_scale * 2^prune_log2 from the
 *     lattice state alone (see rnnt_mi355x_set_prune_log2).  Accepted:
 *     [-inf, -16]; -inf computes every element; NaN (the C macro NAN) = the
 *     process default.  A per-call input: concurrent calls with different
 *     thresholds do not affect each other;
 *   - every function returns an rnnt_mi355x_status; nothing throws or aborts.
 *
 * Limits: 1 <= maxU1 <= 1024, B*maxT*maxU1 < 2^31, (maxT+maxU1+32)*maxU1 < 2^27,
 * V >= 1.  Element offsets into logits are 64-bit.
 */
#ifndef RNNT_MI355X_H_
#define RNNT_MI355X_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  RNNT_MI355X_OK = 0,
  RNNT_MI355X_INVALID_VALUE = 1,    /* null pointer, non-positive size, blank outside [0,V) ... */
  RNNT_MI355X_UNSUPPORTED_SIZE = 2, /* beyond a limit stated in this header */
  RNNT_MI355X_LAUNCH_FAILURE = 3,   /* HIP reported an error at launch/copy */
  RNNT_MI355X_BAD_INPUT_DATA = 4    /* device-side validation failed (see read_status) */
} rnnt_mi355x_status;

/* bits of the device-side validation word returned by rnnt_mi355x_read_status */
#define RNNT_MI355X_FLAG_BAD_LENGTH 1 /* in_len[b] outside [1,maxT] or lab_len[b] outside [0,maxU1-1] */
#define RNNT_MI355X_FLAG_BAD_LABEL 2  /* a used label outside [0,V) (clamped to 0 for the computation) */

/* Bytes of workspace the other entry points need for a batch of this shape.
 * Replaces the scratch allocation the dependency's op does internally behind
 * rnnt_loss (call sites reference util.py:70-72, 113-115). */
int rnnt_mi355x_workspace_bytes(int B, int maxT, int maxU1, size_t* out_bytes);

/* costs[b] = -log P(labels_b | logits_b): the value rnnt_loss returns at
 * reference util.py:71 / :114 (then reshaped to [B] at util.py:74 / :117).
 * Leaves the lattice state in `workspace` for a later rnnt_mi355x_backward*. */
int rnnt_mi355x_forward(const float* logits, const int32_t* labels, const int32_t* in_len, const int32_t* lab_len,
                        int B, int maxT, int maxU1, int V, int blank, float* costs, void* workspace, void* hip_stream);

/* grad = d(sum_b grad_scale[b]*cost_b)/d(logits) from the state a preceding
 * rnnt_mi355x_forward on the SAME logits left in `workspace`.  `grad` may be
 * the logits buffer itself (in place).  grad_scale: [B] floats or NULL (= 1);
 * 1/B reproduces the Keras mean of reference keras_model.py:215-217.  This is
 * the gradient registered on the dependency's op, the multiply by the
 * upstream gradient and the log_softmax backward of util.py:66 / :109 in one
 * pass. */
int rnnt_mi355x_backward(const float* logits, float* grad, const int32_t* labels, const int32_t* in_len,
                         const int32_t* lab_len, int B, int maxT, int maxU1, int V, int blank, const float* grad_scale,
                         void* workspace, void* hip_stream, float prune_log2);

/* Same, overwriting the logits with their gradient. */
int rnnt_mi355x_backward_inplace(float* logits_inout, const int32_t* labels, const int32_t* in_len,
                                 const int32_t* lab_len, int B, int maxT, int maxU1, int V, int blank,
                                 const float* grad_scale, void* workspace, void* hip_stream, float prune_log2);

/* rnnt_mi355x_forward / rnnt_mi355x_backward on tensors whose utterances are
 * `*_batch_stride` ELEMENTS apart (>= maxT*maxU1*V; inside an utterance the
 * layout stays [maxT, maxU1, V] contiguous).  This is how the crop of the
 * first two frames, `acts[:, 2:, :, :]` at reference util.py:63 (and
 * `y_trans[:, 2:, :]` at util.py:101), is taken without copying the tensor:
 * pass the address of frame 2 of utterance 0, the uncropped batch stride and
 * maxT = T0 - 2.  `grad` may alias `logits` when both strides are equal. */
int rnnt_mi355x_forward_strided(const float* logits, size_t logits_batch_stride, const int32_t* labels,
                                const int32_t* in_len, const int32_t* lab_len, int B, int maxT, int maxU1, int V,
                                int blank, float* costs, void* workspace, void* hip_stream);
int rnnt_mi355x_backward_strided(const float* logits, size_t logits_batch_stride, float* grad,
                                 size_t grad_batch_stride, const int32_t* labels, const int32_t* in_len,
                                 const int32_t* lab_len, int B, int maxT, int maxU1, int V, int blank,
                                 const float* grad_scale, void* workspace, void* hip_stream, float prune_log2);

/* The crop itself as an argument: logits_full / grad_full are dense
 * [B, T0, maxU1, V] tensors and the lattice uses frames t_offset .. T0-1 of every
 * utterance (`acts[:, shift:, :, :]`, `input_length -= shift` at reference
 * util.py:62-64; in_len counts frames of the crop, the workspace is the one of
 * rnnt_mi355x_workspace_bytes(B, T0 - t_offset, maxU1)).  The backward writes
 * zeros into the t_offset skipped frames of grad_full (which may be
 * logits_full itself).  Unlike the *_strided forms this tells the library
 * that the tensor is dense, which the small-vocabulary kernels (V <= 128: the
 * reference's own 40/62-symbol vocabularies) need. */
int rnnt_mi355x_forward_cropped(const float* logits_full, const int32_t* labels, const int32_t* in_len,
                                const int32_t* lab_len, int B, int T0, int t_offset, int maxU1, int V, int blank,
                                float* costs, void* workspace, void* hip_stream);
int rnnt_mi355x_backward_cropped(const float* logits_full, float* grad_full, const int32_t* labels,
                                 const int32_t* in_len, const int32_t* lab_len, int B, int T0, int t_offset,
                                 int maxU1, int V, int blank, const float* grad_scale, void* workspace,
                                 void* hip_stream, float prune_log2);

/* forward + backward_inplace in one call: what one training step of
 * reference rnnt/train.py:151-157 spends in the loss layer. */
int rnnt_mi355x_loss_grad(float* logits_inout, const int32_t* labels, const int32_t* in_len, const int32_t* lab_len,
                          int B, int maxT, int maxU1, int V, int blank, const float* grad_scale, float* costs,
                          void* workspace, void* hip_stream, float prune_log2);

/* rnnt_mi355x_loss_grad with optional hipEvent_t handles recorded on
 * `hip_stream` around its kernels: events4[0] before the log-sum-exp pass,
 * [1] between it and the lattice sweep, [2] between the sweep and the gradient
 * pass, [3] after the gradient pass (events4 NULL, or any entry NULL = not
 * recorded).  A measurement aid for callers that want each pass timed on the
 * launch stream; it has no counterpart in the reference. */
int rnnt_mi355x_loss_grad_events(float* logits_inout, const int32_t* labels, const int32_t* in_len,
                                 const int32_t* lab_len, int B, int maxT, int maxU1, int V, int blank,
                                 const float* grad_scale, float* costs, void* workspace, void* hip_stream,
                                 float prune_log2, void* const* events4);

/* rnnt_mi355x_loss_grad for callers that cannot allocate or own device
 * scratch memory: code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc.  It has no counterpart in the reference.  The
 * workspace is an array inside the library's code object
 * (RNNT_MI355X_STATIC_WORKSPACE_BYTES; every GPU the library runs on holds one
 * copy until the process ends), so the call takes no workspace and calls no
 * hipMalloc / hipFree or any other allocating routine.  Shapes whose
 * rnnt_mi355x_workspace_bytes exceeds that size are rejected with
 * RNNT_MI355X_UNSUPPORTED_SIZE.  Optional device outputs replace the calls
 * that would need the workspace pointer: scalars2 (2 doubles: what
 * rnnt_mi355x_reduce_scalars returns) and flags_out (int32: the validation
 * word of rnnt_mi355x_read_status); either may be NULL.  All calls on one GPU
 * share that GPU's array: calls that overlap on one GPU (two streams, two
 * threads) race; calls on one stream are ordered and need no clearing in
 * between (every word the kernels read is written by the same call).  The
 * first call on a device looks the array's address up
 * (hipGetSymbolAddress); make it outside graph capture. */
#define RNNT_MI355X_STATIC_WORKSPACE_BYTES (32u << 20)
int rnnt_mi355x_loss_grad_static(float* logits_inout, const int32_t* labels, const int32_t* in_len,
                                 const int32_t* lab_len, int B, int maxT, int maxU1, int V, int blank,
                                 const float* grad_scale, float* costs, double* scalars2, int32_t* flags_out,
                                 void* hip_stream, float prune_log2);

/* ---- fused additive joint ------------------------------------------------
 * The loss of the reference's additive-joint model, Util.rnnt_lambda_func
 * (reference rnnt/base/util.py:107-115): acts = log_softmax(y_trans[B,T,1,V] +
 * y_pred[B,1,U+1,V]) followed by rnnt_loss(acts, ...), WITHOUT forming the
 * [B,T,U+1,V] tensor.  f = y_trans [B,maxT,V] (utterances f_batch_stride
 * elements apart, >= maxT*V: pass the address of frame 2 and the uncropped
 * stride for the crop of util.py:101), g = y_pred [B,maxU1,V] contiguous.
 * The backward writes d(sum_b grad_scale[b]*cost_b)/df and /dg directly (what
 * TensorFlow obtains by reducing the [B,T,U+1,V] gradient over u and over t,
 * util.py:107-109).  Needs the larger workspace of
 * rnnt_mi355x_joint_workspace_bytes (which depends on V: it holds exp(f - max f)
 * and exp(g - max g), the operands of the matrix-core contractions the sums over
 * V, u and t are computed as); V <= 4096.  rnnt_mi355x_reduce_scalars
 * after a joint backward returns the cost sum and 0 for the norm. */
int rnnt_mi355x_joint_workspace_bytes(int B, int maxT, int maxU1, int V, size_t* out_bytes);
int rnnt_mi355x_joint_forward(const float* f, size_t f_batch_stride, const float* g, const int32_t* labels,
                              const int32_t* in_len, const int32_t* lab_len, int B, int maxT, int maxU1, int V,
                              int blank, float* costs, void* workspace, void* hip_stream);
int rnnt_mi355x_joint_backward(const float* f, size_t f_batch_stride, const float* g, const int32_t* labels,
                               const int32_t* in_len, const int32_t* lab_len, int B, int maxT, int maxU1, int V,
                               int blank, const float* grad_scale, float* df, size_t df_batch_stride, float* dg,
                               void* workspace, void* hip_stream, float prune_log2);

/* ---- first layer of the fully-connected joint --------------------------------
 * The reference's FC-joint model tiles the encoder output [B,T,He] and the
 * prediction-network output [B,U+1,Hd] into [B,T,U+1,He+Hd]
 * (Util.concatenate_lambda, reference rnnt/base/util.py:76-90) and applies
 * Dense(H, tanh) to it (first layer of KerasModel.get_fc, reference
 * rnnt/keras_model.py:83-104).  Because that layer is linear in the
 * concatenation, the caller computes pe = enc * W1[:He] ([B,T,H]) and
 * pd = dec * W1[He:] + b1 ([B,U1,H]) with two small matrix products and these
 * entry points do the rest without the tiled tensor:
 *   forward : h[b,t,u,:] = tanh(pe[b,t,:] + pd[b,u,:])              h: [B,T,U1,H]
 *   backward: d = dh * (1 - h^2) (h recomputed from pe, pd; dh: [B,T,U1,H]),
 *             dpe[b,t,:] = sum_u d, dpd[b,u,:] = sum_t d            (fixed summation order)
 * All tensors float32, contiguous.  The backward needs
 * rnnt_mi355x_fc_joint_workspace_bytes of scratch.  H <= 1536. */
int rnnt_mi355x_fc_joint_workspace_bytes(int B, int T, int U1, int H, size_t* out_bytes);
int rnnt_mi355x_fc_joint_forward(const float* pe, const float* pd, int B, int T, int U1, int H, float* h,
                                 void* hip_stream);
int rnnt_mi355x_fc_joint_backward(const float* pe, const float* pd, const float* dh, int B, int T, int U1, int H,
                                  float* dpe, float* dpd, void* workspace, void* hip_stream);

/* ---- Dense layers over the joint lattice -------------------------------------
 * y[M,N] = act(x[M,K] W[K,N] + bias[N]) for a very tall M = B*T*(U+1) and
 * K, N <= 128: the layers after the first one of KerasModel.get_fc (reference
 * rnnt/keras_model.py:83-104; TimeDistributed(Dense), tanh on all but the last,
 * Keras kernel layout [in, out]).  act: 0 linear, 1 tanh.  All float32,
 * contiguous.  The backward takes the forward output y (used when act == 1)
 * and the upstream gradient dy[M,N] and writes dx[M,K] (skipped when NULL),
 * dw[K,N] and db[N] (skipped when dw is NULL; db may be NULL on its own);
 * dw/db need rnnt_mi355x_dense_workspace_bytes of scratch and are summed in a
 * fixed order. */
int rnnt_mi355x_dense_workspace_bytes(long long M, int K, int N, size_t* out_bytes);
int rnnt_mi355x_dense_forward(const float* x, const float* w, const float* bias, long long M, int K, int N, int act,
                              float* y, void* hip_stream);
int rnnt_mi355x_dense_backward(const float* x, const float* w, const float* y, const float* dy, long long M, int K,
                               int N, int act, float* dx, float* dw, float* db, void* workspace, void* hip_stream);

/* ---- decoder step ---------------------------------------------------------
 * out[n, :] = log_softmax(f[f_index[n], :] + g[g_index[n], :]) over V, n < n_rows:
 * the joint + Util.softmax(out, is_log=True) the reference's beam search
 * evaluates one vector at a time (reference rnnt/rnnt_decoder.py:156-158,
 * 170-171, 200-202; rnnt/base/util.py:295-309), batched over any number of
 * (encoder frame, hypothesis) pairs.  f: [f_rows,V], g: [g_rows,V] or NULL (then
 * out = log_softmax(f rows)); the index arrays are int32 [n_rows] or NULL (= row
 * n).  An index outside its tensor sets *bad_index_flag (device int32, zeroed by
 * the caller) to 1 and row 0 is used instead.  out: [n_rows,V]. */
int rnnt_mi355x_joint_log_softmax(const float* f, int f_rows, const float* g, int g_rows, const int32_t* f_index,
                                  const int32_t* g_index, int n_rows, int V, float* out, int32_t* bad_index_flag,
                                  void* hip_stream);

/* ---- operators around the joint network: dropout, Dense layer, beam step -----------
 * They take float32, bfloat16 and float16 tensors (`dtype`); every sum, softmax statistic
 * and score is held in 32 bits or more. */
#define RNNT_MI355X_FP32 0
#define RNNT_MI355X_BF16 1
#define RNNT_MI355X_FP16 2

/* y = x * m / keep for the Dropout layers of get_fc (reference
 * rnnt/keras_model.py:102-103), keep = 1 - drop16/65536.  x: [rows, cols], rows
 * x_stride >= cols elements apart; y: dense, may be x itself when x_stride ==
 * cols.  The mask is drawn, never stored: element (r, c) uses bits
 * 16*(c%2) .. +15 of word (c%8)/2 of Philox4x32-10 at counter (c/8, r, offset low,
 * offset high), key (seed low, seed high), and is kept when they are >= drop16.
 * The backward pass is the same call on the upstream gradient.  offset_dev
 * (nullable, device) replaces `offset`: a captured graph draws a new mask on every
 * replay when the caller advances it. */
int rnnt_mi355x_dropout(const void* x, long long x_stride, void* y, long long rows, int cols, int dtype, int drop16,
                        uint64_t seed, uint64_t offset, const uint64_t* offset_dev, void* hip_stream);

/* Dense layer of any width with its epilogue (TimeDistributed(Dense) and Dropout of
 * get_fc, reference rnnt/keras_model.py:83-104; rnnt_mi355x_dense_* above are its
 * float32 special case for widths up to 128):
 *   z = x kernel + bias,  y = residual + dropout(act(z))
 *   dz = dropout'(dy) act'(z), dx = dz kernel^T, dkernel = x^T dz, dbias = sum over rows of dz
 * (d residual is dy).  x: [rows, in], kernel: [in, out] (Keras), residual, y, aux,
 * dy: [rows, out]; all of one `dtype`, last dimension contiguous, rows *_stride elements
 * apart (y and aux dense).  float32 products are accurate to float32 rounding (three
 * bfloat16 parts an operand; operands below 2^-102 lose their last places), sums are
 * float32; in 16 bits dz is rounded to the type before its two products.  bias, residual and aux may be NULL.
 * act: RNNT_MI355X_ACT_*; gelu is z Phi(z), off by (24 + 2 z^2) 2^-24 of itself in float32 and by 2^-13 (2^-9.8 below
 * z = -5.9) next to the type's rounding in 16 bits; results below 2^-122 may be 0.  Dropout as rnnt_mi355x_dropout
 * draws it for [rows, out] (drop16 0: none).
 * The backward pass takes the same layer and needs, unless act is linear, aux as the
 * forward pass wrote it: the pre-activation, float32 for float32 and float16 layers,
 * float16 for bfloat16 ones.  Without residual, relu layers and float32 tanh layers may
 * go without it (aux NULL in both passes); y is read instead.  dx, dkernel, dbias may
 * be NULL.  Sums run in a fixed order: equal calls give equal bits.
 * Workspace: the sizes rnnt_mi355x_layer_workspace_bytes gives for the very pointers
 * and strides (their alignment decides the kernels), on a 256-byte boundary; forward 0:
 * may be NULL.  y may be
 * residual itself when its stride is `out`.  rows <= 2^30 - 64, in, out <= 2^24. */
#define RNNT_MI355X_ACT_LINEAR 0
#define RNNT_MI355X_ACT_TANH 1
#define RNNT_MI355X_ACT_RELU 2
#define RNNT_MI355X_ACT_GELU 3
#define RNNT_MI355X_ACT_SILU 4
typedef struct {
  const void *x, *kernel, *bias, *residual;
  void *y, *aux;
  long long x_stride, kernel_stride, residual_stride, rows;
  int in, out, dtype, act, drop16;
  uint64_t seed, offset;
  const uint64_t* offset_dev;
} rnnt_mi355x_layer;
int rnnt_mi355x_layer_workspace_bytes(const rnnt_mi355x_layer* layer, const void* dy, long long dy_stride,
                                      size_t* forward_bytes, size_t* backward_bytes);
int rnnt_mi355x_layer_forward(const rnnt_mi355x_layer* layer, void* workspace, void* hip_stream);
int rnnt_mi355x_layer_backward(const rnnt_mi355x_layer* layer, const void* dy, long long dy_stride, void* dx, void* dkernel,
                               void* dbias, void* workspace, void* hip_stream);

/* One step of a beam search (what reference rnnt/rnnt_decoder.py:95-233 does with the
 * log-probabilities of its inner step).  logits: [B, K, V] (last dimension
 * contiguous, strides in elements), enc: [B, V] or NULL, added to the logits of all
 * beams of an utterance (sum rounded to float32); scores: [B, K]; allowed: bytes
 * [B, V] or NULL, zero forbids a symbol (its logit is not looked at and has no part in
 * the softmax; allowed_batch_stride 0: one mask for all utterances); finished: bytes
 * [B, K] or NULL: such a beam offers itself alone, with its score, at symbol `end`.
 *   total = scores + x - log sum exp x          (ordered in float64; the logarithm is off by at most 2^-21.6)
 * and the `width` largest totals of an utterance, ties to the lowest k*V + v, go to
 * out_scores / out_parent / out_token [B, width]; places without a candidate hold
 * -inf, -1, -1.  A beam whose score is NaN or beyond +-2^30 is empty; so is one whose
 * allowed logits hold a NaN or +inf, or nothing above -inf.  K, width <= 64,
 * K*V <= 2^31 - 2^16, B < 2^22, B*K*(V/2048 rounded up) < 2^26 where V > 2048.
 * `workspace`: rnnt_mi355x_beam_select_workspace_bytes
 * on a 16-byte boundary (0: may be NULL). */
int rnnt_mi355x_beam_select_workspace_bytes(int B, int K, int V, int width, size_t* out_bytes);
int rnnt_mi355x_beam_select(const void* logits, long long logits_batch_stride, long long logits_beam_stride, int dtype,
                            const void* enc, long long enc_batch_stride, const float* scores, const uint8_t* allowed,
                            long long allowed_batch_stride, const uint8_t* finished, int end, int B, int K, int V,
                            int width, float* out_scores, int32_t* out_parent, int32_t* out_token, void* workspace,
                            void* hip_stream);

/* dst[o, b, w, :] = src[o, b, parent[b, w], :], zeros where parent is outside [0, K):
 * the hypotheses' network states in the order beam_select gave them, up to
 * RNNT_MI355X_REORDER_MAX tensors in one launch.  src: rows of row_bytes bytes at
 * the byte strides given; dst: dense [outer, B, width, row_bytes], not
 * overlapping any src. */
#define RNNT_MI355X_REORDER_MAX 16
typedef struct {
  const void* src;
  void* dst;
  long long outer, outer_stride, batch_stride, beam_stride, row_bytes; /* strides in bytes */
} rnnt_mi355x_reorder_tensor;
int rnnt_mi355x_beam_reorder(const rnnt_mi355x_reorder_tensor* tensors, int n_tensors, const int32_t* parent, int B,
                             int K, int width, void* hip_stream);

/* out2[0] = sum_b costs[b], out2[1] = sum of squared gradient elements of the
 * last backward on this workspace (both float64, device memory).  These are
 * the two scalars a data-parallel caller all-reduces: the batch loss of
 * reference keras_model.py:215-217 and the gradient norm the optimizer's
 * clipnorm needs (reference keras_model.py:209-213). */
int rnnt_mi355x_reduce_scalars(const float* costs, int B, void* workspace, double* out2, void* hip_stream);

/* Pruning of the gradient pass.  With gamma = P(path through (t,u) | labels)
 * the occupancy of a lattice cell, p(v) the softmax of its row and p_max the
 * largest of them, the gradient of the row is grad_scale * (gamma*p(v) - the
 * blank's / the label's transition probability at those two v).  Every element
 * is bounded by grad_scale*gamma, and every element except the blank's and
 * the label's by grad_scale*gamma*p_max.  With T = 2^log2_threshold:
 *   gamma < T            the whole row is written as exact zeros;
 *   gamma*p_max < T      (diffuse posteriors) the row is written as exact
 *                        zeros except its blank and label entries, which are
 *                        written exactly from the lattice state alone;
 * in both cases the row's logits are not read a second time, and no element
 * written as zero exceeds grad_scale*T in magnitude.  The fused additive joint
 * applies the first rule only (it reads nothing twice: pruned cells are left
 * out of its contractions), the kernels for V <= 128 whose rows are no
 * multiple of 16 bytes likewise.  Default -28 (T = 3.7e-9); accepted range
 * [-inf, -16] (-inf: every element is computed).  This sets the process-wide
 * default that calls passing NaN as their prune_log2 use; it takes effect for
 * calls made afterwards.  A tuning knob without counterpart in the reference
 * (whose dependency computes every element). */
int rnnt_mi355x_set_prune_log2(float log2_threshold);
float rnnt_mi355x_get_prune_log2(void);

/* *host_cells = lattice cells the last backward on this workspace visited,
 * *host_pruned = how many of their rows were not read a second time (pruned or
 * sparse, see rnnt_mi355x_set_prune_log2).  Runs a
 * small kernel and waits for the stream.  A measurement aid without
 * counterpart in the reference. */
int rnnt_mi355x_read_stats(void* workspace, uint64_t* host_cells, uint64_t* host_pruned, void* hip_stream);

/* Copies the device-side validation word to *host_flags (an OR of
 * RNNT_MI355X_FLAG_*), waiting for the stream.  Returns
 * RNNT_MI355X_BAD_INPUT_DATA when it is non-zero.  Corresponds to the
 * exception the dependency's op raises on malformed inputs. */
int rnnt_mi355x_read_status(const void* workspace, int32_t* host_flags, void* hip_stream);

/* Human-readable text for a status code (static storage). */
const char* rnnt_mi355x_status_string(int status);

/* ABI version of this header: major*100 + minor. */
int rnnt_mi355x_version(void);

#ifdef __cplusplus
}
#endif
#endif /* RNNT_MI355X_H_ */
