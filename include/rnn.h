/*
 * rnn.h -- C ABI of the MI355X (gfx950) GEMM core of rustnn.
 *
 * Drop-in boundary for the reference's L2 kernels (lsiddd/rustnn, Rust): each
 * entry point names the reference function it replaces (file:line).  A thin
 * Rust FFI crate (extern "C" + #[link(name = "rnn")]) keeps the reference call
 * sites in conv.rs / attn.rs / linear.rs / nn.rs unchanged (the crate rnn-sys,
 * generated from this header).
 *
 * Conventions
 *  - Every float pointer is a DEVICE pointer (hipMalloc / torch CUDA tensor)
 *    holding IEEE binary32, row-major, tightly packed unless a stride says
 *    otherwise.  Shapes are element counts.
 *  - Work is enqueued on the context's stream; calls return once the work is
 *    enqueued (use rnn_ctx_synchronize to wait).  The library keeps no pointer
 *    after a call returns.
 *  - Return value: RNN_OK (0) or a negative RNN_E_* code.  rnn_ctx_last_error
 *    gives the message.  The reference aborts on a bad shape (slice bounds
 *    panic, panic=abort); the Rust shim maps a non-zero status to panic!.
 *  - Results are deterministic: every reduction (split-K, dW over images,
 *    attention dtau/drel over images) runs in a fixed order.
 *  - One stream per context; a context may be used from several host threads
 *    (calls are serialised by a per-context lock).
 */
#ifndef RNN_H
#define RNN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    RNN_OK = 0,
    RNN_E_INVALID = -1,     /* bad shape / argument */
    RNN_E_NULL = -2,        /* required pointer is NULL */
    RNN_E_HIP = -3,         /* HIP runtime error (message has hipGetErrorString) */
    RNN_E_NOMEM = -4,       /* device workspace allocation failed */
    RNN_E_UNSUPPORTED = -5, /* shape outside what the kernels implement */
};

typedef struct rnn_ctx rnn_ctx;

/* ------------------------------------------------------------- context */
/* Replaces the process-wide rayon pool + thread-local scratch
 * (main.rs:41-48, gemm.rs:411-420): one device, one stream, one workspace. */
int rnn_ctx_create(int device, rnn_ctx **out);
/* Runs any reductions the deferral below still holds (rnn_ctx_flush), waits
 * for the stream, then frees the context; returns the flush's status. */
int rnn_ctx_destroy(rnn_ctx *ctx);
/* Use `stream` (a hipStream_t; NULL = the null stream) for later calls. */
int rnn_ctx_set_stream(rnn_ctx *ctx, void *stream);
/* Deferred parameter-gradient reductions (no counterpart in the reference:
 * a launch-count device).  While on, the backward entry points whose last
 * step only sums partial results into a parameter gradient leave that step
 * queued: rnn_linear_backward (dW when split over rows, and db),
 * rnn_ln_backward / rnn_ln_backward_add (dgamma, dbeta), the LayerScale
 * backwards (dl), rnn_dwconv3_backward (dw, db), the column sums and
 * rnn_attn_backward up to 64 tokens (dtau, drel).
 * rnn_ctx_flush runs every queued reduction in one launch, in call order,
 * with the same sums in the same order as the immediate path (results are
 * bit-identical); those gradients are complete only after it.  Turning
 * deferral off flushes first.  The partials stay in a context arena that
 * grows (hipMalloc) when a step needs more. */
int rnn_ctx_set_defer(rnn_ctx *ctx, int on);
int rnn_ctx_flush(rnn_ctx *ctx);
void *rnn_ctx_stream(rnn_ctx *ctx);
int rnn_ctx_synchronize(rnn_ctx *ctx);
const char *rnn_ctx_last_error(rnn_ctx *ctx);
const char *rnn_status_string(int status);
/* Bytes of device workspace currently held by the context. */
size_t rnn_ctx_workspace_bytes(rnn_ctx *ctx);

/* Device memory for callers that hold host slices (the Rust shim keeps the
 * reference's Vec<f32> tensors and mirrors them on the device).  No reference
 * counterpart: the reference computes on host memory only. */
int rnn_dev_alloc(rnn_ctx *ctx, size_t bytes, void **out);
int rnn_dev_free(rnn_ctx *ctx, void *p);
/* Host -> device, ordered on the context stream; returns after the copy. */
int rnn_copy_to_device(rnn_ctx *ctx, void *dst_dev, const void *src_host, size_t bytes);
/* Device -> host after all work queued on the context stream. */
int rnn_copy_to_host(rnn_ctx *ctx, void *dst_host, const void *src_dev, size_t bytes);

/* ------------------------------------------------------------ gemm.rs */
/* matmul (gemm.rs:434-493): C[m x n] = op(A) op(B) (+ C if acc).
 * at=0: A is [m x k]; at=1: A is [k x m].  bt=0: B is [k x n]; bt=1: B is
 * [n x k].  m == 0 or n == 0: no-op.  k == 0: C = 0 unless acc. */
int rnn_matmul(rnn_ctx *ctx, size_t m, size_t n, size_t k, const float *a, int at, const float *b,
               int bt, float *c, int acc);

/* gemm_small (gemm.rs:500-545), batched: `count` independent problems,
 * problem i uses a + i*stride_a, b + i*stride_b, c + i*stride_c.  Replaces the
 * per-(image, head) sequential calls made from rayon workers with one launch.
 * k == 0 leaves C untouched (gemm_small quirk). */
int rnn_gemm_small_batched(rnn_ctx *ctx, size_t count, size_t m, size_t n, size_t k,
                           const float *a, size_t stride_a, int at, const float *b,
                           size_t stride_b, int bt, float *c, size_t stride_c, int acc);

/* matmul_dw (gemm.rs:555-598): C[m x n] += A^T B with A [k x m], B [k x n]
 * (dense weight gradient, K = rows). */
int rnn_matmul_dw(rnn_ctx *ctx, size_t m, size_t n, size_t k, const float *a, const float *b,
                  float *c);

/* ------------------------------------------------------------ conv.rs */
/* ConvSpec (conv.rs:9-20); oh/ow follow Conv2d::out_dim (nn.rs:147-150):
 * oh = (h + 2*pad - k)/stride + 1.  W is [cout][cin][k][k] (RowMap order,
 * conv.rs:39-66); x, y, dx, dy are NCHW. */
typedef struct {
    uint32_t cin, cout, k, stride, pad, h, w, oh, ow;
} rnn_conv_spec;

/* Fills oh/ow.  Returns RNN_E_INVALID for k > h + 2*pad, stride 0, ... */
int rnn_conv_spec_init(rnn_conv_spec *sp, uint32_t cin, uint32_t cout, uint32_t k,
                       uint32_t stride, uint32_t pad, uint32_t h, uint32_t w);

/* Conv2d::forward (nn.rs:166-185) -> conv::forward_image (conv.rs:168-203):
 * y[n][cout][oh][ow] = conv(x) (overwritten). */
int rnn_conv2d_forward(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n, const float *x,
                       const float *w, float *y);
/* Conv2d::backward_w (nn.rs:193-227) -> conv::dw_image (conv.rs:277-322):
 * dw[cout][cin*k*k] += sum over images of dY im2col(X)^T. */
int rnn_conv2d_backward_w(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n, const float *dy,
                          const float *x, float *dw);
/* The per-worker half of Conv2d::backward_w (nn.rs:201-219): the batch's
 * dW as *nz partial slabs of cout*cin*k*k floats in `slabs` (slab z: the sum
 * over the pixel tiles workgroup z owns), without the final reduce
 * (nn.rs:220-225).  Adding the slabs in slab order gives what
 * rnn_conv2d_backward_w adds; a train step can fold that sum into its
 * gradient pass.  `slabs` holds rnn_conv2d_backward_w_slab_floats(...)
 * floats (0: no slab plan for the shape -- k not 1 or 3, stride not 1 or 2). */
size_t rnn_conv2d_backward_w_slab_floats(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n);
int rnn_conv2d_backward_w_slabs(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n,
                                const float *dy, const float *x, float *slabs, int *nz);
/* No counterpart in the reference.  For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc): rnn_conv2d_backward_w with its partial slabs in a fixed
 * device scratch array of 16 MiB (RNN_NOALLOC_SCRATCH_BYTES) that the library
 * holds on each device until the process ends, instead of the context's
 * growing workspace.  Same kernels, same summation order, same result.  It
 * calls no hipMalloc / hipFree.  A shape whose slabs need more than the
 * scratch (cout*cin*k*k*4 bytes times the slab count; 9.4 MB for the ResNet
 * convs at batch 128) returns RNN_E_UNSUPPORTED.  Every call on one device
 * shares that scratch.  Outside graph capture the library orders them: a
 * call on another stream than the device's previous call first waits for
 * that call's kernels (hipStreamWaitEvent; one event per device, created by
 * the first such call).  Under graph capture it does not: captured calls
 * that could run at the same time on one GPU race, and the caller orders
 * them (one stream, or graph edges between them).  The scratch address is
 * looked up by the first call on a device (hipGetSymbolAddress); a failed
 * lookup returns RNN_E_HIP from this call only. */
int rnn_conv2d_backward_w_noalloc(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n,
                                  const float *dy, const float *x, float *dw);
/* dX half of Conv2d::backward (nn.rs:230-250) -> conv::dx_image
 * (conv.rs:205-246): dx[n][cin][h][w] = col2im(W^T dY) (overwritten). */
int rnn_conv2d_backward_x(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n, const float *dy,
                          const float *w, float *dx);

/* Packed weights (no counterpart in the reference: for callers that run
 * several forward / dX convolutions between weight updates, such as a train
 * step).  rnn_conv_pack_weights rewrites W into the slab order the forward
 * (dx = 0) or dX (dx = 1) kernel stages through LDS, so that each stage's
 * weights arrive as one contiguous copy; *floats receives the packed size
 * (RNN_E_UNSUPPORTED: the shape has no packed form, use the calls above).
 * The _packed calls take W and its packed copy wp and give results identical
 * to rnn_conv2d_forward / rnn_conv2d_backward_x; wp must be re-packed after
 * W changes. */
int rnn_conv_packed_floats(const rnn_conv_spec *sp, int dx, size_t *floats);
int rnn_conv_pack_weights(rnn_ctx *ctx, const rnn_conv_spec *sp, int dx, const float *w,
                          float *wp);
int rnn_conv2d_forward_packed(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n, const float *x,
                              const float *w, const float *wp, float *y);
int rnn_conv2d_backward_x_packed(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n, const float *dy,
                                 const float *w, const float *wp, float *dx);
/* Packed copies of several convolutions' weights, refreshed together in one
 * launch (no counterpart in the reference: for a network whose convolutions
 * run on packed weights and are re-packed after each weight update, such as
 * the rustvit trunk).  Convolution i has spec specs[i] and weights w[i] (on
 * the device, [cout][cin][k][k]; w[i] must stay allocated, at the same
 * address, while the object lives).  create allocates the packed copies of
 * both directions of every convolution and packs them on the context stream;
 * update re-packs all of them from the current W; get returns convolution
 * i's copy for the forward (dx = 0) or dX (dx = 1) -- for the _packed calls
 * with the same spec -- or NULL when that shape has no packed form. */
typedef struct rnn_conv_packs rnn_conv_packs;
int rnn_conv_packs_create(rnn_ctx *ctx, size_t count, const rnn_conv_spec *specs, const float **w,
                          rnn_conv_packs **out);
int rnn_conv_packs_update(rnn_ctx *ctx, rnn_conv_packs *p);
const float *rnn_conv_packs_get(const rnn_conv_packs *p, size_t i, int dx);
void rnn_conv_packs_destroy(rnn_conv_packs *p);

/* ------------------------------------------------------------ attn.rs */
/* Core (attn.rs:74-84) plus the stride/offset arguments of Core::forward /
 * Core::backward (attn.rs:148-160, 226-242).  Rows of head hd are read at
 * base + r*qstride + qoff + hd*dh (queries) and base + r*kvstride + koff/voff
 * + hd*dh (keys / values).  relidx is a HOST pointer to tq*tk entries
 * (rnn_rel_index); the library uploads it. */
typedef struct {
    uint32_t h, dh, tq, tk;
    size_t qstride, qoff, kvstride, koff, voff;
    uint32_t nrel;
    const uint32_t *relidx;
    int mask_diag;
} rnn_attn_desc;

/* rel_index (attn.rs:53-72): host-side table of th*tw*mh*mw entries;
 * *nrel receives the bias-table length per head. */
int rnn_rel_index(uint32_t th, uint32_t tw, uint32_t mh, uint32_t mw, uint32_t *idx,
                  uint32_t *nrel);

/* Core::forward (attn.rs:148-223): p[n][h][tq][tk] = softmax(tau*QK^T + rel,
 * diagonal masked when mask_diag), o[n][tq][h*dh] = P V. */
int rnn_attn_forward(rnn_ctx *ctx, const rnn_attn_desc *d, size_t n, const float *q,
                     const float *kv, const float *tau, const float *rel, float *p, float *o);
/* Core::backward (attn.rs:226-343): dq, dkv, dtau, drel ACCUMULATE (+=).
 * dq and dkv may alias (disjoint columns, as in SelfAttn, attn.rs:418-438). */
int rnn_attn_backward(rnn_ctx *ctx, const rnn_attn_desc *d, size_t n, const float *q,
                      const float *kv, const float *tau, const float *p, const float *dout,
                      float *dq, float *dkv, float *dtau, float *drel);
/* Core::backward with dq and/or dkv OVERWRITTEN instead of accumulated
 * (flags: RNN_ATTN_SET_DQ, RNN_ATTN_SET_DKV; dtau and drel always
 * accumulate).  SelfAttn::backward (attn.rs:418-438) accumulates into freshly
 * zeroed dq and dkv buffers and CrossAttn::backward (attn.rs:533-551) into a
 * zeroed dq: the same values, without the clearing pass and the read of the
 * old contents.  flags 0 is rnn_attn_backward. */
#define RNN_ATTN_SET_DQ 1u
#define RNN_ATTN_SET_DKV 2u
int rnn_attn_backward_ex(rnn_ctx *ctx, const rnn_attn_desc *d, size_t n, const float *q,
                         const float *kv, const float *tau, const float *p, const float *dout,
                         float *dq, float *dkv, float *dtau, float *drel, uint32_t flags);

/* ------------------------------------------------------- rotary positions */
/* Rotary positions with up to three axes (no counterpart in the reference,
 * whose attention takes its positions from the relative bias): every row holds
 * h heads of dh channels, and the R = p0 + p1 + p2 channel pairs of each head
 * are turned by angles from the row's position.  Axis a owns p_a pairs (axis
 * 0's first); its pair p turns by pos_a * base^(-p / p_a):
 *   (u, v) -> (u cos - v sin, u sin + v cos).
 * Pair j is channels (2j, 2j + 1) when interleaved, else (j, j + R); channels
 * from 2R on are copied.  Angles are computed and reduced in 64 bits, so that
 * far positions keep theirs, and rounded to 32 for the sine and cosine.
 * Rows are read at x + r*xstride + xoff and written at y + r*ystride + yoff;
 * only the h*dh channels of a row are written.  y may be x when strides and
 * offsets agree (in place), else the two must not overlap. */
typedef struct {
    uint32_t h, dh;
    size_t xstride, xoff, ystride, yoff;
    uint32_t axes;       /* 1, 2 or 3 */
    uint32_t p0, p1, p2; /* pairs of each axis (0 beyond axes) */
    uint32_t g0, g1, g2; /* grid of an image's tokens, last axis fastest (1 beyond axes) */
    int interleaved;
    float base;
} rnn_rotary_desc;
/* Checks a description for n images of t tokens with (have_pos) or without
 * explicit positions; host only.  RNN_OK or the code rnn_rotary returns. */
int rnn_rotary_check(const rnn_rotary_desc *d, size_t n, size_t t, int have_pos);
/* Turns the rows of n images of t tokens.  pos NULL: token i of an image sits
 * at its grid coordinates (t = the product of the grid's axes); else pos
 * [n*t][axes] holds every row's position, which may be fractional or negative.
 * inverse: by the negated angles, which is the backward pass (x = dy, y = dx). */
int rnn_rotary(rnn_ctx *ctx, const rnn_rotary_desc *d, size_t n, size_t t, const float *x,
               const float *pos, float *y, int inverse);

/* Norm and rotary position of each head in one pass (no counterpart in the
 * reference): of the h heads of a row (h, dh, the positions and the layouts of x
 * and y as rnn_rotary takes them), the first hq are queries, the rest keys.
 *   x^ = x / sqrt(mean(x^2) + eps),  y = turn(gain x^)
 * gain [2][dh]: queries', keys' (NULL: 1).  Channels past the pairs are normed and
 * not turned.  dh <= 256 (RNN_E_UNSUPPORTED above), eps > 0.  Squares are summed in
 * 64 bits, so that heads of any size keep their norm.  A NaN gives NaN in its
 * head, an infinity in its channel's pair and zeros in the others of its head.
 * y may be x when strides and offsets agree; else it overlaps no operand, though the
 * two may be columns of one buffer (RNN_E_INVALID otherwise). */
int rnn_norm_rotary_forward(rnn_ctx *ctx, const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n,
                            size_t t, const float *x, const float *gain, const float *pos, float *y);
/* Checks the arguments and gives the bytes of device workspace that a backward
 * with dgain needs; host only.  The workspace is the caller's, 256-byte aligned,
 * holds nothing between calls and is not shared by calls that may run at the same
 * time. */
int rnn_norm_rotary_workspace(const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n, size_t t,
                              int have_pos, size_t *bytes);
/* From the forward's input x and dy (rows of dystride floats, heads from dyoff on):
 * dx, laid out as y, is overwritten; dgain [2][dh] (NULL: not wanted) accumulates,
 * in a fixed order.  dx may be dy when their layouts agree and overlaps nothing
 * else (RNN_E_INVALID). */
int rnn_norm_rotary_backward(rnn_ctx *ctx, const rnn_rotary_desc *d, uint32_t hq, float eps, size_t n,
                             size_t t, const float *x, const float *gain, const float *pos,
                             const float *dy, size_t dystride, size_t dyoff, void *ws, size_t ws_bytes,
                             float *dx, float *dgain);

/* Norm of each head times SiLU of a gate (no counterpart in the reference): rows
 * of h heads of d channels, x and y [rows][h][d], z at z + r*zstride + zoff.
 *   y = gain x / sqrt(mean(x^2) + eps) z / (1 + exp(-z))
 * gain [h][d] (NULL: 1); the mean is a head's.  d <= 512, h <= 65536, eps > 0.  y
 * may be x and overlaps nothing else (RNN_E_INVALID).  A NaN in x gives NaN in its
 * head, an infinity NaN in its channel and zeros in the others of its head; either
 * in z stays in its channel.  z / (1 + exp(-z)) is 0 below z = -120. */
int rnn_head_gate_forward(rnn_ctx *ctx, size_t rows, size_t h, size_t d, float eps, const float *x,
                          const float *z, size_t zstride, size_t zoff, const float *gain, float *y);
/* Bytes of device workspace that a backward with dgain needs, as
 * rnn_norm_rotary_workspace; host only. */
int rnn_head_gate_workspace(size_t rows, size_t h, size_t d, size_t *bytes);
/* Its backward: dx [rows][h][d] and dz (at dz + r*dzstride + dzoff) are
 * overwritten, dgain [h][d] (NULL: not wanted) accumulates in a fixed order.  dx
 * may be dy or x, dz may be z where their layouts agree; they overlap nothing else
 * (RNN_E_INVALID, as for dz and z given as one buffer of two layouts). */
int rnn_head_gate_backward(rnn_ctx *ctx, size_t rows, size_t h, size_t d, float eps, const float *x,
                           const float *z, size_t zstride, size_t zoff, const float *gain,
                           const float *dy, void *ws, size_t ws_bytes, float *dx, float *dz,
                           size_t dzstride, size_t dzoff, float *dgain);

/* ----------------------------------------------- linear attention with decay */
/* Linear attention with a decay for each head (no counterpart in the reference).
 * Head j reads queries of dk channels at q + r*qstride + qoff + j*dk; key head
 * g = j / (h / hkv) has keys at k + r*kstride + koff + g*dk and values of dv
 * channels at v + r*vstride + voff + g*dv; q, k and v may be one buffer.  With
 * gamma_j = exp(-exp(rate[j])), over the tokens i of a sequence in order,
 *   S_i = gamma S_(i-1) + k_i^T v_i,   y_i = scale q_i S_i
 * which is y_i = scale sum_(l <= i) gamma^(i-l) (q_i . k_l) v_l.  The last
 * `reverse` heads take the tokens from the last to the first.
 * Sequence b has min(lens[b], t) tokens (device array; NULL: t): rows behind them
 * are padding, which is never read and may hold anything; y is 0 there.
 * state_in [n][h][dk][dv] is S before the first token (NULL: 0), state_out S
 * after the last (NULL: not wanted; may be state_in): a sequence may be given in
 * pieces, or token by token.  gamma is within [0, 1] for any rate; -infinity: 1, no
 * decay.  Products, sums and states are fp32; powers of gamma are formed with their
 * exponent in 48 bits or more, so that long memories keep theirs.  A NaN or an
 * infinity shows, as NaN or infinity, in the tokens that see it and in no others. */
typedef struct {
    uint32_t h, hkv, dk, dv;
    size_t qstride, qoff, kstride, koff, vstride, voff;
    uint32_t reverse;
    float scale;
} rnn_decay_attn_desc;
/* Checks a description and gives the bytes of device workspace that the forward
 * (backward = 0) or the backward needs for n sequences of t tokens; host only.
 * The workspace is the caller's, 256-byte aligned, holds nothing between calls
 * and is not shared by calls that may run at the same time.  dk and dv <= 128, row
 * strides, y's among them, <= 2^22, t < 2^29, n * h < 2^22, n * h * t and
 * n * h * dk * dv < 2^31 (RNN_E_UNSUPPORTED above), scale finite. */
int rnn_decay_attn_workspace(const rnn_decay_attn_desc *d, size_t n, size_t t, int backward,
                             size_t *bytes);
/* y [n][t][h][dv] and state_out, which overlap no other operand (but state_out may
 * be state_in), else RNN_E_INVALID. */
int rnn_decay_attn_forward(rnn_ctx *ctx, const rnn_decay_attn_desc *d, size_t n, size_t t,
                           const float *q, const float *k, const float *v, const float *rate,
                           const uint32_t *lens, const float *state_in, void *ws, size_t ws_bytes,
                           float *y, float *state_out);
/* From the forward's inputs, dy [n][t][h][dv] and, where state_out was used, its
 * gradient dstate_out (NULL: 0): dq, dk and dv, laid out as q, k and v, ACCUMULATE or
 * are overwritten as flags say (RNN_ATTN_SET_DQ, RNN_ATTN_SET_DKV: the columns of the
 * heads, padding rows included, which receive 0); drate [h] (NULL: not wanted)
 * accumulates; dstate_in (NULL: not wanted) is overwritten.  dq, dk and dv may be one
 * buffer with disjoint columns; but for that, no gradient overlaps another one or
 * another operand, else RNN_E_INVALID.  Sums run in a fixed order. */
int rnn_decay_attn_backward(rnn_ctx *ctx, const rnn_decay_attn_desc *d, size_t n, size_t t,
                            const float *q, const float *k, const float *v, const float *rate,
                            const uint32_t *lens, const float *state_in, const float *dy,
                            const float *dstate_out, void *ws, size_t ws_bytes, float *dq, float *dk,
                            float *dv, float *drate, float *dstate_in, uint32_t flags);

/* -------------------------------------------------- differential attention */
/* Differential attention (no counterpart in the reference): the difference of
 * two softmax maps, with a norm over each head's output.  Head j has two query
 * maps of dh channels, at q + r*qstride + qoff + (2j + m)*dh (m = 0, 1); key
 * head g = j / (h / hkv) has two key maps, at kv + r*kvstride + koff +
 * (2g + m)*dh, and values of 2 dh channels at kv + r*kvstride + voff + 2g*dh.
 *   P_m = softmax(scale Q_m K_m^T) over the keys that the query sees
 *   lambda = exp(lq1 . lk1) - exp(lq2 . lk2) + lam_init
 *   O = (P_1 - lambda P_2) V
 *   y = (1 - lam_init) gain O / sqrt(mean(O^2) + eps)   (gain NULL: y = O)
 * lam [lam_heads][4][dh] holds lq1, lk1, lq2, lk2, one set for all heads
 * (lam_heads 1) or one for each (lam_heads h); gain [2 dh] serves every head.
 * Image b has min(qlen[b], tq) queries and min(klen[b], tk) keys (device
 * arrays; NULL: tq, tk): rows behind them are padding, which is never read and
 * may hold anything.  causal: query i sees keys j <= i + (keys - queries), the
 * two sequences aligned at their ends; mask_diag: not key j = i.  A query that
 * sees no key, and a padding query, give y = 0.  A NaN or an infinity gives NaN:
 * in a query to its row, in a key to every row that sees it, in a value to rows
 * that do not see it as well, in dy to its row of dq and to what sums over rows.
 * (An infinity also leaves its image's other keys steps of 2^-24, and NaN past
 * 2^15; its other values, in rows that are not NaN already, 2^-20 and 2^19.)
 * So do scores past a float's range.  The backward forms P again from scores that
 * are within 2^-22 of themselves: those above 2^15 leave it few bits.
 * Products are taken in two fp16 parts under a power of two (of a row, of
 * a tile, or in sums of all tiles so far; dS of its own row in dq, its own key in
 * dkv): elements down to 2^-12 of the largest keep 2^-23 of themselves, smaller
 * ones 2^-35 of the largest.  Sums are fp32: dq, a sum over the keys, is within
 * some 2^-24 sqrt(3 tk / 16) of its terms' size besides (3e-7 at 256 keys, 2e-6
 * measured at 65536). */
typedef struct {
    uint32_t h, hkv, dh, tq, tk;
    size_t qstride, qoff, kvstride, koff, voff;
    uint32_t lam_heads;
    int mask_diag, causal;
    float scale, lam_init, eps;
} rnn_diff_attn_desc;
/* Checks a description and gives the bytes of device workspace that the
 * forward (backward = 0) or the backward needs for n images; host only.  The
 * workspace is the caller's, 256-byte aligned, holds nothing between calls
 * and is not shared by calls that may run at the same time.  dh <= 64
 * and row strides <= 2^22, n * max(tq, tk) * h < 2^30 (RNN_E_UNSUPPORTED above),
 * scale > 0, 0 <= lam_init < 1. */
int rnn_diff_attn_workspace(const rnn_diff_attn_desc *d, size_t n, int backward, size_t *bytes);
/* y [n][tq][h][2 dh].  For a backward: o12 [n][tq][h][2][2 dh] receives each
 * map's P_m V and stats [n][tq][h][4] (16-byte aligned) each map's largest score
 * and the reciprocal of its softmax sum, as the backward takes them; both NULL:
 * not kept. */
int rnn_diff_attn_forward(rnn_ctx *ctx, const rnn_diff_attn_desc *d, size_t n, const float *q,
                          const float *kv, const float *lam, const float *gain,
                          const uint32_t *qlen, const uint32_t *klen, void *ws, size_t ws_bytes,
                          float *y, float *o12, float *stats);
/* From dy [n][tq][h][2 dh] and the forward's o12 and stats: dq and dkv, laid
 * out as q and kv, ACCUMULATE or are overwritten as flags say
 * (RNN_ATTN_SET_DQ, RNN_ATTN_SET_DKV: the columns of queries, or of keys and
 * values, padding rows included, which receive 0); dlam [lam_heads][4][dh] and
 * dgain [2 dh] (NULL with gain) accumulate.  dq and dkv may be one buffer with
 * disjoint columns, and overlap no other operand.  Sums run in a fixed order. */
int rnn_diff_attn_backward(rnn_ctx *ctx, const rnn_diff_attn_desc *d, size_t n, const float *q,
                           const float *kv, const float *lam, const float *gain,
                           const uint32_t *qlen, const uint32_t *klen, const float *o12,
                           const float *stats, const float *dy, void *ws, size_t ws_bytes,
                           float *dq, float *dkv, float *dlam, float *dgain, uint32_t flags);

/* ---------------------------------------------------------- linear.rs */
/* Linear::forward (linear.rs:44-63): y[rows x fout] = x W^T + b (b may be NULL). */
int rnn_linear_forward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *x,
                       const float *w, const float *b, float *y);
/* Linear::forward feeding a residual branch (vit.rs:155-176): y = x W^T + b
 * as rnn_linear_forward, and out += (y l) m with m = mask[r / rpi] (mask may
 * be NULL: m = 1) -- rnn_residual_add_scaled(out, y, ...) -- in the GEMM's
 * epilogue (two passes when rpi is not a power of two).  out is neither x
 * nor y. */
int rnn_linear_forward_residual(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout,
                                const float *x, const float *w, const float *b, float *y,
                                const float *l, const float *mask, size_t rpi, float *out);
/* Linear::backward (linear.rs:66-96): dw += dy^T x; db += colsum(dy) (db may
 * be NULL); dx = dy W (overwritten). */
int rnn_linear_backward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *dy,
                        const float *x, const float *w, float *dw, float *db, float *dx);
/* rnn_linear_backward with dx accumulated instead of overwritten when flags
 * has RNN_LINEAR_ACC_DX: dx += dy W, the old value first, as add_ (nn.rs:441-443)
 * of a separately computed dx.  Block::backward (vit.rs:175-232) sums its
 * branches' input gradients this way without a separate pass. */
#define RNN_LINEAR_ACC_DX 1u
int rnn_linear_backward_ex(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *dy,
                           const float *x, const float *w, float *dw, float *db, float *dx,
                           uint32_t flags);

/* The Linear product with an activation and a residual (no counterpart in the
 * reference, whose MLP is SwiGLU): z = x W^T + b, y = act(z) + res (b, res may
 * be NULL; res [rows x fout], may be y).  slope [rows x fout] receives act'(z)
 * for the backward (NULL: not kept; not needed for RNN_ACT_NONE).  act:
 * RNN_ACT_NONE z, RNN_ACT_RELU max(z, 0), RNN_ACT_GELU z (1 + erf(z / sqrt 2)) /
 * 2, RNN_ACT_GELU_TANH z (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2,
 * RNN_ACT_SILU z / (1 + exp(-z)); RELU's slope at 0 is 0.  rows <= 2^30 - 128, fin
 * and fout <= 2^20.  Products are taken in two fp16 parts under a power of two of
 * what one sum takes (a row of x, W or dz, a column of W, dz or x): elements down
 * to 2^-12 of its largest so far keep 2^-23 of themselves, smaller ones 2^-35 of the
 * largest.  An infinity or a NaN in x, W or dy gives NaN in the sums that take it. */
#define RNN_ACT_NONE 0u
#define RNN_ACT_RELU 1u
#define RNN_ACT_GELU 2u
#define RNN_ACT_GELU_TANH 3u
#define RNN_ACT_SILU 4u
int rnn_linear_act_forward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *x,
                           const float *w, const float *b, uint32_t act, const float *res,
                           float *slope, float *y);
/* Bytes of device workspace that the backward needs; host only.  The workspace
 * is the caller's, 256-byte aligned, holds nothing between calls and is not
 * shared by calls that may run at the same time. */
int rnn_linear_act_workspace(size_t rows, size_t fin, size_t fout, size_t *bytes);
/* Its backward, from the forward's slope (NULL: RNN_ACT_NONE): dz = dy slope,
 * dx = dz W (added with RNN_LINEAR_ACC_DX), dw += dz^T x, db += colsum(dz) (db may
 * be NULL, and is with fin = 0).  The residual's gradient is dy itself.  Sums run
 * in a fixed order. */
int rnn_linear_act_backward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *dy,
                            const float *x, const float *w, const float *slope, void *ws,
                            size_t ws_bytes, float *dw, float *db, float *dx, uint32_t flags);

/* ------------------------------------------ host-slice forms (Rust shim) */
/* The same entry points over HOST memory, for the Rust shim, whose callers
 * keep the reference's Vec<f32> tensors (nn.rs Tensor, linear.rs, attn.rs
 * Tok): each call copies its operands into a device staging block the
 * context keeps (it only grows), runs the device entry point on the context
 * stream, runs any deferred reductions, copies the outputs back and returns
 * after the stream has finished.  Arguments, accumulation and the k = 0 /
 * empty cases are those of the device form; a host pointer passed for two
 * operands (a fused QKV buffer as q and kv; dq == dkv as SelfAttn::backward
 * passes them, attn.rs:418-438) is staged once.  Each replaces the same
 * reference function as its device form:
 *   rnn_matmul_host              matmul        (gemm.rs:434-493)
 *   rnn_gemm_small_batched_host  gemm_small    (gemm.rs:500-545), C read back whole
 *   rnn_matmul_dw_host           matmul_dw     (gemm.rs:555-598)
 *   rnn_conv2d_forward_host      Conv2d::forward    (nn.rs:166-185)
 *   rnn_conv2d_backward_w_host   Conv2d::backward_w (nn.rs:193-227)
 *   rnn_conv2d_backward_x_host   dX of Conv2d::backward (nn.rs:230-250)
 *   rnn_attn_forward_host        Core::forward (attn.rs:148-223)
 *   rnn_attn_backward_host       Core::backward (attn.rs:226-343)
 *   rnn_linear_forward_host      Linear::forward (linear.rs:44-64)
 *   rnn_linear_backward_host     Linear::backward (linear.rs:66-96) */
int rnn_matmul_host(rnn_ctx *ctx, size_t m, size_t n, size_t k, const float *a, int at,
                    const float *b, int bt, float *c, int acc);
int rnn_gemm_small_batched_host(rnn_ctx *ctx, size_t count, size_t m, size_t n, size_t k,
                                const float *a, size_t stride_a, int at, const float *b,
                                size_t stride_b, int bt, float *c, size_t stride_c, int acc);
int rnn_matmul_dw_host(rnn_ctx *ctx, size_t m, size_t n, size_t k, const float *a,
                       const float *b, float *c);
int rnn_conv2d_forward_host(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n, const float *x,
                            const float *w, float *y);
int rnn_conv2d_backward_w_host(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n,
                               const float *dy, const float *x, float *dw);
int rnn_conv2d_backward_x_host(rnn_ctx *ctx, const rnn_conv_spec *sp, size_t n,
                               const float *dy, const float *w, float *dx);
int rnn_attn_forward_host(rnn_ctx *ctx, const rnn_attn_desc *d, size_t n, const float *q,
                          const float *kv, const float *tau, const float *rel, float *p,
                          float *o);
int rnn_attn_backward_host(rnn_ctx *ctx, const rnn_attn_desc *d, size_t n, const float *q,
                           const float *kv, const float *tau, const float *p, const float *dout,
                           float *dq, float *dkv, float *dtau, float *drel);
int rnn_linear_forward_host(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *x,
                            const float *w, const float *b, float *y);
int rnn_linear_backward_host(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout,
                             const float *dy, const float *x, const float *w, float *dw,
                             float *db, float *dx);

/* -------------------------------------------------------------- nn.rs */
/* The ResNet layers around the convs.  Elementwise formulas round exactly as
 * the reference's (no FMA contraction); per-channel sums are f64 in a fixed
 * order.  x, y, dy, dx are NCHW [n][c][hw]; per-channel arrays hold c floats. */

/* BatchNorm2d::forward / forward_relu in train mode (nn.rs:253-348): batch
 * statistics (f64 sums), y = [relu](gamma*(x - mean)*invstd + beta), running
 * mean / unbiased running variance updated with `momentum` (0.1 in rustnn).
 * mean and invstd are written for rnn_bn_backward.  y may alias x; the
 * reference keeps xhat for the backward, this API keeps x instead (a caller
 * that normalises in place must keep a copy of x).  running_mean and
 * running_var may both be NULL (statistics only, no running update). */
int rnn_bn_forward_train(rnn_ctx *ctx, size_t n, size_t c, size_t hw, const float *x, float *y,
                         const float *gamma, const float *beta, float *running_mean,
                         float *running_var, float *mean, float *invstd, float momentum, float eps,
                         int relu);
/* BatchNorm2d forward in eval mode (run_eval, nn.rs:350-365). */
int rnn_bn_forward_eval(rnn_ctx *ctx, size_t n, size_t c, size_t hw, const float *x, float *y,
                        const float *gamma, const float *beta, const float *running_mean,
                        const float *running_var, float eps, int relu);
/* BatchNorm2d::backward (nn.rs:379-425): dx overwritten, dgamma / dbeta
 * ACCUMULATE.  x, mean, invstd as passed to / written by the train forward.
 * relu_out (may be NULL): apply relu_back_ (nn.rs:432-439) to dy first, i.e.
 * use 0 where relu_out <= 0 (dy itself is not modified). */
int rnn_bn_backward(rnn_ctx *ctx, size_t n, size_t c, size_t hw, const float *dy,
                    const float *relu_out, const float *x, const float *mean, const float *invstd,
                    const float *gamma, float *dx, float *dgamma, float *dbeta);
/* relu_back_ (nn.rs:432-439): d = 0 where y <= 0. */
int rnn_relu_back(rnn_ctx *ctx, size_t len, float *d, const float *y);
/* add_ (nn.rs:441-443): a += b. */
int rnn_add(rnn_ctx *ctx, size_t len, float *a, const float *b);
/* add_ after relu_back_ (nn.rs:432-443) without changing b: a += b where
 * y > 0 (the value relu_back_(b, y) then add_(a, b) leave in a); a must
 * not be b. */
int rnn_add_relu_back(rnn_ctx *ctx, size_t len, float *a, const float *b, const float *y);
/* add_relu_ (nn.rs:446-450): a = max(a + b, 0). */
int rnn_add_relu(rnn_ctx *ctx, size_t len, float *a, const float *b);
/* gap_forward (nn.rs:455-463): y[n][c] = plane sum (pixel order) / hw. */
int rnn_gap_forward(rnn_ctx *ctx, size_t n, size_t c, size_t hw, const float *x, float *y);
/* gap_backward (nn.rs:465-473): dx[n][c][p] = dy[n][c] / hw. */
int rnn_gap_backward(rnn_ctx *ctx, size_t n, size_t c, size_t hw, const float *dy, float *dx);
/* nn.rs Linear (the ResNet classifier, nn.rs:475-564), bit-identical to the
 * reference's scalar loops.  forward: y[i][o] = b[o] + sum_j w[o][j] x[i][j].
 * backward: dw, db ACCUMULATE over rows in order; dx (may be NULL) is
 * overwritten. */
int rnn_fc_forward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *x,
                   const float *w, const float *b, float *y);
int rnn_fc_backward(rnn_ctx *ctx, size_t rows, size_t fin, size_t fout, const float *dy,
                    const float *x, const float *w, float *dw, float *db, float *dx);
/* softmax_ce (nn.rs:566-637): dlogits = (softmax - smoothed target) / rows;
 * *loss (device, may be NULL) = mean loss; *correct (device u32, may be NULL)
 * = rows whose first maximal logit is the label.  labels: device u32[rows].
 * rows <= 8192, nclass <= 1024.  A label >= nclass (a panic in the reference)
 * gives NaN for that row instead of an out-of-bounds read. */
int rnn_softmax_ce(rnn_ctx *ctx, size_t rows, size_t nclass, const float *logits,
                   const uint32_t *labels, float smooth, float *dlogits, float *loss,
                   uint32_t *correct);
/* Param::step (nn.rs:102-110): Nesterov SGD, g zeroed.  Pass wd = 0 for the
 * parameters the reference does not decay (BN gamma / beta, biases). */
int rnn_sgd_step(rnn_ctx *ctx, size_t len, float *v, float *g, float *m, float lr, float momentum,
                 float wd);

/* ----------------------------------------------------------- norm.rs */
/* Token tensors are [rows = n*t][c] row-major, channel fastest (tok.rs).
 * Parameter gradients (dg, db, dl, dw, dp) accumulate (+=), as Param::g does;
 * dx is overwritten. */
/* LayerNorm::forward (norm.rs:38-85): per row f64 sums, mu, var = max(s2/c -
 * mu^2, 0) as f32, invstd = 1/sqrt(var + eps); y = g (x - mu) invstd + b.
 * Training keeps xhat [rows][c] and invstd [rows]; pass both NULL for eval. */
int rnn_ln_forward(rnn_ctx *ctx, size_t rows, size_t c, const float *x, const float *g,
                   const float *b, float eps, float *y, float *xhat, float *invstd);
/* LayerNorm::backward (norm.rs:87-137). */
int rnn_ln_backward(rnn_ctx *ctx, size_t rows, size_t c, const float *dy, const float *xhat,
                    const float *invstd, const float *g, float *dx, float *dg, float *db);
/* rnn_ln_backward followed by add_ (Block::backward, vit.rs:175-232: the
 * norm's input gradient plus the residual's, dy = n2.backward(dh2) + dz and
 * dy += n1.backward(dh)): dx = the LayerNorm input gradient + add, in the
 * same pass for c <= 512.  add may be dx (in place). */
int rnn_ln_backward_add(rnn_ctx *ctx, size_t rows, size_t c, const float *dy, const float *xhat,
                        const float *invstd, const float *g, const float *add, float *dx,
                        float *dg, float *db);
/* rnn_ln_backward_add, then the DropPath + LayerScale backward that reads
 * its dx (the next block's first op in a backward over Blocks, vit.rs:175-
 * 232): lsdx = (dx m) l and dl += sum (dx m) lsx, m = mask[r / rpi] or 1
 * when NULL -- the values rnn_ln_backward_add then
 * rnn_drop_layerscale_backward(dx, lsx, l, mask, rpi, lsdx, dl) give, bit
 * for bit, in the same pass for c <= 512.  lsdx must not overlap dy, add,
 * dx or lsx. */
int rnn_ln_backward_add_ls(rnn_ctx *ctx, size_t rows, size_t c, const float *dy,
                           const float *xhat, const float *invstd, const float *g,
                           const float *add, float *dx, float *dg, float *db, const float *lsx,
                           const float *l, const float *mask, size_t rpi, float *lsdx,
                           float *dl);
/* LayerScale::forward / backward (norm.rs:166-212): y = x l per channel (y may
 * be x); dl += sum dy x, dx = dy l (dx may be dy). */
int rnn_layerscale_forward(rnn_ctx *ctx, size_t rows, size_t c, const float *x, const float *l,
                           float *y);
int rnn_layerscale_backward(rnn_ctx *ctx, size_t rows, size_t c, const float *dy, const float *x,
                            const float *l, float *dx, float *dl);
/* DropPath::backward then LayerScale::backward (vit.rs:61-73,
 * norm.rs:182-212) in one pass that reads dy without changing it:
 * g = dy * mask[r / rpi] (mask NULL: g = dy), dl += sum_r g x, dx = g l
 * (dx must not be dy).  Block::backward's branches (vit.rs:175-232) read the
 * same dy twice or three times, so no copy of it is needed. */
int rnn_drop_layerscale_backward(rnn_ctx *ctx, size_t rows, size_t c, const float *dy,
                                 const float *x, const float *l, const float *mask, size_t rpi,
                                 float *dx, float *dl);
/* The first residual's branch gradients in a Block backward (vit.rs:175-232)
 * in one pass over dy: da = (dy m1) l1 with dl1 += sum (dy m1) a (the
 * DropPath + LayerScale of the attention branch), ddw = da gamma with
 * dgamma += sum da dwo (the depthwise branch's gamma gate) and, for a reader
 * block (cm set), dc = (dy m2) lm with dlm += sum (dy m2) cm.  Each value
 * equals what rnn_drop_layerscale_backward (lsm, then ls1) and
 * rnn_layerscale_backward (gamma) called in turn write; m1 / m2 = mask[r /
 * rpi] or 1 when NULL.  dy, a, dwo and cm are not changed; the outputs must
 * not overlap them or each other. */
int rnn_block_branch_backward(rnn_ctx *ctx, size_t rows, size_t c, const float *dy,
                              const float *a, const float *l1, const float *m1, const float *dwo,
                              const float *gamma, const float *cm, const float *lm,
                              const float *m2, size_t rpi, float *da, float *dl1, float *ddw,
                              float *dgamma, float *dc, float *dlm);
/* y = x + (a l) m, m = mask[r / rpi] per image (mask may be NULL: m = 1): one
 * residual branch of Block::forward, x + DropPath(LayerScale(a))
 * (vit.rs:155-176: the LayerScale, the DropPath scaling and add_ in that
 * rounding order) in one pass.  y may be x (in place); a is left unchanged,
 * as the LayerScale backward (rnn_drop_layerscale_backward) reads it. */
int rnn_residual_add_scaled(rnn_ctx *ctx, size_t rows, size_t c, const float *x, const float *a,
                            const float *l, const float *mask, size_t rpi, float *y);
/* The SwiGLU gate between SwiGlu's two Linear calls (norm.rs:250-288): ab is
 * [rows][2h] (a | b), u = a sigmoid(a) b [rows][h]; the backward writes
 * dab [rows][2h] from du [rows][h]. */
int rnn_swiglu_forward(rnn_ctx *ctx, size_t rows, size_t h, const float *ab, float *u);
int rnn_swiglu_backward(rnn_ctx *ctx, size_t rows, size_t h, const float *du, const float *ab,
                        float *dab);
/* DwConv3 (norm.rs:296-457): depthwise 3x3, pad 1, over n images of th x tw
 * tokens, channel-last; w [9][c] (tap-major), b [c]. */
int rnn_dwconv3_forward(rnn_ctx *ctx, size_t n, size_t th, size_t tw, size_t c, const float *x,
                        const float *w, const float *b, float *y);
int rnn_dwconv3_backward(rnn_ctx *ctx, size_t n, size_t th, size_t tw, size_t c, const float *dy,
                         const float *x, const float *w, float *dx, float *dw, float *db);
/* rnn_dwconv3_backward with dx accumulated (dx += the input gradient, the old
 * value first) when flags has RNN_DW3_ACC_DX; dx must not be dy. */
#define RNN_DW3_ACC_DX 1u
int rnn_dwconv3_backward_ex(rnn_ctx *ctx, size_t n, size_t th, size_t tw, size_t c,
                            const float *dy, const float *x, const float *w, float *dx, float *dw,
                            float *db, uint32_t flags);
/* Block::forward's first branch (vit.rs:150-160) in one pass: d =
 * DwConv3(h) as rnn_dwconv3_forward computes it; a += gamma d (rnn_axpy_cols);
 * y = x + (a l) m, m = mask[image] (mask may be NULL; rnn_residual_add_scaled
 * with th * tw rows per image).  h, a, x, y, d are [n][th][tw][c]; gamma, l
 * [c]; a is updated in place and y may be x; d, a, h and y are distinct, and x
 * is not a. */
int rnn_dwconv3_branch_forward(rnn_ctx *ctx, size_t n, size_t th, size_t tw, size_t c,
                               const float *h, const float *w, const float *b, float *d, float *a,
                               const float *gamma, const float *x, const float *l,
                               const float *mask, float *y);
/* SeqPool (norm.rs:459-586): w = softmax_t(x p), z = sum_t w_t x_t; z [n][c];
 * the forward writes the softmax weights w [n][t] that the backward reads.
 * t <= 1024. */
int rnn_seqpool_forward(rnn_ctx *ctx, size_t n, size_t t, size_t c, const float *x,
                        const float *p, float *z, float *w);
int rnn_seqpool_backward(rnn_ctx *ctx, size_t n, size_t t, size_t c, const float *dz,
                         const float *w, const float *x, const float *p, float *dx, float *dp);

/* ----------------------------------------------------------- loss.rs */
/* Soft targets of a batch (targets, train.rs:121-155): tf [n][nf] = lam a +
 * (1 - lam) b with a / b the targets of labels[i] / labels[perm[i]] --
 * taxo_target (loss.rs:11-28, sibling share sib of eps, parent [nf] the
 * superclass of each fine class) when taxo, else uniform_target
 * (loss.rs:30-34); tc [n][nc] (may be NULL) the same over coarse labels with
 * uniform smoothing.  perm NULL = identity, lam NULL = all 1. */
int rnn_soft_targets(rnn_ctx *ctx, size_t n, size_t nf, size_t nc, const uint32_t *labels,
                     const uint32_t *coarse, const uint32_t *perm, const float *lam,
                     const uint32_t *parent, int taxo, float eps, float sib, float *tf,
                     float *tc);
/* The dominant label of each mixed image (Trainer::make_batch,
 * train.rs:313-320): dom[i] = labels[i] when lam[i] >= 0.5, else
 * labels[perm[i]] -- the hard label ce_soft counts hits against. */
int rnn_mix_dominant(rnn_ctx *ctx, size_t n, const uint32_t *labels, const uint32_t *perm,
                     const float *lam, uint32_t *dom);
/* ce_soft (loss.rs:39-83): dz [n][nclass] overwritten with scale (softmax -
 * target) / n; *loss (device, may be NULL) the mean loss; *correct (device,
 * may be NULL) the argmax hits against hard. */
int rnn_ce_soft(rnn_ctx *ctx, size_t n, size_t nclass, const float *logits, const float *target,
                const uint32_t *hard, float scale, float *dz, float *loss, uint32_t *correct);
/* kl_distill (loss.rs:87-130): teacher detached; dz += temp (ps - pt) / n *
 * scale; *loss = mean of temp^2 KL(pt || ps). */
int rnn_kl_distill(rnn_ctx *ctx, size_t n, size_t nclass, const float *student,
                   const float *teacher, float temp, float scale, float *dz, float *loss);
/* hint_mse (loss.rs:133-151): dz += 2 (pred - target) / (n c) * scale; *loss =
 * scale * mean squared error. */
int rnn_hint_mse(rnn_ctx *ctx, size_t n, size_t c, const float *pred, const float *target,
                 float scale, float *dz, float *loss);
/* build_loss (train.rs:70-118) in one call: the soft-target cross-entropy of
 * the logits (scale 1), of the coarse head when coarse_w > 0 and taxo (scale
 * coarse_w), and with the exits (io->e1 set): the exits' cross-entropies
 * (exit_w1, exit_w2), their distillation from the logits when alpha > 0
 * (loss::kl_distill, temp) and the hint MSEs of h1 / h2 against feat when
 * beta > 0.  Gradients are written (the reference's zeroed Grads receive
 * them): dlogits, dcoarse (zeros without the coarse term), de1 / de2 (their
 * cross-entropy, then the distillation added), dh1 / dh2 (zeros when beta
 * is 0).  *total = ce (+ coarse_w lc) (+ (w1 l1 + w2 l2)) (+ alpha (k1 + k2))
 * (+ (h1 + h2)) in f32, the reference's order and grouping; *ce the logits'
 * loss; *correct its argmax hits (device pointers, any may be NULL).  nc:
 * coarse classes (0: no coarse head); d4: the width of h1 / h2 / feat. */
typedef struct {
    float coarse_w, exit_w1, exit_w2, alpha, temp, beta;
    int taxo;
} rnn_loss_cfg;
typedef struct {
    const float *logits, *coarse, *e1, *e2, *h1, *h2, *feat;
    float *dlogits, *dcoarse, *de1, *de2, *dh1, *dh2;
} rnn_loss_io;
int rnn_build_loss(rnn_ctx *ctx, size_t n, size_t nf, size_t nc, size_t d4, const float *tf,
                   const float *tc, const uint32_t *hard, const uint32_t *hardc,
                   const rnn_loss_cfg *cfg, const rnn_loss_io *io, float *total, float *ce,
                   uint32_t *correct);

/* ----------------------------------------------------------- vit.rs */
/* DropPath (vit.rs:25-74) on n images of `per` floats, in place: image i is
 * kept with the i-th uniform of Rng::new(seed) (rng.rs) below 1 - p and
 * scaled by 1 / (1 - p), else zeroed; mask [n] (device) receives the factors
 * for the backward.  0 < p < 1 (the reference skips the layer otherwise). */
int rnn_drop_path_forward(rnn_ctx *ctx, size_t n, size_t per, float *x, float p, uint64_t seed,
                          float *mask);
int rnn_drop_path_backward(rnn_ctx *ctx, size_t n, size_t per, float *dy, const float *mask);
/* The masks alone of `count` DropPath layers over n images, in one launch:
 * masks[k] (device, [n]) receives rnn_drop_path_forward's factors for p[k]
 * and seeds[k] (p, seeds and masks are host arrays).  A layer whose mask is
 * drawn here is applied with rnn_drop_path_backward (the same per-image
 * scaling).  Batches DropPath::forward's draws (vit.rs:44-51) of a step. */
int rnn_drop_path_masks(rnn_ctx *ctx, size_t count, size_t n, const float *p,
                        const uint64_t *seeds, float *const *masks);
/* y[r][j] += l[j] x[r][j]: Block's depthwise gate a += gamma * dw(h)
 * (vit.rs:150-158).  Its backward is rnn_layerscale_backward. */
int rnn_axpy_cols(rnn_ctx *ctx, size_t rows, size_t c, float *y, const float *l, const float *x);
/* token_merge / token_merge_back (vit.rs:612-650): [n][th*th][c] <->
 * [n][(th/2)^2][4c], the 2x2 neighbours (0,0), (0,1), (1,0), (1,1)
 * concatenated; th even; the backward overwrites dz. */
int rnn_token_merge(rnn_ctx *ctx, size_t n, size_t th, size_t c, const float *z, float *y);
int rnn_token_merge_backward(rnn_ctx *ctx, size_t n, size_t th, size_t c, const float *dy,
                             float *dz);
/* TaxoHead (vit.rs:282-312): zf[i][j] += zc[i][parent[j]]; the backward's
 * coarse gradient dc = dzc + the fine gradients summed by parent (in class
 * order).  parent (device u32 [nf]). */
int rnn_taxo_head_combine(rnn_ctx *ctx, size_t n, size_t nf, size_t nc, const uint32_t *parent,
                          float *zf, const float *zc);
int rnn_taxo_head_combine_backward(rnn_ctx *ctx, size_t n, size_t nf, size_t nc,
                                   const uint32_t *parent, const float *dzf, const float *dzc,
                                   float *dc);
/* Tok::from_tensor / to_tensor (tok.rs): [n][c][hw] <-> [n][hw][c]. */
int rnn_nchw_to_tokens(rnn_ctx *ctx, size_t n, size_t c, size_t hw, const float *x, float *t);
int rnn_tokens_to_nchw(rnn_ctx *ctx, size_t n, size_t c, size_t hw, const float *t, float *x);

/* ----------------------------------------------------------- data.rs */
/* make_batch_train (data.rs:384-416): for batch slot b, image idx[b] of the
 * device-resident dataset (images [nimg][3][32][32] u8, fine / coarse labels
 * u8), with Rng::new(seed ^ b * 0x9E3779B97F4A7C15): ra_n RandAugment
 * operations of magnitude ra_mag (none when ra_mag <= 0; ra_n <= 16), crop
 * offsets in [-pad, pad], a horizontal flip,
 * normalisation (border = -mean/std), random erasing with probability erase
 * of an erase_side square of N(0,1) noise.  out [bs][3][32][32]; labels,
 * coarse_out [bs] u32.  An index past nimg gives a NaN image and label
 * 0xffffffff. */
int rnn_cifar_batch_train(rnn_ctx *ctx, const uint8_t *images, const uint8_t *fine,
                          const uint8_t *coarse, size_t nimg, const uint32_t *idx, size_t bs,
                          size_t pad, float ra_mag, size_t ra_n, float erase, size_t erase_side,
                          uint64_t seed, float *out, uint32_t *labels, uint32_t *coarse_out);
/* make_batch_eval (data.rs:494-512): images start .. start + bs normalised
 * (mirrored when flip); labels may be NULL. */
int rnn_cifar_batch_eval(rnn_ctx *ctx, const uint8_t *images, const uint8_t *fine, size_t nimg,
                         size_t start, size_t bs, int flip, float *out, uint32_t *labels);
/* FNV-1a 64 continued over host bytes, or over host floats' bit patterns as
 * 4 little-endian bytes each (fnv_f32, train.rs:478-484): the building blocks
 * of Trainer::fingerprint (train.rs:450-470).  Host only. */
uint64_t rnn_fnv1a_bytes(uint64_t hash, const uint8_t *bytes, size_t n);
uint64_t rnn_fnv1a_f32(uint64_t hash, const float *values, size_t n);
/* The host generator of the trainer (rng.rs): state = Rng::new(seed); next. */
int rnn_rng_seed(uint64_t seed, uint64_t *state);
uint64_t rnn_rng_next_u64(uint64_t *state);
/* Normal draws from the caller's generator state (4 u64, advanced), host
 * only: rand_vec (rng.rs:70-72) times scale -- Param::kaiming (nn.rs:95-100)
 * with scale = sqrt(2 / fan_in) as f32 -- and Param::trunc_normal
 * (nn.rs:77-89): up to 8 redraws while |z| > 2, clamped to [-2, 2], times
 * std.  The initial weights of the reference's models, bit for bit. */
int rnn_rng_normal_vec(uint64_t *state, size_t n, float scale, float *out);
int rnn_rng_trunc_normal(uint64_t *state, size_t n, float std_, float *out);
/* mix_batch's draws (data.rs:469-492) from the caller's generator state (4
 * u64, advanced): perm [bs] (shuffle), lam [bs], *cut (cutmix or mixup), *l
 * and, for cutmix, rect = y0, y1, x0, x1.  Host only. */
int rnn_mix_plan(uint64_t *rng_state, size_t bs, float alpha_mix, float alpha_cut, float sw,
                 uint32_t *perm, float *lam, int *cut, float *l, int *rect);
/* The blend of that plan on the device (cutmix / mixup, data.rs:434-467):
 * out [bs][3][32][32] from x (not aliased), perm on the device, rect on the
 * host. */
int rnn_mix_apply(rnn_ctx *ctx, const float *x, float *out, size_t bs, const uint32_t *perm,
                  int cut, float l, const int *rect);

/* ----------------------------------------------------------- optim.rs */
/* Newton-Schulz orthogonalisation (newton_schulz, optim.rs:124-145), in
 * place on `count` [rows x cols] matrices at g + i*stride: X = G (G^T when
 * rows > cols) / (||G||_F + 1e-7), then `steps` quintic steps
 * X = a X + (b A + c A A) X with A = X X^T (a, b, c = 3.4445, -4.7750,
 * 2.0315), each product a batched GEMM over the matrices. */
int rnn_newton_schulz(rnn_ctx *ctx, size_t count, size_t rows, size_t cols, size_t steps,
                      float *g, size_t stride);

/* One parameter of Optim::step_all (nn.rs Param, nn.rs:43-53): device
 * buffers; v2 (AdamW's second moment, zero-initialised) may be NULL for a
 * Muon matrix; rows = 0 marks a tensor that is not a matrix. */
typedef struct {
    float *v, *g, *m, *v2;
    size_t len, rows, cols;
    int decay;
} rnn_param;

/* Optim (optim.rs:147-235).  rnn_optim_create = Optim::new(muon, ns_steps)
 * with mom 0.95, b1 0.9, b2 0.999, eps 1e-8, t 0 (rnn_optim_set changes
 * them).  rnn_optim_step = Optim::step_all(params, lr, wd): matrices with
 * both sides > 1 take the Muon step when muon is set (Nesterov momentum,
 * Newton-Schulz, v -= lr (0.2 sqrt(max(rows, cols)) g + wd v)), the rest
 * AdamW with bias corrections at t + 1; every g is zeroed; t += 1.  Same-shape
 * matrices run Newton-Schulz together. */
typedef struct rnn_optim rnn_optim;
int rnn_optim_create(rnn_ctx *ctx, int muon, size_t ns_steps, rnn_optim **out);
int rnn_optim_destroy(rnn_optim *opt);
int rnn_optim_set(rnn_optim *opt, float mom, float b1, float b2, float eps, size_t t);
size_t rnn_optim_t(const rnn_optim *opt);
int rnn_optim_step(rnn_optim *opt, size_t nparam, const rnn_param *params, float lr, float wd);
/* clip_ (optim.rs:237-251) on a flat gradient: the f64 sum of squares in a
 * fixed order; norm = sqrt as f32; above `max` every element is scaled by
 * max / norm.  *norm (device, may be NULL) receives the norm. */
int rnn_clip_grad_norm(rnn_ctx *ctx, size_t len, float *g, float max, float *norm);
/* clip_ (optim.rs:237-251) over the gradients of a parameter list, as the
 * reference calls it (train.rs:372-375): one f64 sum of squares over every
 * gradient, norm = sqrt as f32 into *norm (device, may be NULL); above `max`
 * every gradient is scaled by max / norm.  The list's pointer table is kept on
 * the device and uploaded again only when the list changes. */
int rnn_clip_params(rnn_ctx *ctx, size_t nparam, const rnn_param *params, float max,
                    float *norm);
/* Ema::update (optim.rs:283-287): w = d w + (1 - d) v, with d computed by
 * the caller as min(decay, (1 + t) / (10 + t)). */
int rnn_ema_update(rnn_ctx *ctx, size_t len, float *w, const float *v, float d);
/* Ema::update over a whole parameter list (train.rs:377-379): w[i] = d w[i] +
 * (1 - d) params[i].v, one launch for the list (pointer table cached as in
 * rnn_clip_params). */
int rnn_ema_update_params(rnn_ctx *ctx, size_t nparam, float *const *w, const rnn_param *params,
                          float d);
/* f32::powi as the reference's bias corrections compute it. */
float rnn_powi_f32(float a, int b);
/* lr_at (train.rs:21-28), host only: linear warm-up over `warm` steps, then a
 * cosine from peak down to lo at step `total`, in f32. */
float rnn_lr_at(float peak, float lo, size_t step, size_t total, size_t warm);

/* ----------------------------------------------------------- model.rs */
/* Device-resident CIFAR ResNet (ResNet::new, model.rs:113-135): depth_n
 * blocks per stage (6n+2 layers), widths width/2w/4w, nclass outputs, Kaiming
 * initialisation from rng.rs seeded with `seed` (bit-identical to the
 * reference's).  Parameters, gradients, momenta, running statistics and the
 * activations of the last train forward live on the device. */
typedef struct rnn_resnet rnn_resnet;
int rnn_resnet_create(rnn_ctx *ctx, size_t depth_n, size_t width, size_t nclass, uint64_t seed,
                      rnn_resnet **out);
int rnn_resnet_destroy(rnn_resnet *net);
/* Total floats of all parameters / BN running buffers; number of parameter
 * tensors and the length (and weight-decay flag) of tensor i, in the
 * reference's for_each_param order (model.rs:164-175). */
size_t rnn_resnet_num_params(const rnn_resnet *net);
size_t rnn_resnet_num_buffers(const rnn_resnet *net);
size_t rnn_resnet_num_tensors(const rnn_resnet *net);
int rnn_resnet_tensor_len(const rnn_resnet *net, size_t i, size_t *len, int *decay);
/* Device copies of the state in for_each_param order (which 0 = values,
 * 1 = gradients, 2 = momenta) or for_each_buffer order (which 3 = BN running
 * mean / var): exactly one of dst (read out) and src (write in) is set. */
int rnn_resnet_copy(rnn_resnet *net, int which, float *dst, const float *src);
/* ResNet::forward (model.rs:138-150): x [n][3][h][w] -> logits [n][nclass].
 * train = 1 uses batch statistics, updates the running ones and keeps the
 * activations for rnn_resnet_backward. */
int rnn_resnet_forward(rnn_resnet *net, size_t n, size_t h, size_t w, const float *x, int train,
                       float *logits);
/* ResNet::backward (model.rs:152-162): gradients ACCUMULATE into the
 * parameters' g after the last train forward. */
int rnn_resnet_backward(rnn_resnet *net, const float *dlogits);
/* ResNet::step (model.rs:205-207): Param::step on every parameter. */
int rnn_resnet_step(rnn_resnet *net, float lr, float momentum, float wd);
/* One train step (train.rs:686-699): forward(train), softmax_ce with label
 * smoothing, backward, step.  labels: device u32[n].  loss / correct (device,
 * may be NULL) receive the mean loss and the hit count.  Replayed from a
 * hipGraph from the second call on for a given (n, h, w).  x and labels both
 * NULL: the batch is the one already in the network's input slots
 * (rnn_resnet_inputs), nothing is copied. */
int rnn_resnet_train_step(rnn_resnet *net, size_t n, size_t h, size_t w, const float *x,
                          const uint32_t *labels, float smooth, float lr, float momentum, float wd,
                          float *loss, uint32_t *correct);
/* The network's own input slots for batches of n x 3 x h x w (planning that
 * shape): device x[n][3][h][w] and labels u32[n] that a loader may fill in
 * place before rnn_resnet_train_step(x = labels = NULL) -- the batch
 * assembly of train.rs:670-684 writing straight to where the step reads.
 * Valid until the shape changes or the network is destroyed. */
int rnn_resnet_inputs(rnn_resnet *net, size_t n, size_t h, size_t w, float **x,
                      uint32_t **labels);
/* Logits of the last forward (device [n][nclass]). */
int rnn_resnet_logits(rnn_resnet *net, float *logits);
/* Train-step graph: enable / disable (drops a recorded graph); state 1 when a
 * graph is recorded, 0 otherwise, with *why the reason recording failed. */
int rnn_resnet_set_graph(rnn_resnet *net, int on);
int rnn_resnet_graph_state(const rnn_resnet *net, const char **why);
/* ResNet::flops (model.rs:179-198): forward FLOP per image at h x w. */
uint64_t rnn_resnet_flops(const rnn_resnet *net, size_t h, size_t w);

/* ------------------------------------------ debug exports (bit-exact tests) */
/* im2col of ONE image through the same staging index math the conv kernels
 * use: col[cin*k*k][oh*ow] (gather_span, conv.rs:68-120). */
/* The device buffers the train step keeps for block `block` of a ResNet
 * (test access, read-only): which = 0 y1 (c1 output), 1 h (b1 + ReLU), 2 y2
 * (c2 output), 3 ys (shortcut conv output), 4 out (block output), 5 / 6 / 7
 * the output gradients of c1 / c2 / the shortcut conv of the last backward,
 * 8 / 9 the batch mean then invstd of b1 / b2 ([2 cout]), 10 the block's
 * input (the previous block's output; for block 0 the stem's ReLU output).
 * *len: floats. */
int rnn_dbg_resnet_buffer(rnn_resnet *net, size_t block, int which, const float **ptr,
                          size_t *len);
/* The grouped weight-gradient launch(es) of the train step (every 3x3
 * stride-1 conv's dW in one persistent launch), enqueued once more on the
 * context's stream over the buffers the last backward left (its output
 * gradients and activations; the slabs are rewritten with the same values),
 * when `launch` is set.  *flops: the launch's algorithmic FLOP (0 when the
 * current plan has no grouped launch).  No counterpart in the reference: it
 * exists to time that kernel alone (benchmarks). */
int rnn_dbg_resnet_dw_group(rnn_resnet *net, int launch, double *flops);
int rnn_dbg_im2col(rnn_ctx *ctx, const rnn_conv_spec *sp, const float *x_img, float *col);
/* The tile of the specialised forward (dx = 0) or dX kernel for n images on a
 * chip of `cus` CUs: plan[6] = output rows, images, source channels a stage,
 * 32-position groups a wave, waves along output channels, window positions.
 * RNN_E_UNSUPPORTED: the generic kernel.  Host only. */
int rnn_dbg_conv_plan(const rnn_conv_spec *sp, int dx, size_t n, size_t cus, int *plan);
/* PackedA::pack / pack_t (gemm.rs:54-113) into out[nb*256*mpad] (positions the
 * reference never writes are left untouched). */
int rnn_dbg_pack_a(rnn_ctx *ctx, const float *a, size_t m, size_t k, int transposed, float *out);
/* PackedB::pack / pack_t (gemm.rs:340-400) into out[nb*256*npad]. */
int rnn_dbg_pack_b(rnn_ctx *ctx, const float *b, size_t n, size_t k, int transposed, float *out);
/* rel_index computed on the device into idx (device, th*tw*mh*mw u32). */
int rnn_dbg_rel_index(rnn_ctx *ctx, uint32_t th, uint32_t tw, uint32_t mh, uint32_t mw,
                      uint32_t *idx);

#ifdef __cplusplus
}
#endif
#endif
