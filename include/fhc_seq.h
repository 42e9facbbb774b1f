/* fhc_seq: operators of a recurrent block on rows of channels, on MI355X (gfx950), as a C ABI: a gated linear
 * recurrence along a sequence, the norms around a block with its gate and the scaled residual, a gated feed-forward
 * block, a short causal convolution along a sequence, a selective state space scan, and a matrix product with bias,
 * activation and residual, each with its backward pass. The rows are tokens of sequences, or the pixels of NHWC feature
 * maps over the frames of a stream (a frame's map is then one time step, a pixel one sequence). The reference has no
 * counterpart: its network keeps nothing from one frame pair to the next.
 *
 * Conventions are those of fhc_conv.h: 0 on success, a negative value on error with the message in fhc_last_error()
 * (thread-local); nothing aborts or throws; the library allocates nothing and never synchronises, so calls can be
 * captured in a HIP graph. Calls are asynchronous on `stream` (a hipStream_t; NULL = the null stream) of the current
 * device. Workspaces are the caller's: of the size the *_bytes function gives for the same descriptor, 256-byte
 * aligned, uninitialised, not shared by calls that may overlap. Values are held in `dtype`; sums, norms, states and
 * everything between an input and an output are f32 unless a comment says otherwise, and each output is rounded once
 * (to nearest even). An output must not overlap an input or another output, except where a comment allows it.
 */
#ifndef FHC_SEQ_H
#define FHC_SEQ_H
#include <stddef.h>
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

#define FHC_F16 0u
#define FHC_BF16 1u
#define FHC_F32 2u

/* Element (b, t, ch) of a sequence tensor at p[b * bs + t * ts + ch], strides in elements. A dense [b][t][d] tensor
 * has bs = t * d, ts = d; frames of feature maps, [t][pixels][d], have bs = d, ts = pixels * d. An input's elements may
 * coincide (bs = 0: one sequence for all; windows that overlap), an output's may not. */
typedef struct fhc_seq {
    void* p;
    int64_t bs, ts;
} fhc_seq;

/* ---- The gated linear recurrence, per sequence b and channel ch, from the state h_0:
 *     log a_t = -rate * softplus(lam[ch]) * sigmoid(r_t)
 *     h_t     = a_t * h_(t-1) + sqrt(1 - a_t^2) * sigmoid(i_t) * x_t,   y_t = h_t
 * r and i are the logits of the recurrence and input gates, lam an f32 weight. With `lengths` (device memory, one per
 * sequence, clamped to [0, t]) positions at and past a sequence's length are not read, y and the gradients there are
 * 0, and the state stays as it is. */
typedef struct fhc_glr_desc {
    uint32_t dtype;         /* FHC_F16, FHC_BF16 or FHC_F32: of x, r, i, y and their gradients                     */
    uint32_t b, t, d;       /* sequences, steps, channels; any may be 0. b * d below 2^31                            */
    float rate;             /* finite, >= 0                                                                          */
    const float* lam;       /* device, [d]                                                                           */
    const int32_t* lengths; /* device, [b], or NULL: every sequence has t steps                                      */
} fhc_glr_desc;

/* Bytes of the states that a training forward keeps for the backward pass, and of the workspace of either call
 * (0 for many shapes: a NULL workspace is then fine). 0 for a bad descriptor. */
size_t fhc_glr_states_bytes(const fhc_glr_desc* g);
size_t fhc_glr_workspace_bytes(const fhc_glr_desc* g, int backward);

/* h0: [b][d] f32, or NULL for zeros. ht: the state after the last step, [b][d] f32, or NULL; it may be h0 itself
 * (a server's state, updated in place). states: NULL, or the buffer that the backward pass of the same descriptor
 * takes. A call with t = 1 is the single-token step. */
int fhc_glr_forward(const fhc_glr_desc* g, const fhc_seq* x, const fhc_seq* r, const fhc_seq* i, const float* h0,
                    const fhc_seq* y, float* ht, float* states, void* ws, size_t ws_bytes, void* stream);

/* The gradients of a loss with dy = dL/dy and dht = dL/dht ([b][d] f32, or NULL for zeros): dx, dr, di in dtype, dlam
 * [d] f32, dh0 [b][d] f32 (NULL: not wanted). The inputs are those of the forward call, `states` what it wrote. */
int fhc_glr_backward(const fhc_glr_desc* g, const fhc_seq* x, const fhc_seq* r, const fhc_seq* i, const float* states,
                     const fhc_seq* dy, const float* dht, const fhc_seq* dx, const fhc_seq* dr, const fhc_seq* di,
                     float* dlam, float* dh0, void* ws, size_t ws_bytes, void* stream);

/* ---- The norms around a block, its gate and the scaled residual, for each row of c channels:
 *     y = alpha * x + gate[row / rows_per_group] * w_post * o / rms(o),   rms(v) = sqrt(mean(v^2) + eps)
 *     u = w_pre * y / rms(y)                                             (of y before its rounding)
 * o is the block's output, x the residual stream, u the next block's input. o NULL leaves the block out (y = alpha *
 * x: the first block's norm); w_post, gate or w_pre NULL is 1. gate is dense [groups][c] in dtype (a FiLM vector per
 * image, a vector per sequence, or per row with rows_per_group 1), the last group may be short. */
typedef struct fhc_norm_desc {
    uint32_t dtype;
    uint32_t rows, c;            /* c <= 16384; rows 0 is a no-op (the backward pass still writes its sums: 0)      */
    uint32_t rows_per_group;     /* >= 1; read only where gate is given                                              */
    float alpha, eps;            /* finite; eps > 0                                                                  */
    const void *w_post, *w_pre;  /* device, [c] in dtype, or NULL                                                    */
    const void* gate;            /* device, or NULL                                                                  */
} fhc_norm_desc;

/* Element (row, ch) at p[row * ld + ch]; ld >= c. */
typedef struct fhc_rows {
    void* p;
    int64_t ld;
} fhc_rows;

/* y or u NULL: not wanted (not both). y may be x, and u may be o or x, element for element. */
int fhc_norm_block(const fhc_norm_desc* n, const fhc_rows* x, const fhc_rows* o, const fhc_rows* y, const fhc_rows* u,
                   void* stream);

size_t fhc_norm_block_workspace_bytes(const fhc_norm_desc* n);

/* dy, du: dL/dy and dL/du (NULL for zeros, not both). dx and dout (= dL/do) in dtype, the sums dw_post, dw_pre [c] and
 * dgate [groups][c] in f32. Without o: dout, dw_post and dgate are NULL. Sums that are not wanted may be NULL. dx may
 * be dy, dout may be du, element for element. */
int fhc_norm_block_backward(const fhc_norm_desc* n, const fhc_rows* x, const fhc_rows* o, const fhc_rows* dy,
                            const fhc_rows* du, const fhc_rows* dx, const fhc_rows* dout, float* dw_post, float* dgate,
                            float* dw_pre, void* ws, size_t ws_bytes, void* stream);

/* ---- The gated feed-forward block on rows of c channels, f wide inside:
 *     y = h wd^T,   h = act(x wg^T) * (x wu^T)      act: silu, v sigmoid(v), or gelu in its tanh form
 * wg, wu are dense [f][c], wd dense [c][f], in dtype (f16 or bf16). The products accumulate in f32; h, and in the
 * backward pass dL/d(x wg^T) and dL/d(x wu^T), are rounded to dtype once, since they are the next products' operands
 * (the matrix units take 16 bits). A training forward keeps x wg^T and x wu^T in f32, or, for few channels and many
 * rows, the backward pass computes them again: no gradient is taken at a rounded value. f16: the caller scales the loss
 * so that these stay in f16's range. */
#define FHC_ACT_SILU 0u
#define FHC_ACT_GELU 1u

typedef struct fhc_ffn_desc {
    uint32_t dtype; /* FHC_F16 or FHC_BF16 */
    uint32_t act;   /* FHC_ACT_SILU, FHC_ACT_GELU */
    uint32_t rows, c, f; /* c, f <= 2^20 */
} fhc_ffn_desc;

/* Bytes of what a training forward keeps for the backward pass, and of the workspace of either call. */
size_t fhc_ffn_saved_bytes(const fhc_ffn_desc* d);
size_t fhc_ffn_workspace_bytes(const fhc_ffn_desc* d, int backward);

/* saved: NULL, or a 256-byte aligned buffer that the backward pass of the same descriptor takes. */
int fhc_ffn_forward(const fhc_ffn_desc* d, const fhc_rows* x, const void* wg, const void* wu, const void* wd,
                    const fhc_rows* y, void* saved, void* ws, size_t ws_bytes, void* stream);

/* dx and the weights' gradients (dense, in dtype) for dy; those that are not wanted may be NULL. Without rows x, dy and
 * dx are not read, and the weights' gradients are 0. */
int fhc_ffn_backward(const fhc_ffn_desc* d, const fhc_rows* x, const void* wg, const void* wu, const void* wd,
                     const void* saved, const fhc_rows* dy, const fhc_rows* dx, void* dwg, void* dwu, void* dwd,
                     void* ws, size_t ws_bytes, void* stream);

/* ---- The short causal convolution along a sequence, per channel, over k taps (2 to 4). With e the k - 1 rows of
 * `state` and then the sequence's own n rows:
 *     y_t = act(v_t),   v_t = bias[ch] + sum over j < k of w[ch][j] * e[t + j]       (tap k - 1 meets x_t itself)
 * and e's last k - 1 rows are the state of a call that goes on from here. With `lengths` positions at and past a
 * sequence's length are not read, and y and the gradients there are 0. */
#define FHC_ACT_IDENTITY 2u

typedef struct fhc_short_conv_desc {
    uint32_t dtype;         /* FHC_F16, FHC_BF16 or FHC_F32: of x, w, bias, the states, y, dx                        */
    uint32_t act;           /* FHC_ACT_SILU or FHC_ACT_IDENTITY                                                      */
    uint32_t b, t, d, k;    /* sequences, steps, channels (any may be 0, b * d below 2^31); 2 <= k <= 4              */
    const void* w;          /* device, dense [d][k]                                                                  */
    const void* bias;       /* device, [d], or NULL                                                                  */
    const int32_t* lengths; /* device, [b], or NULL: every sequence has t steps                                      */
} fhc_short_conv_desc;

/* state: [b][k - 1][d], the oldest row first, or NULL for zeros. state_out: the same layout, or NULL; it may be state
 * itself (a server's state, updated in place). */
int fhc_short_conv_forward(const fhc_short_conv_desc* g, const fhc_seq* x, const void* state, const fhc_seq* y,
                           void* state_out, void* stream);

/* 0 for a bad descriptor */
size_t fhc_short_conv_workspace_bytes(const fhc_short_conv_desc* g);

/* The gradients of a loss with dy = dL/dy and dstate_out = dL/dstate_out ([b][k - 1][d] in dtype, or NULL for zeros): dx
 * in dtype, dw [d][k] and dbias [d] in f32, dstate [b][k - 1][d] in dtype (each may be NULL: not wanted). */
int fhc_short_conv_backward(const fhc_short_conv_desc* g, const fhc_seq* x, const void* state, const fhc_seq* dy,
                            const void* dstate_out, const fhc_seq* dx, float* dw, float* dbias, void* dstate, void* ws,
                            size_t ws_bytes, void* stream);

/* ---- The selective state space scan. Every channel of a sequence has n states; B and C are vectors of n for each
 * position and group of channels (channel ch is in group ch / (d / groups)):
 *     D_t    = softplus(dt_t + dt_bias[ch])
 *     h_t[k] = exp(D_t a[ch][k]) h_(t-1)[k] + D_t x_t B_t[k]
 *     y_t    = (sum over k of C_t[k] h_t[k] + skip[ch] x_t) silu(z_t)
 * a, dt_bias and skip are f32 weights; z may be left out (no gate). With `lengths` positions at and past a sequence's
 * length are not read, y and the gradients there are 0, and the state stays as it is. a may be above 0 (states that grow) as
 * long as a step's exp(D a) is in f32's range. From a step on whose D or D x is not finite, its channel's y and states are
 * infinite or NaN. */
typedef struct fhc_ssm_desc {
    uint32_t dtype;          /* FHC_F16, FHC_BF16 or FHC_F32: of x, dt, z, B, C, y and their gradients               */
    uint32_t b, t, d;        /* sequences, steps, channels; any may be 0. b * d below 2^31                            */
    uint32_t n, groups;      /* states a channel, 1 to 64; groups, a divisor of d. groups * n below 2^31              */
    const float* a;          /* device, dense [d][n]                                                                  */
    const float* dt_bias;    /* device, [d], or NULL: zeros                                                           */
    const float* skip;       /* device, [d], or NULL: zeros                                                           */
    const int32_t* lengths;  /* device, [b], or NULL                                                                  */
} fhc_ssm_desc;

/* Bytes of the states that a training forward keeps for the backward pass, and of the workspace of either call
 * (0 for many shapes: a NULL workspace is then fine). 0 for a bad descriptor. */
size_t fhc_ssm_states_bytes(const fhc_ssm_desc* g);
size_t fhc_ssm_workspace_bytes(const fhc_ssm_desc* g, int backward);

/* bm and cm: B and C, sequence tensors of groups * n channels. z NULL: no gate. h0: [b][d][n] f32, or NULL for zeros.
 * ht: the state after the last step, [b][d][n] f32, or NULL; it may be h0 itself. states: NULL, or the 256-byte aligned
 * buffer that the backward pass of the same descriptor takes. A call with t = 1 is the single-token step. */
int fhc_ssm_forward(const fhc_ssm_desc* g, const fhc_seq* x, const fhc_seq* dt, const fhc_seq* bm, const fhc_seq* cm,
                    const fhc_seq* z, const float* h0, const fhc_seq* y, float* ht, float* states, void* ws,
                    size_t ws_bytes, void* stream);

/* The gradients of a loss with dy = dL/dy and dht = dL/dht ([b][d][n] f32, or NULL for zeros): dx, ddt, dbm, dcm and dz
 * (NULL without z) in dtype; da [d][n], ddt_bias [d], dskip [d] and dh0 [b][d][n] in f32 (those may be NULL: not wanted).
 * The inputs are those of the forward call, `states` what it wrote. */
int fhc_ssm_backward(const fhc_ssm_desc* g, const fhc_seq* x, const fhc_seq* dt, const fhc_seq* bm, const fhc_seq* cm,
                     const fhc_seq* z, const float* states, const fhc_seq* dy, const float* dht, const fhc_seq* dx,
                     const fhc_seq* ddt, const fhc_seq* dbm, const fhc_seq* dcm, const fhc_seq* dz, float* da,
                     float* ddt_bias, float* dskip, float* dh0, void* ws, size_t ws_bytes, void* stream);

/* ---- The matrix product with its epilogue, on rows of c channels, f wide:
 *     y = act(v) + residual,   v = x w^T + bias
 * w is dense [f][c], bias [f], in dtype (f16 or bf16); act FHC_ACT_SILU, FHC_ACT_GELU or FHC_ACT_IDENTITY. v and the sum
 * are f32, y is rounded once. A training forward with silu or gelu keeps v in f32. dx and dw are products of dL/dv as two
 * numbers of dtype, its rounding and the remainder; FHC_LINEAR_ROUND_DV, added to act, leaves the remainder out, for half
 * the work at silu and gelu (dbias sums dL/dv before its rounding in both). The residual's gradient is dy itself. */
#define FHC_LINEAR_ROUND_DV 0x100u

typedef struct fhc_linear_desc {
    uint32_t dtype; /* FHC_F16 or FHC_BF16 */
    uint32_t act;   /* and FHC_LINEAR_ROUND_DV, which the forward pass does not look at */
    uint32_t rows, c, f; /* c, f <= 2^20 */
} fhc_linear_desc;

/* Bytes of what a training forward keeps for the backward pass (0: nothing, NULL is then fine), and of the workspace of
 * either call. */
size_t fhc_linear_saved_bytes(const fhc_linear_desc* d);
size_t fhc_linear_workspace_bytes(const fhc_linear_desc* d, int backward);

/* bias and residual may be NULL. y may be the residual, element for element. saved: NULL, or a 256-byte aligned buffer
 * that the backward pass of the same descriptor takes. */
int fhc_linear_forward(const fhc_linear_desc* d, const fhc_rows* x, const void* w, const void* bias,
                       const fhc_rows* residual, const fhc_rows* y, void* saved, void* ws, size_t ws_bytes,
                       void* stream);

/* dx and dw (dense) in dtype, dbias [f] f32, for dy; those that are not wanted may be NULL. Without rows x, dy and dx are
 * not read, and dw and dbias are 0. */
int fhc_linear_backward(const fhc_linear_desc* d, const fhc_rows* x, const void* w, const void* saved,
                        const fhc_rows* dy, const fhc_rows* dx, void* dw, float* dbias, void* ws, size_t ws_bytes,
                        void* stream);

#ifdef __cplusplus
}
#endif
#endif
