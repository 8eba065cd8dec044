/*
 * evamx_dense: products on 16-bit weights for MI355X (gfx950), one matrix for all rows or one for each
 * expert's sorted rows (evamx_sort_tokens), with bias, activation and residual, and their gradients. A
 * library of its own (libevamx_dense.so) beside libevamx.so, with the same conventions: device pointers,
 * a hipStream_t, no allocation and no synchronisation with the host, negative codes with a message from
 * evamx_dense_last_error() (thread-local). No counterpart in the reference.
 */
#ifndef EVAMX_DENSE_H
#define EVAMX_DENSE_H

#include "evamx.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { EVAMX_DENSE_VERSION = 1 };
enum { EVAMX_ACT_NONE = 0, EVAMX_ACT_SILU = 1, EVAMX_ACT_GELU = 2, EVAMX_ACT_RELU = 3, EVAMX_ACT_SWIGLU = 4 };

const char* evamx_dense_last_error(void);
int evamx_dense_version(void);

/* y[r] = act(W_e x[r] + b_e) + residual[r] for the rows starts[e] .. starts[e + 1] - 1 of each expert e, or for all rows
 * with starts == NULL (experts = 1). Rows behind starts[experts] are not read, and zeros in y. act: SiLU, GELU (x Phi(x)),
 * ReLU, or SwiGLU, min(silu(v[n]), limit) * clamp(v[inter + n], -limit, limit) for n < inter = n_out / 2 (limit 0: none; the first
 * half of W's rows are the gate's, the second the up product's). All of dtype (fp16 or bf16); fp32 sums, rounded once. Rows
 * with unit column strides of any alignment; rows of 16-byte addresses and strides are faster, others may be copied first. starts
 * of any content neither read nor write outside of the given rows. No output overlaps an input, but y may be the residual. A SwiGLU
 * matrix (with its row stride) of 3.75 GiB or more is refused for more than a few rows. */
typedef struct evamx_linear_args {
    const void* x;               /* [rows][x_stride] */
    const void* w;               /* [experts][w_expert_stride]: rows [n_out][w_stride] */
    const void* bias;            /* [experts][n_out] or NULL */
    const void* residual;        /* [rows][residual_stride], n_out (inter) values a row, or NULL */
    void* y;                     /* [rows][y_stride] */
    float* pre;                  /* fp32 [rows][n_out], what the activation takes (for the gradient), or NULL; rows behind
                                  * starts[experts] stay as they were */
    const int32_t* starts;       /* [experts + 1] or NULL */
    void* workspace;             /* 16-byte aligned, evamx_linear_workspace_bytes bytes; needs no clearing */
    size_t workspace_bytes;
    int64_t x_stride, w_stride, w_expert_stride, residual_stride, y_stride;   /* elements */
    int32_t dtype, rows, n_in, n_out, experts, act;
    float limit;
} evamx_linear_args;
/* rows 0..2^24, n_in and n_out 1..EVAMX_W4_MAX_DIM, experts 1..1024. May be 0. direct: x and w (for the gradient also grad) have 16-byte addresses and strides (w's matrices too), no row stride is above 2^21, and n_in (n_out) is a
 * multiple of 8 values; otherwise a call may copy them into the workspace. */
size_t evamx_linear_workspace_bytes(int rows, int n_in, int n_out, int experts, int grouped, int direct);
int evamx_linear(const evamx_linear_args* args, evamx_stream_t stream);

/* The gradients of evamx_linear. With D = act'(pre) * grad (rounded to dtype where there is an activation),
 *   grad_x[r] = W_e^T D[r],  grad_w_e = sum_r D[r] x[r]^T,  grad_bias_e = sum_r D[r]  over the expert's rows,
 * in fp32, rounded once; zeros for rows behind the last and for experts without rows. The residual's gradient is grad. */
typedef struct evamx_linear_grad_args {
    const void* grad;            /* [rows][grad_stride], n_out (inter) values a row */
    const void* x;               /* as in evamx_linear_args; may be NULL without grad_w */
    const void* w;               /* may be NULL without grad_x */
    const float* pre;            /* fp32 [rows][n_out] of the forward call; NULL without activation */
    const int32_t* starts;
    void* grad_x;                /* [rows][grad_x_stride] or NULL */
    void* grad_w;                /* [experts][n_out][n_in] or NULL */
    void* grad_bias;             /* [experts][n_out] or NULL */
    void* workspace;
    size_t workspace_bytes;
    int64_t grad_stride, x_stride, w_stride, w_expert_stride, grad_x_stride;
    int32_t dtype, rows, n_in, n_out, experts, act;
    float limit;
} evamx_linear_grad_args;
size_t evamx_linear_grad_workspace_bytes(int rows, int n_in, int n_out, int experts, int grouped, int act, int direct);
int evamx_linear_grad(const evamx_linear_grad_args* args, evamx_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* EVAMX_DENSE_H */
