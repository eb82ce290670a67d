/* ugdr model operators around the MoE exchange: the experts' gated feed-forward block (forward and
 * backward) on rows grouped by expert, as ugdr_x_moe_dispatch leaves them in the receive area, and
 * the global gradient norm with clipping.  No counterpart in the reference.
 *
 * All launch functions are asynchronous on `stream` (a cudaStream_t of the current device, NULL
 * for the legacy stream), allocate nothing, may be captured into a CUDA graph, and return a
 * cudaError_t value: cudaErrorInvalidValue for refused arguments, with nothing launched.  Calls on
 * different streams may run at the same time as long as they share no output or scratch memory. */
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define UGDR_X_TYPE_BF16 0
#define UGDR_X_TYPE_FP16 1
#define UGDR_X_TYPE_FP32 2

#define UGDR_X_ACT_SILU 0 /* a(g) = g / (1 + exp(-g)) */
#define UGDR_X_ACT_GELU 1 /* a(g) = g (1 + erf(g / sqrt 2)) / 2 */

#define UGDR_X_EXPERTS_MAX 4096             /* experts */
#define UGDR_X_EXPERTS_MAX_ROWS (1u << 28)   /* rows of a call */
#define UGDR_X_EXPERTS_MAX_SIZE (1 << 20)    /* hidden and inner */

/* A rank's experts and the grouping of the rows: expert e's rows are the counts[e] rows after those
 * of experts 0 .. e - 1.  The counts are read on the device, so no call waits for the host; rows
 * behind the last group are neither read for a result nor written.  Tensors are contiguous and
 * 16-byte aligned, hidden and inner multiples of 8, type BF16 or FP16.  Sums are fp32; h, dg and du
 * are rounded to the type once, as operands of the next product (so with FP16 they must stay within
 * its range, as x and y must).
 * *status (a device word, not cleared by the calls) becomes 1 when a bounded wait inside a kernel
 * ran out and 2 when a count is negative or the counts add up to more than `rows`; negative counts
 * then count as 0 and rows past `rows` are dropped. */
typedef struct ugdr_x_experts {
    const int32_t *counts; /* [nexp] */
    const void *w_in;      /* [nexp][2][inner][hidden]: the gate's, then the up projection's rows */
    const void *w_out;     /* [nexp][hidden][inner] */
    unsigned int *status;
    uint64_t rows;         /* rows of x, dy, y, ... */
    int nexp;
    int hidden;
    int inner;
    int type;
    int act;
} ugdr_x_experts;

/* Bound, in ns, of every wait inside the kernels of the calls below that are launched from now on (0: the
 * default, 5 s).  Returns the one before.  A wait takes as long as the longest tile of a product, so a
 * bound of less than some milliseconds can run out in calls that are fine. */
uint64_t ugdr_x_set_expert_wait_ns(uint64_t ns);

/* Forward: g = x Wg^T, u = x Wu^T, h = a(g) * u, y = h Wo^T.  `h` ([rows][inner]) is scratch of a
 * serving call; with `gu` ([rows][2][inner] floats on a 32-byte boundary, may be NULL) g and u are kept
 * too, and h and gu are what the backward pass takes.  y may be x itself (the products with x are over by then). */
int ugdr_x_expert_ffn(const ugdr_x_experts *m, const void *x, void *y, void *h, float *gu, void *stream);

/* Backward of y with respect to x and the weights, from dy and what the forward pass kept:
 * dh = dy Wo, dg = dh * u * a'(g), du = dh * a(g), dx = dg Wg + du Wu, dw_in = (dg^T x, du^T x),
 * dw_out = dy^T h.  The gradients of an expert without rows are zeros.  `dgu` ([rows][2][inner]) is
 * scratch.  dx may be x or dy itself; the other outputs overlap nothing. */
int ugdr_x_expert_ffn_backward(const ugdr_x_experts *m, const void *dy, const void *x, const void *h, const float *gu,
                               void *dgu, void *dx, void *dw_in, void *dw_out, void *stream);

/* One gradient tensor of a plan: `count` elements of `grad_type` at `grad`, scaled into `out` as
 * elements of `out_type` (grad_type, or FP32).  `out` is `grad` itself, with the same type, or memory
 * that overlaps no gradient and no other output; ugdr_x_grad_plan refuses a tensor whose `out` overlaps
 * its own `grad` in any other way.  Pointers are aligned to their element. */
typedef struct ugdr_x_grad {
    const void *grad;
    void *out;
    uint64_t count;
    int32_t grad_type;
    int32_t out_type;
} ugdr_x_grad;

/* A plan is the tensor list as the kernels read it.  ugdr_x_grad_plan_bytes gives its size for n
 * tensors; ugdr_x_grad_plan writes it to host memory and its chunk count to *chunks; the caller
 * copies it to 16-byte aligned device memory and passes it with n and the chunk count to the calls
 * below.  `partials` is scratch of UGDR_X_GRAD_PARTIALS doubles of a call's own. */
#define UGDR_X_GRAD_PARTIALS 2048
size_t ugdr_x_grad_plan_bytes(int n);
int ugdr_x_grad_plan(const ugdr_x_grad *grads, int n, void *plan, uint64_t *chunks);

/* *sum_squares = sum over all tensors of the squares of their elements (a double on the device). */
int ugdr_x_grad_sum_squares(const void *plan, int n, uint64_t chunks, double *partials, double *sum_squares,
                            void *stream);

/* norm = sqrt(s), out = grad * min(1, max_norm / (norm + 1e-6)), *norm_out = norm, where s is
 * *sum_squares, or with sum_squares NULL the sum over this plan.  Gradients that are scaled in
 * place and are within the limit are not written. */
int ugdr_x_grad_clip(const void *plan, int n, uint64_t chunks, double *partials, const double *sum_squares,
                     float max_norm, float *norm_out, void *stream);

#ifdef __cplusplus
}
#endif
