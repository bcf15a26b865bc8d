/*
 * enc_hip.h -- C ABI of libenc_hip.so: the operators of a transformer encoder layer around its attention op, for AMD
 * MI355X (gfx950), hand-written HIP.
 *
 * Conventions (all entry points):
 *   - tensor pointers are DEVICE pointers, inputs are read-only; rows are contiguous and `*_stride` is the number of
 *     elements from one row to the next;
 *   - `dtype` is the type of every tensor of the call that is not declared float; sums are fp32 or wider;
 *   - `stream` is a hipStream_t passed as void* (NULL = the default stream); work is enqueued asynchronously on the
 *     current device, nothing synchronises with the host and nothing is allocated: scratch memory is the caller's
 *     `workspace` (256-byte aligned, at least the size that the *_workspace_bytes query gives, contents irrelevant
 *     before and after; calls that share one must be ordered on one stream);
 *   - no exceptions; return 0 on success, non-zero on error, and enc_last_error() then returns a thread-local text;
 *   - results do not depend on the run: no atomics on sums.
 */
#ifndef ENC_HIP_H_
#define ENC_HIP_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ENC_OK 0
#define ENC_ERR_INVALID_ARGUMENT 1
#define ENC_ERR_LAUNCH 2

#define ENC_F32 0
#define ENC_BF16 1
#define ENC_F16 2
/* enc_orthogonalize and its workspace query: | ENC_BF16 or ENC_F16, the result's type, of an update in fp32 */
#define ENC_UPDATE_F32 16
/* the workspace queries of the feed-forward block: | the dtype, for a call whose tensors can be read where they lie: every
 * address a multiple of 16 bytes, every row stride a multiple of 8 elements and below 2^22.  Without it there is room to lay
 * all of them out, which is enough for any call. */
#define ENC_IN_PLACE 32

#define ENC_ACT_SILU 0
#define ENC_ACT_GELU 1 /* x * Phi(x), by the error function */
#define ENC_ACT_SIGMOID 2
#define ENC_ACT_RELU 3

int enc_abi_version(void);
const char *enc_last_error(void);
uint64_t enc_launch_count(void);

/*
 * Gated feed-forward block.
 *   [a | b] = x W_in^T + b_in        x [tokens, width], w_in [2 * hidden, width], b_in [2 * hidden] or NULL
 *   h = a * act(b)                   a: the first `hidden` columns (value), b: the others (gate), the order of F.glu
 *   y = h W_out^T + b_out            w_out [out_width, hidden], b_out [out_width] or NULL, y [tokens, out_width]
 * Weights are contiguous.  `pre`: NULL, or enc_gated_ffn_pre_floats(tokens, hidden) floats (16-byte aligned) that the
 * backward pass takes: a and b in fp32, in the library's own order.
 * Backward: `grad` = gradient of y.  Any of the five results may be NULL; the others are fully written.
 * Limits: every size < 2^22, tokens < 2^31 / 256.
 */
size_t enc_gated_ffn_forward_workspace_bytes(int dtype, int64_t tokens, int64_t width, int64_t hidden, int64_t out_width);
size_t enc_gated_ffn_backward_workspace_bytes(int dtype, int64_t tokens, int64_t width, int64_t hidden, int64_t out_width);

size_t enc_gated_ffn_pre_floats(int64_t tokens, int64_t hidden);

int enc_gated_ffn_forward(int dtype, int activation, const void *x, int64_t x_stride, const void *w_in, const void *b_in,
                          const void *w_out, const void *b_out, int64_t tokens, int64_t width, int64_t hidden,
                          int64_t out_width, void *y, float *pre, void *workspace, size_t workspace_bytes, void *stream);

int enc_gated_ffn_backward(int dtype, int activation, const void *x, int64_t x_stride, const void *w_in,
                           const void *w_out, const float *pre, const void *grad, int64_t grad_stride, int64_t tokens,
                           int64_t width, int64_t hidden, int64_t out_width, void *d_x, void *d_w_in, void *d_b_in,
                           void *d_w_out, void *d_b_out, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Residual norm: the norms before and after a block, with the block's gate and residual scale.
 *   z = norm_inner(y)  (y itself: ENC_NORM_NONE)
 *   r = x + gate * scale * z
 *   n = norm_outer(r)
 *   norm: ENC_NORM_LAYER (v - mean) / sqrt(var + eps) * weight + bias;  ENC_NORM_RMS v / sqrt(mean(v^2) + eps) * weight + bias
 * x, y [rows, width]; gate NULL or [rows / gate_group, width], row i / gate_group belongs to row i (gate_group 1: a gate
 * for each row); scale, weights and biases NULL (absent) or [width].  Width at most ENC_NORM_MAX_WIDTH; rows need no alignment.
 * residual: r, may be NULL if there is an outer norm; normed: n, not written without one.  stats: NULL, or 4 floats a
 * row (16-byte aligned) that the backward pass takes.
 * Backward: d_normed is needed with an outer norm; d_residual may be NULL with one and is needed without.  d_x and d_y
 * may be NULL.  Any of the others may be NULL; those given are fully written (zeros for no rows).
 */
#define ENC_NORM_NONE 0
#define ENC_NORM_LAYER 1
#define ENC_NORM_RMS 2
#define ENC_NORM_MAX_WIDTH 16384

size_t enc_residual_norm_backward_workspace_bytes(int64_t rows, int64_t width, int64_t gate_group);

int enc_residual_norm_forward(int dtype, int inner, int outer, float eps, const void *x, int64_t x_stride, const void *y,
                              int64_t y_stride, const void *gate, int64_t gate_stride, int64_t gate_group, const void *scale,
                              const void *inner_weight, const void *inner_bias, const void *outer_weight,
                              const void *outer_bias, int64_t rows, int64_t width, void *residual, void *normed, float *stats,
                              void *stream);

int enc_residual_norm_backward(int dtype, int inner, int outer, const void *x, int64_t x_stride, const void *y, int64_t y_stride,
                               const void *gate, int64_t gate_stride, int64_t gate_group, const void *scale,
                               const void *inner_weight, const void *inner_bias, const void *outer_weight, const float *stats,
                               const void *d_residual, int64_t d_residual_stride, const void *d_normed,
                               int64_t d_normed_stride, int64_t rows, int64_t width, void *d_x, void *d_y, void *d_gate,
                               void *d_scale, void *d_inner_weight, void *d_inner_bias, void *d_outer_weight,
                               void *d_outer_bias, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Orthogonalised update (Newton-Schulz steps of the Muon optimiser), a batch of contiguous matrices [batch, rows, cols]:
 *   X = update / max(|update|, eps)   (Frobenius norm, summed in 64 bits)
 *   `steps` times:  A = X X^T;  X = a X + (b A + c A A) X      (on the short side: A = X^T X and X from the left if rows > cols)
 * out: X in `dtype`; it may be `update` itself.  Iterates keep 24 bits (ENC_F32) or 16 (the 16-bit types).  With
 * ENC_UPDATE_F32 the update is fp32 and only the result has 16 bits: values that the type does not reach keep their direction.
 * Limits: steps 1 to 100, batch < 65536, the short side at most 65536.
 */
size_t enc_orthogonalize_workspace_bytes(int dtype, int64_t batch, int64_t rows, int64_t cols);

int enc_orthogonalize(int dtype, const void *update, void *out, int64_t batch, int64_t rows, int64_t cols, int steps, float a,
                      float b, float c, float eps, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ENC_HIP_H_ */
