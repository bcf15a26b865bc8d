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
 * Weights are contiguous.  `pre`: NULL, or [tokens, 2 * round_up(hidden, 8)] floats that the backward pass takes
 * (a in the first half of a row, b in the second).
 * Backward: `grad` = gradient of y.  Any of the five results may be NULL; the others are fully written.
 * Limits: every size < 2^22, tokens < 2^31 / 256.
 */
size_t enc_gated_ffn_forward_workspace_bytes(int dtype, int64_t tokens, int64_t width, int64_t hidden, int64_t out_width);
size_t enc_gated_ffn_backward_workspace_bytes(int dtype, int64_t tokens, int64_t width, int64_t hidden, int64_t out_width);

int enc_gated_ffn_forward(int dtype, int activation, const void *x, int64_t x_stride, const void *w_in, const void *b_in,
                          const void *w_out, const void *b_out, int64_t tokens, int64_t width, int64_t hidden,
                          int64_t out_width, void *y, float *pre, void *workspace, size_t workspace_bytes, void *stream);

int enc_gated_ffn_backward(int dtype, int activation, const void *x, int64_t x_stride, const void *w_in,
                           const void *w_out, const float *pre, const void *grad, int64_t grad_stride, int64_t tokens,
                           int64_t width, int64_t hidden, int64_t out_width, void *d_x, void *d_w_in, void *d_b_in,
                           void *d_w_out, void *d_b_out, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ENC_HIP_H_ */
