// enc_hip.hip -- the operators of a transformer encoder layer around its attention op, for gfx950 (MI355X):
// the gated feed-forward block, the residual norm, and the orthogonalised update that trains their weights.
// Hand-written HIP; wave = 64 lanes.  C ABI declared in include/enc_hip.h.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <atomic>
#include <tuple>
#include <type_traits>

#include "enc_hip.h"

namespace {
#include "enc_common.inc"
#include "enc_gemm.inc"
#include "enc_skinny.inc"
#include "enc_pack.inc"
#include "enc_norm.inc"

// ---------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------
// A launch has failed if the runtime says so of that launch.  (The thread's pending error does not tell: one that some other
// library left there, or an earlier failure of the same kind, would hide it.)  Our own failure is reported and does not
// stay pending; an error that was there before a call that succeeds is left alone.
struct Call {
  const char *who;
  hipStream_t st;
  Call(const char *w, void *stream) : who(w), st(static_cast<hipStream_t>(stream)) {}
  template <typename... P, typename... A>
  int launch(void (*kernel)(P...), dim3 blocks, dim3 threads, A... args) const {
    static_assert(sizeof...(P) == sizeof...(A), "the kernel's arguments");
    std::tuple<P...> values(static_cast<P>(args)...);
    void *pointers[sizeof...(P)];
    int at = 0;
    std::apply([&](auto &...v) { ((pointers[at++] = &v), ...); }, values);
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), blocks, threads, pointers, 0, st);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      return fail(ENC_ERR_LAUNCH, "%s: kernel launch failed: %s", who, hipGetErrorString(e));
    }
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return ENC_OK;
  }
};

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }
uint32_t round8(uint32_t v) { return (v + 7u) & ~7u; }
uint32_t ceil_div(size_t a, size_t b) { return (uint32_t)((a + b - 1) / b); }
bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool known_type(int dtype) { return dtype == ENC_F32 || dtype == ENC_BF16 || dtype == ENC_F16; }
int parts_of(int dtype) { return dtype == ENC_F32 ? 3 : 1; }

// Hands out pieces of the caller's workspace; with base == nullptr it only counts.
struct Carve {
  char *base;
  size_t used = 0;
  explicit Carve(void *b) : base(static_cast<char *>(b)) {}
  template <typename T>
  T *take(size_t n) {
    T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
    used += align256(n * sizeof(T));
    return p;
  }
};

#include "enc_ffn_host.inc"
#include "enc_norm_host.inc"
#include "enc_muon_host.inc"

}  // namespace

extern "C" {

int enc_abi_version(void) { return 1; }
const char *enc_last_error(void) { return g_err; }
uint64_t enc_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }

size_t enc_gated_ffn_forward_workspace_bytes(int dtype, int64_t tokens, int64_t width, int64_t hidden, int64_t out_width) {
  return ffn_workspace(dtype, tokens, width, hidden, out_width, false);
}
size_t enc_gated_ffn_backward_workspace_bytes(int dtype, int64_t tokens, int64_t width, int64_t hidden, int64_t out_width) {
  return ffn_workspace(dtype, tokens, width, hidden, out_width, true);
}

size_t enc_gated_ffn_pre_floats(int64_t tokens, int64_t hidden) {
  return tokens < 0 || hidden <= 0 || hidden >= MAX_SIZE ? 0 : pre_floats(tokens, hidden);
}

int enc_gated_ffn_forward(int dtype, int activation, const void *x, int64_t x_stride, const void *w_in, const void *b_in,
                          const void *w_out, const void *b_out, int64_t tokens, int64_t width, int64_t hidden,
                          int64_t out_width, void *y, float *pre, void *workspace, size_t workspace_bytes, void *stream) {
  FfnArgs a = {};
  a.dtype = dtype, a.act = activation, a.x = x, a.x_stride = x_stride, a.w_in = w_in, a.b_in = b_in, a.w_out = w_out;
  a.b_out = b_out, a.M = tokens, a.D = width, a.F = hidden, a.O = out_width, a.y = y, a.pre = pre;
  return ffn_forward(Call("enc_gated_ffn_forward", stream), a, workspace, workspace_bytes);
}

int enc_gated_ffn_backward(int dtype, int activation, const void *x, int64_t x_stride, const void *w_in,
                           const void *w_out, const float *pre, const void *grad, int64_t grad_stride, int64_t tokens,
                           int64_t width, int64_t hidden, int64_t out_width, void *d_x, void *d_w_in, void *d_b_in,
                           void *d_w_out, void *d_b_out, void *workspace, size_t workspace_bytes, void *stream) {
  FfnArgs a = {};
  a.dtype = dtype, a.act = activation, a.x = x, a.x_stride = x_stride, a.w_in = w_in, a.w_out = w_out;
  a.M = tokens, a.D = width, a.F = hidden, a.O = out_width, a.pre = const_cast<float *>(pre);
  a.grad = grad, a.grad_stride = grad_stride, a.d_x = d_x, a.d_w_in = d_w_in, a.d_b_in = d_b_in;
  a.d_w_out = d_w_out, a.d_b_out = d_b_out;
  return ffn_backward(Call("enc_gated_ffn_backward", stream), a, workspace, workspace_bytes);
}

size_t enc_residual_norm_backward_workspace_bytes(int64_t rows, int64_t width, int64_t gate_group) {
  if (check_norm("enc_residual_norm_backward_workspace_bytes", ENC_F32, rows, width, gate_group, NORM_NONE, NORM_NONE)) return 0;
  return norm_backward_workspace(rows, width, gate_group);
}

int enc_residual_norm_forward(int dtype, int inner, int outer, float eps, const void *x, int64_t x_stride, const void *y,
                              int64_t y_stride, const void *gate, int64_t gate_stride, int64_t gate_group, const void *scale,
                              const void *inner_weight, const void *inner_bias, const void *outer_weight,
                              const void *outer_bias, int64_t rows, int64_t width, void *residual, void *normed, float *stats,
                              void *stream) {
  NormArgs a = {};
  a.x = x, a.y = y, a.gate = gate, a.scale = scale, a.iw = inner_weight, a.ib = inner_bias, a.ow = outer_weight, a.ob = outer_bias;
  a.x_ld = (size_t)x_stride, a.y_ld = (size_t)y_stride, a.gate_ld = (size_t)gate_stride;
  a.inner = inner, a.outer = outer, a.eps = eps, a.residual = residual, a.normed = normed, a.stats = stats;
  return norm_forward(Call("enc_residual_norm_forward", stream), dtype, rows, width, gate_group, a);
}

int enc_residual_norm_backward(int dtype, int inner, int outer, const void *x, int64_t x_stride, const void *y, int64_t y_stride,
                               const void *gate, int64_t gate_stride, int64_t gate_group, const void *scale,
                               const void *inner_weight, const void *inner_bias, const void *outer_weight, const float *stats,
                               const void *d_residual, int64_t d_residual_stride, const void *d_normed,
                               int64_t d_normed_stride, int64_t rows, int64_t width, void *d_x, void *d_y, void *d_gate,
                               void *d_scale, void *d_inner_weight, void *d_inner_bias, void *d_outer_weight,
                               void *d_outer_bias, void *workspace, size_t workspace_bytes, void *stream) {
  NormArgs a = {};
  a.x = x, a.y = y, a.gate = gate, a.scale = scale, a.iw = inner_weight, a.ib = inner_bias, a.ow = outer_weight;
  a.x_ld = (size_t)x_stride, a.y_ld = (size_t)y_stride, a.gate_ld = (size_t)gate_stride;
  a.inner = inner, a.outer = outer, a.stats = const_cast<float *>(stats);
  a.d_residual = d_residual, a.dr_ld = (size_t)d_residual_stride, a.d_normed = d_normed, a.dn_ld = (size_t)d_normed_stride;
  a.dx = d_x, a.dy = d_y;
  void *const sums[5] = {d_scale, d_inner_weight, d_inner_bias, d_outer_weight, d_outer_bias};
  return norm_backward(Call("enc_residual_norm_backward", stream), dtype, rows, width, gate_group, a, sums, d_gate, workspace,
                       workspace_bytes);
}

size_t enc_orthogonalize_workspace_bytes(int dtype, int64_t batch, int64_t rows, int64_t cols) {
  if (check_muon("enc_orthogonalize_workspace_bytes", dtype, batch, rows, cols, 1)) return 0;
  return muon_room(dtype, (size_t)batch, (size_t)rows, (size_t)cols, nullptr).bytes;
}

int enc_orthogonalize(int dtype, const void *update, void *out, int64_t batch, int64_t rows, int64_t cols, int steps, float a,
                      float b, float c, float eps, void *workspace, size_t workspace_bytes, void *stream) {
  return orthogonalize(Call("enc_orthogonalize", stream), dtype, update, out, batch, rows, cols, steps, a, b, c, eps, workspace,
                       workspace_bytes);
}

}  // extern "C"
