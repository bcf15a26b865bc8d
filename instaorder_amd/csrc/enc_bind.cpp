// enc_bind.cpp -- Python binding of the layer operators that are called several times a training step: checks,
// allocation, torch's current stream and the autograd nodes, on top of the C ABI of libenc_hip.so (include/enc_hip.h).
// Host code only.  A ctypes binding with Python autograd functions spent 170-200 us a forward and backward call, ten
// times the kernels of a small block; this one holds the interpreter for the forward call alone.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <string>

#include "enc_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

int dtype_code(const char *what, const Tensor &x) {
  switch (x.scalar_type()) {
    case at::kFloat: return ENC_F32;
    case at::kBFloat16: return ENC_BF16;
    case at::kHalf: return ENC_F16;
    default: TORCH_CHECK(false, what, ": not implemented for ", x.scalar_type());
  }
}

int activation_code(const std::string &name) {
  if (name == "silu") return ENC_ACT_SILU;
  if (name == "gelu") return ENC_ACT_GELU;
  if (name == "sigmoid") return ENC_ACT_SIGMOID;
  if (name == "relu") return ENC_ACT_RELU;
  TORCH_CHECK(false, "gated_feed_forward: unknown activation '", name, "' (one of gelu, relu, sigmoid, silu)");
}

int norm_code(const std::optional<std::string> &name) {
  if (!name) return ENC_NORM_NONE;
  if (*name == "layer") return ENC_NORM_LAYER;
  if (*name == "rms") return ENC_NORM_RMS;
  TORCH_CHECK(false, "residual_norm: inner and outer are None, 'layer' or 'rms', got '", *name, "'");
}

// Defined tensors: on x's device, of its dtype, of the shape.
void check(const char *what, const Tensor &x, const char *name, const Tensor &t, at::IntArrayRef shape) {
  if (!t.defined()) return;
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), what, ": ", name, " has dtype ", t.scalar_type(), ", not ", x.scalar_type());
  TORCH_CHECK(t.device() == x.device(), what, ": ", name, " is on ", t.device(), ", not on ", x.device());
  TORCH_CHECK(t.sizes() == shape, what, ": ", name, " has shape ", t.sizes(), ", not ", shape);
}

Tensor given(const MaybeTensor &t) { return t ? *t : Tensor(); }
Tensor flat(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// A tensor (or a 2-D view or copy of it) with contiguous rows, and the elements from one to the next.
struct Rows {
  Tensor t;
  int64_t stride = 0;
  Rows() = default;
  explicit Rows(const Tensor &v) {
    if (!v.defined()) return;
    const int64_t width = v.size(-1);
    t = v, stride = width;
    if (v.is_contiguous()) return;
    t = v.reshape({-1, width});
    if ((t.stride(1) != 1 && width != 1) || (t.size(0) > 1 && t.stride(0) < width)) t = t.contiguous();
    if (t.size(0) > 1) stride = t.stride(0);
  }
};

void *stream_of(const Tensor &x) { return c10::hip::getCurrentHIPStream(x.device().index()).stream(); }
Tensor workspace(size_t bytes, const Tensor &x) {
  return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}
void done(const char *what, int rc) { TORCH_CHECK(rc == ENC_OK, what, ": ", enc_last_error()); }
void on_gpu(const Tensor &x) { TORCH_CHECK(x.is_cuda(), "Not implemented on the CPU"); }

// A trace records torch's own operators: of a call here it would keep the allocation of the result and lose the launch that
// fills it.  Under a mode of fake tensors there is no memory to launch on.
void not_traced(const char *what) {
  typedef c10::impl::TorchDispatchModeTLS Modes;
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY) &&
                  !Modes::get_mode(c10::impl::TorchDispatchModeKey::FAKE),
              what, ": cannot be traced (the trace would not hold the kernels)");
}

// The kernels carry no tangents: a dual tensor's would be lost without a word.
void no_tangents(const char *what, at::ArrayRef<Tensor> tensors) {
  for (const Tensor &t : tensors)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), what, ": forward-mode derivatives are not implemented");
}

// Gradients that were formed by kernels: differentiating them again is an error, not zero.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor &g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is differentiable once", (int64_t)grads.size());
  return (*error)(std::move(grads));
}

// Optional inputs that are absent have no edge in the graph: which of a node's inputs are there, as bits, and whether
// input i wants its gradient.
int64_t present(std::initializer_list<Tensor> inputs) {
  int64_t bits = 0, bit = 1;
  for (const Tensor &t : inputs) {
    if (t.defined()) bits |= bit;
    bit <<= 1;
  }
  return bits;
}
bool needs(AutogradContext *ctx, int i) {
  const int64_t bits = ctx->saved_data["present"].toInt();
  if (!((bits >> i) & 1)) return false;
  return ctx->needs_input_grad((size_t)__builtin_popcountll((uint64_t)bits & ((1ull << i) - 1)));
}
MaybeTensor maybe(const Tensor &t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

// ---- gated feed-forward block -----------------------------------------------------------------
struct FfnSizes {
  int64_t width, hidden, out_width;
};
FfnSizes check_ffn(const Tensor &x, const Tensor &w_in, const Tensor &b_in, const Tensor &w_out, const Tensor &b_out) {
  const char *what = "gated_feed_forward";
  dtype_code(what, x);
  TORCH_CHECK(x.dim() >= 1 && w_in.dim() == 2 && w_out.dim() == 2 && w_in.size(0) % 2 == 0, what,
              ": expected x [..., width], w_in [2 * hidden, width], w_out [out_width, hidden]");
  const FfnSizes s = {x.size(-1), w_in.size(0) / 2, w_out.size(0)};
  TORCH_CHECK(s.width >= 1 && s.hidden >= 1 && s.out_width >= 1, what, ": width, hidden and out_width must be at least 1");
  check(what, x, "w_in", w_in, {2 * s.hidden, s.width});
  check(what, x, "b_in", b_in, {2 * s.hidden});
  check(what, x, "w_out", w_out, {s.out_width, s.hidden});
  check(what, x, "b_out", b_out, {s.out_width});
  return s;
}

// The workspace query's type: can the tensors be read where they lie?
bool aligned16(const Tensor &t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
bool lies_well(const Rows &r) { return aligned16(r.t) && r.stride % 8 == 0 && r.stride < ((int64_t)1 << 22); }

Tensor ffn_forward(const Tensor &x, const Tensor &w_in, const Tensor &b_in, const Tensor &w_out, const Tensor &b_out, int act, Tensor *pre) {
  const char *what = "gated_feed_forward";
  not_traced(what);
  const FfnSizes s = check_ffn(x, w_in, b_in, w_out, b_out);
  on_gpu(x);
  const c10::DeviceGuard guard(x.device());
  const Rows rows(x);
  const Tensor wi = flat(w_in), bi = flat(b_in), wo = flat(w_out), bo = flat(b_out);
  const int code = dtype_code(what, x);
  const int64_t tokens = x.numel() / s.width;
  auto shape = x.sizes().vec();
  shape.back() = s.out_width;
  const Tensor y = at::empty(shape, x.options().requires_grad(false));
  if (pre) *pre = at::empty({(int64_t)enc_gated_ffn_pre_floats(tokens, s.hidden)}, x.options().dtype(at::kFloat).requires_grad(false));
  const int placed = lies_well(rows) && aligned16(wi) && aligned16(wo) ? ENC_IN_PLACE : 0;
  const size_t bytes = enc_gated_ffn_forward_workspace_bytes(code | placed, tokens, s.width, s.hidden, s.out_width);
  const Tensor ws = workspace(bytes, x);
  done(what, enc_gated_ffn_forward(code, act, ptr(rows.t), rows.stride, ptr(wi), ptr(bi), ptr(wo), ptr(bo), tokens, s.width, s.hidden,
                                   s.out_width, ptr(y), pre ? pre->data_ptr<float>() : nullptr, ptr(ws), bytes, stream_of(x)));
  return y;
}

// Saves x, the two weights and the pre-activations a, b in fp32 (8 bytes a hidden value, what a 16-bit eager block keeps in
// four tensors): activation, slope, h, da and db are formed from unrounded values, and the last three rounded to the type
// once, where they become operands.
struct GatedFeedForward : public torch::autograd::Function<GatedFeedForward> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w_in, const MaybeTensor &b_in, const Tensor &w_out,
                        const MaybeTensor &b_out, int64_t act) {
    Tensor pre;
    const Tensor bi = given(b_in), bo = given(b_out), y = ffn_forward(x, w_in, bi, w_out, bo, (int)act, &pre);
    ctx->saved_data["act"] = act;
    ctx->saved_data["present"] = present({x, w_in, bi, w_out, bo});
    ctx->save_for_backward({x, w_in, w_out, pre});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const char *what = "gated_feed_forward backward";
    not_traced(what);
    no_tangents(what, grads);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &pre = saved[3], &grad = grads[0];
    const c10::DeviceGuard guard(x.device());
    const Tensor wi = flat(saved[1]), wo = flat(saved[2]);
    const int64_t width = x.size(-1), hidden = wo.size(1), out_width = wo.size(0), tokens = x.numel() / width;
    auto shape = x.sizes().vec();
    shape.back() = out_width;
    check(what, x, "grad", grad, shape);
    const Rows rows(x), g(grad);
    const int code = dtype_code(what, x);
    const auto options = x.options().requires_grad(false);
    const std::vector<int64_t> shapes[5] = {x.sizes().vec(), {2 * hidden, width}, {2 * hidden}, {out_width, hidden}, {out_width}};
    variable_list out(6);
    for (int i = 0; i < 5; ++i)
      if (needs(ctx, i)) out[i] = at::empty(shapes[i], options);
    const int placed = lies_well(rows) && lies_well(g) && aligned16(wi) && aligned16(wo) ? ENC_IN_PLACE : 0;
    const size_t bytes = enc_gated_ffn_backward_workspace_bytes(code | placed, tokens, width, hidden, out_width);
    const Tensor ws = workspace(bytes, x);
    done(what, enc_gated_ffn_backward(code, (int)ctx->saved_data["act"].toInt(), ptr(rows.t), rows.stride, ptr(wi), ptr(wo),
                                      pre.data_ptr<float>(), ptr(g.t), g.stride, tokens, width, hidden, out_width, ptr(out[0]), ptr(out[1]),
                                      ptr(out[2]), ptr(out[3]), ptr(out[4]), ptr(ws), bytes, stream_of(x)));
    return once(std::move(out));
  }
};

bool wants_grad(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor &t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

Tensor gated_feed_forward(const Tensor &x, const Tensor &w_in, const MaybeTensor &b_in, const Tensor &w_out, const MaybeTensor &b_out,
                          const std::string &activation) {
  const int act = activation_code(activation);
  const Tensor bi = given(b_in), bo = given(b_out);
  no_tangents("gated_feed_forward", {x, w_in, bi, w_out, bo});
  if (wants_grad({x, w_in, bi, w_out, bo})) return GatedFeedForward::apply(x, w_in, maybe(bi), w_out, maybe(bo), (int64_t)act);
  return ffn_forward(x, w_in, bi, w_out, bo, act, nullptr);
}

// ---- residual norm ----------------------------------------------------------------------------
struct NormInputs {
  Tensor x, y, gate, scale, iw, ib, ow, ob;
};
// Rows of x that share one row of the gate.
int64_t check_norm(const NormInputs &t, int inner, int outer, bool want_residual) {
  const char *what = "residual_norm";
  dtype_code(what, t.x);
  TORCH_CHECK(t.x.dim() >= 1 && t.x.size(-1) >= 1 && t.x.size(-1) <= ENC_NORM_MAX_WIDTH, what, ": x must be [..., width] with a width of 1 to ",
              ENC_NORM_MAX_WIDTH);
  TORCH_CHECK(outer != ENC_NORM_NONE || want_residual, what, ": without an outer norm the residual is the only result");
  const auto shape = t.x.sizes();
  const at::IntArrayRef width = shape.slice(shape.size() - 1);
  check(what, t.x, "y", t.y, shape);
  check(what, t.x, "scale", t.scale, width);
  check(what, t.x, "inner_weight", t.iw, width);
  check(what, t.x, "inner_bias", t.ib, width);
  check(what, t.x, "outer_weight", t.ow, width);
  check(what, t.x, "outer_bias", t.ob, width);
  TORCH_CHECK((inner != ENC_NORM_NONE || (!t.iw.defined() && !t.ib.defined())) && (outer != ENC_NORM_NONE || (!t.ow.defined() && !t.ob.defined())),
              what, ": a weight or bias of a norm that is None");
  if (!t.gate.defined()) return 1;
  // x's shape, or ones in the last dimensions before the width: rows that share a gate (a dimension of x that is 1 itself
  // among them adds none)
  size_t k = shape.size() - 1;
  if (t.gate.dim() == t.x.dim())
    while (k && t.gate.size(k - 1) == 1) --k;
  auto want = shape.vec();
  int64_t group = 1;
  for (size_t i = k; i + 1 < shape.size(); ++i) {
    group *= shape[i];
    want[i] = 1;
  }
  check(what, t.x, "gate", t.gate, want);
  return group < 1 ? 1 : group;
}

struct NormResults {
  Tensor residual, normed, stats;
  int64_t group;
};
NormResults norm_forward(const NormInputs &t, int inner, int outer, double eps, bool want_residual, bool keep) {
  const char *what = "residual_norm";
  not_traced(what);
  NormResults r;
  r.group = check_norm(t, inner, outer, want_residual);
  on_gpu(t.x);
  const c10::DeviceGuard guard(t.x.device());
  const Rows x(t.x), y(t.y), gate(t.gate);
  const Tensor scale = flat(t.scale), iw = flat(t.iw), ib = flat(t.ib), ow = flat(t.ow), ob = flat(t.ob);
  const int64_t width = t.x.size(-1), rows = t.x.numel() / width;
  const auto options = t.x.options().requires_grad(false);
  if (want_residual) r.residual = at::empty(t.x.sizes(), options);
  if (outer != ENC_NORM_NONE) r.normed = at::empty(t.x.sizes(), options);
  if (keep) r.stats = at::empty({rows, 4}, options.dtype(at::kFloat));
  done(what, enc_residual_norm_forward(dtype_code(what, t.x), inner, outer, (float)eps, ptr(x.t), x.stride, ptr(y.t), y.stride, ptr(gate.t),
                                       gate.stride, r.group, ptr(scale), ptr(iw), ptr(ib), ptr(ow), ptr(ob), rows, width, ptr(r.residual),
                                       ptr(r.normed), static_cast<float *>(ptr(r.stats)), stream_of(t.x)));
  return r;
}

// Saves the inputs and four statistics a row; both rows are formed again in the backward pass.
struct ResidualNorm : public torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &y, const MaybeTensor &gate, const MaybeTensor &scale,
                               const MaybeTensor &iw, const MaybeTensor &ib, const MaybeTensor &ow, const MaybeTensor &ob, int64_t inner,
                               int64_t outer, double eps, bool want_residual) {
    const NormInputs t = {x, y, given(gate), given(scale), given(iw), given(ib), given(ow), given(ob)};
    const NormResults r = norm_forward(t, (int)inner, (int)outer, eps, want_residual, true);
    ctx->saved_data["present"] = present({t.x, t.y, t.gate, t.scale, t.iw, t.ib, t.ow, t.ob});
    ctx->saved_data["inner"] = inner;
    ctx->saved_data["outer"] = outer;
    ctx->saved_data["group"] = r.group;
    ctx->saved_data["residual"] = want_residual;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, y, t.gate, t.scale, t.iw, t.ib, t.ow, r.stats});
    variable_list out;
    if (want_residual) out.push_back(r.residual);
    if (outer != ENC_NORM_NONE) out.push_back(r.normed);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    const char *what = "residual_norm backward";
    not_traced(what);
    no_tangents(what, grads);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &y = saved[1], &gate = saved[2], &stats = saved[7];
    const int inner = (int)ctx->saved_data["inner"].toInt(), outer = (int)ctx->saved_data["outer"].toInt();
    const bool has_residual = ctx->saved_data["residual"].toBool();
    const int64_t group = ctx->saved_data["group"].toInt();
    variable_list out(12);
    const Tensor d_residual = has_residual ? grads[0] : Tensor();
    Tensor d_normed = outer != ENC_NORM_NONE ? grads[has_residual ? 1 : 0] : Tensor();
    if (!d_residual.defined() && !d_normed.defined()) return out;
    const c10::DeviceGuard guard(x.device());
    check(what, x, "d_residual", d_residual, x.sizes());
    check(what, x, "d_normed", d_normed, x.sizes());
    if (outer != ENC_NORM_NONE && !d_normed.defined()) d_normed = at::zeros(x.sizes(), x.options().requires_grad(false));
    const Rows xr(x), yr(y), gr(gate), dr(d_residual), dn(d_normed);
    const Tensor scale = flat(saved[3]), iw = flat(saved[4]), ib = flat(saved[5]), ow = flat(saved[6]);
    const int64_t width = x.size(-1), rows = x.numel() / width;
    const auto options = x.options().requires_grad(false);
    // y added as it is: x and y have one gradient, the same tensor, as for x + y
    const bool plain = !gate.defined() && !scale.defined() && inner == ENC_NORM_NONE;
    const bool need_x = needs(ctx, 0), need_y = needs(ctx, 1);
    if (need_x || (plain && need_y)) out[0] = at::empty(x.sizes(), options);
    if (need_y && !plain) out[1] = at::empty(x.sizes(), options);
    if (needs(ctx, 2)) out[2] = rows ? at::empty(gate.sizes(), options) : at::zeros(gate.sizes(), options);   // a gate of no rows
    for (int i = 3; i < 8; ++i)
      if (needs(ctx, i)) out[i] = at::empty({width}, options);
    const size_t bytes = enc_residual_norm_backward_workspace_bytes(rows, width, group);
    const Tensor ws = workspace(bytes, x);
    done(what, enc_residual_norm_backward(dtype_code(what, x), inner, outer, ptr(xr.t), xr.stride, ptr(yr.t), yr.stride, ptr(gr.t), gr.stride,
                                          group, ptr(scale), ptr(iw), ptr(ib), ptr(ow), stats.data_ptr<float>(), ptr(dr.t), dr.stride,
                                          ptr(dn.t), dn.stride, rows, width, ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(out[3]), ptr(out[4]),
                                          ptr(out[5]), ptr(out[6]), ptr(out[7]), ptr(ws), bytes, stream_of(x)));
    if (plain && need_y) out[1] = out[0];
    if (!need_x) out[0] = Tensor();
    return once(std::move(out));
  }
};

std::tuple<MaybeTensor, MaybeTensor> residual_norm(const Tensor &x, const Tensor &y, const MaybeTensor &gate, const MaybeTensor &scale,
                                                   const std::optional<std::string> &inner, const MaybeTensor &inner_weight,
                                                   const MaybeTensor &inner_bias, const std::optional<std::string> &outer,
                                                   const MaybeTensor &outer_weight, const MaybeTensor &outer_bias, double eps,
                                                   bool want_residual) {
  const NormInputs t = {x, y, given(gate), given(scale), given(inner_weight), given(inner_bias), given(outer_weight), given(outer_bias)};
  const int in = norm_code(inner), out = norm_code(outer);
  Tensor residual, normed;
  no_tangents("residual_norm", {t.x, t.y, t.gate, t.scale, t.iw, t.ib, t.ow, t.ob});
  if (wants_grad({t.x, t.y, t.gate, t.scale, t.iw, t.ib, t.ow, t.ob})) {
    const variable_list r = ResidualNorm::apply(t.x, t.y, maybe(t.gate), maybe(t.scale), maybe(t.iw), maybe(t.ib), maybe(t.ow), maybe(t.ob), (int64_t)in, (int64_t)out, eps, want_residual);
    if (want_residual) residual = r[0];
    if (out != ENC_NORM_NONE) normed = r.back();
  } else {
    const NormResults r = norm_forward(t, in, out, eps, want_residual, false);
    residual = r.residual, normed = r.normed;
  }
  return {maybe(residual), maybe(normed)};
}

// ---- orthogonalised update --------------------------------------------------------------------
typedef std::optional<at::ScalarType> MaybeType;
// The C entry's type: the result's, the update's own if none is given; of an fp32 update also a 16-bit one.
int check_orthogonalize(const Tensor &update, int64_t steps, MaybeType type) {
  const char *what = "orthogonalize";
  int code = dtype_code(what, update);
  if (type && *type != update.scalar_type()) {
    TORCH_CHECK(code == ENC_F32 && (*type == at::kBFloat16 || *type == at::kHalf), what, ": a result of ", *type, " is not made of an update of ",
                update.scalar_type());
    code = (*type == at::kHalf ? ENC_F16 : ENC_BF16) | ENC_UPDATE_F32;
  }
  TORCH_CHECK(update.dim() >= 2 && update.size(-1) >= 1 && update.size(-2) >= 1, what, ": update must be [..., rows, cols] with at least one of each");
  TORCH_CHECK(steps >= 1 && steps <= 100, what, ": steps must be 1 to 100");
  return code;
}

Tensor orthogonalize(const Tensor &given_update, int64_t steps, double a, double b, double c, double eps, MaybeType type) {
  const char *what = "orthogonalize";
  not_traced(what);
  no_tangents(what, {given_update});
  const int code = check_orthogonalize(given_update, steps, type);
  on_gpu(given_update);
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(given_update.device());
  const Tensor update = given_update.contiguous();
  const Tensor out = at::empty(update.sizes(), update.options().dtype(type ? *type : update.scalar_type()).requires_grad(false));
  const int64_t rows = update.size(-2), cols = update.size(-1), batch = update.numel() / (rows * cols);
  const size_t bytes = enc_orthogonalize_workspace_bytes(code, batch, rows, cols);
  const Tensor ws = workspace(bytes, update);
  done(what, enc_orthogonalize(code, ptr(update), ptr(out), batch, rows, cols, (int)steps, (float)a, (float)b, (float)c, (float)eps, ptr(ws),
                               bytes, stream_of(update)));
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("gated_feed_forward", &gated_feed_forward);
  m.def("residual_norm", &residual_norm);
  m.def("orthogonalize", &orthogonalize, py::arg("update"), py::arg("steps"), py::arg("a"), py::arg("b"), py::arg("c"), py::arg("eps"),
        py::arg("dtype") = py::none());
  m.def("launch_count", &enc_launch_count);
}
