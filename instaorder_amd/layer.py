"""Operators of an encoder layer around its attention op, on the kernels of libenc_hip.so:

    gated_feed_forward(x, w_in, b_in, w_out, b_out, activation)
    residual_norm(x, y, gate=, scale=, inner=, outer=, ...)

GPU tensors always take the HIP kernels (errors propagate; the autograd nodes are in csrc/enc_bind.cpp); CPU tensors take
an elementary PyTorch path by explicit device dispatch, as ``MSDeformAttn`` does.  On GPU tensors a call refuses to be traced
(``torch.jit.trace``, ``make_fx``): the trace would hold the result's allocation and not the kernels; and it refuses dual
tensors, whose tangents the kernels do not carry."""
import torch
import torch.nn.functional as F

from . import layer_checks, layer_ext

ACTIVATIONS = {"silu": F.silu, "gelu": F.gelu, "sigmoid": torch.sigmoid, "relu": F.relu}


def autocast_dtype(x):
    """The type that autocast runs products in on x's device, None where it is off."""
    device = "cuda" if x.is_cuda else "cpu"
    return torch.get_autocast_dtype(device) if torch.is_autocast_enabled(device) else None


def _cast(tensors, dtype):
    """What autocast casts: floating point tensors below 64 bits.  (Each call casts for itself: nothing is kept.)"""
    return [t.to(dtype) if t is not None and t.is_floating_point() and t.dtype != torch.float64 else t for t in tensors]


def gated_feed_forward(x, w_in, b_in, w_out, b_out, activation="silu"):
    """y = (a * act(b)) W_out^T + b_out with [a | b] = x W_in^T + b_in.

    x [..., width]; w_in [2 * hidden, width] (value rows first, then gate rows -- the order of ``F.glu``); w_out
    [out_width, hidden]; biases may be None.  activation: "silu", "gelu" (by the error function), "sigmoid", "relu".
    fp32, bf16 or fp16, one type for all; sums are fp32, h is rounded to the type at most once (up to 16 tokens it is held in
    two parts of the type, so that there an Inf in w_out gives NaN).  Differentiable once in all five tensors.  fp32 goes through three bf16 parts in the backward pass and in forward passes of many tokens: there an Inf among
    the inputs gives NaN (its parts multiply zeros), a NaN stays one, and values below 2^-110 lose their low bits (their
    parts end at 2^-133).  Under autocast all five are cast to its type, as for ``F.linear``."""
    dtype = autocast_dtype(x)
    if dtype is not None:
        x, w_in, b_in, w_out, b_out = _cast((x, w_in, b_in, w_out, b_out), dtype)
    if x.is_cuda:
        return (layer_ext._bind or layer_ext.bind()).gated_feed_forward(x, w_in, b_in, w_out, b_out, activation)
    layer_checks.gated_feed_forward(x, w_in, b_in, w_out, b_out, activation, ACTIVATIONS)
    dtype = x.dtype                                     # 32 bits inside, one rounding of the result
    x, w_in, b_in, w_out, b_out = _cast((x, w_in, b_in, w_out, b_out), torch.float32)
    with torch.autocast("cpu", enabled=False):
        a, b = F.linear(x, w_in, b_in).chunk(2, -1)
        return F.linear(a * ACTIVATIONS[activation](b), w_out, b_out).to(dtype)


def _cpu_norm(v, kind, weight, bias, eps):
    if kind == "layer":
        return F.layer_norm(v, v.shape[-1:], weight, bias, eps)
    v = v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)
    v = v if weight is None else v * weight
    return v if bias is None else v + bias


def residual_norm(x, y, *, gate=None, scale=None, inner=None, inner_weight=None, inner_bias=None, outer="layer",
                  outer_weight=None, outer_bias=None, eps=1e-5, want_residual=True):
    """The norms before and after a block, with the block's gate and residual scale, in one pass over the rows:

        z = norm_inner(y);  residual = x + gate * scale * z;  normed = norm_outer(residual)

    -> (residual or None, normed or None).  x, y [..., width]; inner / outer: None, "layer" or "rms", each with an
    optional weight and bias [width]; scale [width]; gate of x's shape, or with ones in its last dimensions before the
    width (x [batch, tokens, width], gate [batch, 1, width]: one gate for a sample).  want_residual=False leaves the
    residual in registers.  fp32, bf16 or fp16, one type for all; fp32 inside, each result rounded once.  Differentiable
    once in all eight tensors.  Under autocast all are cast to fp32, as for ``F.layer_norm``."""
    if autocast_dtype(x) is not None:
        x, y, gate, scale, inner_weight, inner_bias, outer_weight, outer_bias = _cast(
            (x, y, gate, scale, inner_weight, inner_bias, outer_weight, outer_bias), torch.float32)
    if x.is_cuda:
        return (layer_ext._bind or layer_ext.bind()).residual_norm(x, y, gate, scale, inner, inner_weight, inner_bias, outer,
                                                                   outer_weight, outer_bias, eps, want_residual)
    layer_checks.residual_norm(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias, want_residual)
    dtype = x.dtype                                     # 32 bits inside, one rounding of each result
    x, y, gate, scale, inner_weight, inner_bias, outer_weight, outer_bias = _cast(
        (x, y, gate, scale, inner_weight, inner_bias, outer_weight, outer_bias), torch.float32)
    z = y if inner is None else _cpu_norm(y, inner, inner_weight, inner_bias, eps)
    z = z if gate is None else z * gate
    r = x + (z if scale is None else z * scale)
    n = None if outer is None else _cpu_norm(r, outer, outer_weight, outer_bias, eps).to(dtype)
    return r.to(dtype) if want_residual else None, n
