"""Checks of the layer operators' arguments for their CPU paths: what the compiled binding (csrc/enc_bind.cpp) checks for GPU
tensors, with the same words, so that CPU tensors need no build.  Under torch.jit.trace, where sizes are values of the trace and
asking about them is not, nothing is checked beyond what torch's own operators check."""
import functools

import torch

from .layer_ext import DTYPES, NORM_MAX_WIDTH


def _require(condition, text, *args):
    if not condition:
        raise RuntimeError(text % args)


_NAMES = {torch.float32: "Float", torch.float64: "Double", torch.float16: "Half", torch.bfloat16: "BFloat16", torch.bool: "Bool",
          torch.uint8: "Byte", torch.int8: "Char", torch.int16: "Short", torch.int32: "Int", torch.int64: "Long"}


def _name(dtype):
    return _NAMES.get(dtype, str(dtype))


def _not_while_tracing(check):
    @functools.wraps(check)
    def checked(*args):
        if not torch.jit.is_tracing():
            check(*args)
    return checked


def _type(what, x):
    _require(x.dtype in DTYPES, "%s: not implemented for %s", what, _name(x.dtype))


def _like(what, x, name, t, shape):
    """t, unless absent: of x's dtype, on x's device, of the shape."""
    if t is None:
        return
    _require(t.dtype == x.dtype, "%s: %s has dtype %s, not %s", what, name, _name(t.dtype), _name(x.dtype))
    _require(t.device == x.device, "%s: %s is on %s, not on %s", what, name, t.device, x.device)
    _require(list(t.shape) == list(shape), "%s: %s has shape %s, not %s", what, name, list(t.shape), list(shape))


@_not_while_tracing
def gated_feed_forward(x, w_in, b_in, w_out, b_out, activation, activations):
    what = "gated_feed_forward"
    _require(activation in activations, "%s: unknown activation '%s' (one of %s)", what, activation, ", ".join(sorted(activations)))
    _type(what, x)
    _require(x.dim() >= 1 and w_in.dim() == 2 and w_out.dim() == 2 and w_in.shape[0] % 2 == 0,
             "%s: expected x [..., width], w_in [2 * hidden, width], w_out [out_width, hidden]", what)
    width, hidden, out_width = x.shape[-1], w_in.shape[0] // 2, w_out.shape[0]
    _require(min(width, hidden, out_width) >= 1, "%s: width, hidden and out_width must be at least 1", what)
    for name, t, shape in (("w_in", w_in, (2 * hidden, width)), ("b_in", b_in, (2 * hidden,)), ("w_out", w_out, (out_width, hidden)),
                           ("b_out", b_out, (out_width,))):
        _like(what, x, name, t, shape)


@_not_while_tracing
def residual_norm(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias, want_residual):
    what = "residual_norm"
    for kind in (inner, outer):
        _require(kind in (None, "layer", "rms"), "%s: inner and outer are None, 'layer' or 'rms', got '%s'", what, kind)
    _type(what, x)
    _require(x.dim() >= 1 and 1 <= x.shape[-1] <= NORM_MAX_WIDTH, "%s: x must be [..., width] with a width of 1 to %d", what,
             NORM_MAX_WIDTH)
    _require(outer is not None or want_residual, "%s: without an outer norm the residual is the only result", what)
    _like(what, x, "y", y, x.shape)
    for name, t in (("scale", scale), ("inner_weight", inner_weight), ("inner_bias", inner_bias), ("outer_weight", outer_weight),
                    ("outer_bias", outer_bias)):
        _like(what, x, name, t, x.shape[-1:])
    _require((inner is not None or (inner_weight is None and inner_bias is None))
             and (outer is not None or (outer_weight is None and outer_bias is None)), "%s: a weight or bias of a norm that is None", what)
    if gate is None:
        return
    lead = list(x.shape[:-1])                           # x's shape, or ones in the last dimensions before the width
    k = len(lead)
    while gate.dim() == x.dim() and k and gate.shape[k - 1] == 1:
        k -= 1
    _like(what, x, "gate", gate, lead[:k] + [1] * (len(lead) - k) + [x.shape[-1]])


def orthogonalize(update, steps, dtype):
    what = "orthogonalize"
    _type(what, update)
    _require(dtype in (None, update.dtype) or (update.dtype == torch.float32 and dtype in DTYPES),
             "%s: a result of %s is not made of an update of %s", what, _name(dtype or update.dtype), _name(update.dtype))
    _require(update.dim() >= 2 and min(update.shape[-2:]) >= 1, "%s: update must be [..., rows, cols] with at least one of each", what)
    _require(1 <= steps <= 100, "%s: steps must be 1 to 100", what)
