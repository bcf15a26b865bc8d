"""Host side of libenc_hip.so (include/enc_hip.h): the operators of an encoder layer around its attention op.  Checks,
allocation and the current stream are here, as ``ext.py`` has them for the attention op: outputs are new tensors on the
inputs' device, kernels are enqueued on torch's current HIP stream without synchronising, every error is a RuntimeError,
and there is no fallback -- a missing library, a CPU tensor or a failed launch raises.

Nothing is kept between calls: workspaces come from torch's caching allocator, so calls on several streams, and captured
graphs with their own memory pools, share none."""
import ctypes
import math
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "libenc_hip.so")
_lib = None

_I, _L, _Z, _P, _F = ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_float

NORMS = {None: 0, "layer": 1, "rms": 2}
NORM_MAX_WIDTH = 16384
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2, "relu": 3}


def _load():
    """dlopen libenc_hip.so (after torch, so both share one HIP runtime)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(_LIB_PATH):
        raise RuntimeError("libenc_hip.so is not built: run `python -m instaorder_amd.build_ext` (needs hipcc); "
                           "there is no fallback implementation")
    lib = ctypes.CDLL(_LIB_PATH)
    for name, args, res in (
            ("enc_abi_version", [], _I), ("enc_last_error", [], ctypes.c_char_p), ("enc_launch_count", [], ctypes.c_uint64),
            ("enc_gated_ffn_forward_workspace_bytes", [_I] + [_L] * 4, _Z),
            ("enc_gated_ffn_backward_workspace_bytes", [_I] + [_L] * 4, _Z),
            ("enc_gated_ffn_pre_floats", [_L, _L], _Z),
            ("enc_gated_ffn_forward", [_I, _I, _P, _L] + [_P] * 4 + [_L] * 4 + [_P] * 3 + [_Z, _P], _I),
            ("enc_gated_ffn_backward", [_I, _I, _P, _L] + [_P] * 4 + [_L] * 5 + [_P] * 6 + [_Z, _P], _I),
            ("enc_orthogonalize_workspace_bytes", [_I] + [_L] * 3, _Z),
            ("enc_orthogonalize", [_I, _P, _P] + [_L] * 3 + [_I] + [_F] * 4 + [_P, _Z, _P], _I),
            ("enc_residual_norm_backward_workspace_bytes", [_L] * 3, _Z),
            ("enc_residual_norm_forward",
             [_I, _I, _I, _F, _P, _L, _P, _L, _P, _L, _L] + [_P] * 5 + [_L, _L] + [_P] * 4, _I),
            ("enc_residual_norm_backward",
             [_I, _I, _I, _P, _L, _P, _L, _P, _L, _L] + [_P] * 5 + [_P, _L, _P, _L, _L, _L] + [_P] * 9 + [_Z, _P], _I)):
        f = getattr(lib, name)
        f.argtypes, f.restype = args, res
    if lib.enc_abi_version() != 1:
        raise RuntimeError("libenc_hip.so ABI version mismatch")
    _lib = lib
    return lib


def launch_count():
    """Kernel launches issued through the library so far (proof the HIP path ran)."""
    return int(_load().enc_launch_count())


def _raise(lib, what):
    raise RuntimeError("%s: %s" % (what, lib.enc_last_error().decode("utf-8", "replace")))


# The hot calls below take microseconds on the GPU, so their host side is kept short: one pass over the arguments, no
# views of contiguous tensors, the stream's handle without a Stream object.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _check(what, device, dtype, *triples):
    """Each (name, tensor or None, shape): on the device, of the dtype, of the shape."""
    for name, t, shape in triples:
        if t is None:
            continue
        if t.dtype != dtype:
            raise RuntimeError("%s: %s has dtype %s, not %s" % (what, name, t.dtype, dtype))
        if t.device != device:
            raise RuntimeError("%s: %s is on %s, not on %s" % (what, name, t.device, device))
        if t.shape != shape:
            raise RuntimeError("%s: %s has shape %s, not %s" % (what, name, tuple(t.shape), tuple(shape)))


def _rows(t):
    """(t, or a 2-D view or copy of it, with contiguous rows; elements from one row to the next)"""
    if t.is_contiguous():
        return t, t.shape[-1]
    t = t.reshape(-1, t.shape[-1])
    if (t.stride(1) != 1 and t.shape[1] != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _flat(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _here(t):
    """The index of t's device when it is the current one (launches and allocations go there), else None: the caller
    enters `torch.cuda.device(t.device)` and starts again."""
    if not t.is_cuda:
        raise RuntimeError("Not implemented on the CPU")
    index = t.get_device()
    return index if index == torch.cuda.current_device() else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, device):
    return torch.empty((nbytes,), dtype=torch.uint8, device=device) if nbytes else None


# ---- gated feed-forward block -----------------------------------------------------------------
def check_gated_ffn(x, w_in, b_in, w_out, b_out, activation):
    """(hidden, out_width); raises what the block refuses."""
    what = "gated_feed_forward"
    if activation not in ACTIVATIONS:
        raise RuntimeError("%s: unknown activation %r (one of %s)" % (what, activation, ", ".join(sorted(ACTIVATIONS))))
    if x.dtype not in DTYPES:
        raise RuntimeError("%s: not implemented for %s" % (what, x.dtype))
    if x.dim() < 1 or w_in.dim() != 2 or w_out.dim() != 2 or w_in.shape[0] % 2:
        raise RuntimeError("%s: expected x [..., width], w_in [2 * hidden, width], w_out [out_width, hidden]" % what)
    width, hidden, out_width = x.shape[-1], w_in.shape[0] // 2, w_out.shape[0]
    if min(width, hidden, out_width) < 1:
        raise RuntimeError("%s: width, hidden and out_width must be at least 1" % what)
    _check(what, x.device, x.dtype, ("w_in", w_in, (2 * hidden, width)), ("b_in", b_in, (2 * hidden,)),
           ("w_out", w_out, (out_width, hidden)), ("b_out", b_out, (out_width,)))
    return hidden, out_width


def gated_ffn_forward(x, w_in, b_in, w_out, b_out, activation, keep):
    """-> (y [..., out_width], pre); pre: what the backward pass takes, or None unless `keep`."""
    hidden, out_width = check_gated_ffn(x, w_in, b_in, w_out, b_out, activation)
    here = _here(x)
    if here is None:
        with torch.cuda.device(x.device):
            return gated_ffn_forward(x, w_in, b_in, w_out, b_out, activation, keep)
    lib = _lib or _load()
    rows, stride = _rows(x)
    w_in, b_in, w_out, b_out = _flat(w_in), _flat(b_in), _flat(w_out), _flat(b_out)
    width, code, device = x.shape[-1], DTYPES[x.dtype], x.device
    tokens = x.numel() // width
    y = torch.empty((*x.shape[:-1], out_width), dtype=x.dtype, device=device)
    pre = torch.empty((lib.enc_gated_ffn_pre_floats(tokens, hidden),), dtype=torch.float32, device=device) if keep else None
    nbytes = lib.enc_gated_ffn_forward_workspace_bytes(code, tokens, width, hidden, out_width)
    ws = _workspace(nbytes, device)
    if lib.enc_gated_ffn_forward(code, ACTIVATIONS[activation], rows.data_ptr(), stride, w_in.data_ptr(), _ptr(b_in),
                                 w_out.data_ptr(), _ptr(b_out), tokens, width, hidden, out_width, y.data_ptr(), _ptr(pre),
                                 _ptr(ws), nbytes, _raw_stream(here)):
        _raise(lib, "gated_feed_forward")
    return y, pre


def gated_ffn_backward(x, w_in, w_out, pre, grad, activation, needs):
    """-> (d_x, d_w_in, d_b_in, d_w_out, d_b_out), None where `needs` says False.  The other arguments are the forward
    call's, which checked them."""
    here = _here(x)
    if here is None:
        with torch.cuda.device(x.device):
            return gated_ffn_backward(x, w_in, w_out, pre, grad, activation, needs)
    width, hidden, out_width = x.shape[-1], w_in.shape[0] // 2, w_out.shape[0]
    _check("gated_feed_forward backward", x.device, x.dtype, ("grad", grad, (*x.shape[:-1], out_width)))
    lib = _lib or _load()
    rows, stride = _rows(x)
    g, g_stride = _rows(grad)
    w_in, w_out = _flat(w_in), _flat(w_out)
    code, device, dtype = DTYPES[x.dtype], x.device, x.dtype
    tokens = x.numel() // width
    shapes = (x.shape, w_in.shape, (2 * hidden,), w_out.shape, (out_width,))
    outs = [torch.empty(s, dtype=dtype, device=device) if n else None for s, n in zip(shapes, needs)]
    nbytes = lib.enc_gated_ffn_backward_workspace_bytes(code, tokens, width, hidden, out_width)
    ws = _workspace(nbytes, device)
    if lib.enc_gated_ffn_backward(code, ACTIVATIONS[activation], rows.data_ptr(), stride, w_in.data_ptr(), w_out.data_ptr(),
                                  pre.data_ptr(), g.data_ptr(), g_stride, tokens, width, hidden, out_width,
                                  *[None if t is None else t.data_ptr() for t in outs], _ptr(ws), nbytes, _raw_stream(here)):
        _raise(lib, "gated_feed_forward backward")
    return outs


# ---- residual norm ----------------------------------------------------------------------------
def check_residual_norm(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias, want_residual):
    """Rows of x that share one row of the gate; raises what the operator refuses."""
    what = "residual_norm"
    if inner not in NORMS or outer not in NORMS:
        raise RuntimeError("%s: inner and outer are None, 'layer' or 'rms'" % what)
    if x.dtype not in DTYPES:
        raise RuntimeError("%s: not implemented for %s" % (what, x.dtype))
    if x.dim() < 1 or not 1 <= x.shape[-1] <= NORM_MAX_WIDTH:
        raise RuntimeError("%s: x must be [..., width] with a width of 1 to %d" % (what, NORM_MAX_WIDTH))
    if outer is None and not want_residual:
        raise RuntimeError("%s: without an outer norm the residual is the only result" % what)
    width = x.shape[-1:]
    _check(what, x.device, x.dtype, ("y", y, x.shape), ("scale", scale, width), ("inner_weight", inner_weight, width),
           ("inner_bias", inner_bias, width), ("outer_weight", outer_weight, width), ("outer_bias", outer_bias, width))
    if (inner is None and not (inner_weight is None and inner_bias is None)) or (
            outer is None and not (outer_weight is None and outer_bias is None)):
        raise RuntimeError("%s: a weight or bias of a norm that is None" % what)
    if gate is None:
        return 1
    # x's shape, or ones in the last dimensions before the width: rows that share a gate
    lead, given = x.shape[:-1], gate.shape[:-1]
    k = len(lead)
    if gate.dim() == x.dim():
        while k and given[k - 1] == 1 and lead[k - 1] != 1:
            k -= 1
    _check(what, x.device, x.dtype, ("gate", gate, (*lead[:k], *[1] * (len(lead) - k), *width)))
    return max(math.prod(lead[k:]), 1)


def residual_norm_forward(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias, eps,
                          want_residual, keep):
    """-> (residual or None, normed or None, stats or None, rows that share a gate)"""
    group = check_residual_norm(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias,
                                want_residual)
    here = _here(x)
    if here is None:
        with torch.cuda.device(x.device):
            return residual_norm_forward(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias,
                                         eps, want_residual, keep)
    lib = _lib or _load()
    xr, x_ld = _rows(x)
    yr, y_ld = _rows(y)
    gr, g_ld = (None, 0) if gate is None else _rows(gate)
    scale, inner_weight, inner_bias, outer_weight, outer_bias = [
        None if t is None else _flat(t) for t in (scale, inner_weight, inner_bias, outer_weight, outer_bias)]
    width = x.shape[-1]
    rows = x.numel() // width
    residual = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_residual else None
    normed = torch.empty(x.shape, dtype=x.dtype, device=x.device) if outer is not None else None
    stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if keep else None
    if lib.enc_residual_norm_forward(
            DTYPES[x.dtype], NORMS[inner], NORMS[outer], eps, xr.data_ptr(), x_ld, yr.data_ptr(), y_ld, _ptr(gr), g_ld, group,
            *[None if t is None else t.data_ptr() for t in (scale, inner_weight, inner_bias, outer_weight, outer_bias)],
            rows, width, _ptr(residual), _ptr(normed), _ptr(stats), _raw_stream(here)):
        _raise(lib, "residual_norm")
    return residual, normed, stats, group


def residual_norm_backward(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias, stats, group,
                           d_residual, d_normed, needs):
    """-> gradients of (x, y, gate, scale, inner_weight, inner_bias, outer_weight, outer_bias), None where `needs` says
    False.  Where y is added as it is, x and y have one gradient: the same tensor, as for x + y.  The other arguments are
    the forward call's, which checked them."""
    here = _here(x)
    if here is None:
        with torch.cuda.device(x.device):
            return residual_norm_backward(x, y, gate, scale, inner, inner_weight, inner_bias, outer, outer_weight, outer_bias,
                                          stats, group, d_residual, d_normed, needs)
    _check("residual_norm backward", x.device, x.dtype, ("d_residual", d_residual, x.shape), ("d_normed", d_normed, x.shape))
    lib = _lib or _load()
    xr, x_ld = _rows(x)
    yr, y_ld = _rows(y)
    gr, g_ld = (None, 0) if gate is None else _rows(gate)
    dr, dr_ld = (None, 0) if d_residual is None else _rows(d_residual)
    dn, dn_ld = (None, 0) if d_normed is None else _rows(d_normed)
    params = [None if t is None else _flat(t) for t in (scale, inner_weight, inner_bias, outer_weight)]
    width, dtype, device = x.shape[-1], x.dtype, x.device
    rows = x.numel() // width
    plain = gate is None and scale is None and inner is None
    new = [torch.empty(t.shape, dtype=dtype, device=device) if n and t is not None else None for t, n in zip(
        (x, y, gate, scale, inner_weight, inner_bias, outer_weight, outer_bias),
        (needs[0] or (plain and needs[1]), needs[1] and not plain, *needs[2:]))]
    nbytes = lib.enc_residual_norm_backward_workspace_bytes(rows, width, group)
    ws = _workspace(nbytes, device)
    if lib.enc_residual_norm_backward(
            DTYPES[dtype], NORMS[inner], NORMS[outer], xr.data_ptr(), x_ld, yr.data_ptr(), y_ld, _ptr(gr), g_ld, group,
            *[None if t is None else t.data_ptr() for t in params], stats.data_ptr(), _ptr(dr), dr_ld, _ptr(dn), dn_ld, rows,
            width, *[None if t is None else t.data_ptr() for t in new], _ptr(ws), nbytes, _raw_stream(here)):
        _raise(lib, "residual_norm backward")
    if plain and needs[1]:
        new[1] = new[0]
        if not needs[0]:
            new[0] = None
    return new


# ---- orthogonalised update --------------------------------------------------------------------
def check_orthogonalize(update, steps):
    what = "orthogonalize"
    if update.dtype not in DTYPES:
        raise RuntimeError("%s: not implemented for %s" % (what, update.dtype))
    if update.dim() < 2 or min(update.shape[-2:]) < 1:
        raise RuntimeError("%s: update must be [..., rows, cols] with at least one of each" % what)
    if not 1 <= steps <= 100:
        raise RuntimeError("%s: steps must be 1 to 100" % what)


def orthogonalize(update, steps, coefficients, eps):
    """-> a new tensor of update's shape and dtype"""
    check_orthogonalize(update, steps)
    here = _here(update)
    if here is None:
        with torch.cuda.device(update.device):
            return orthogonalize(update, steps, coefficients, eps)
    lib = _lib or _load()
    a, b, c = coefficients
    update = _flat(update)
    out = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    rows, cols = update.shape[-2:]
    batch = update.numel() // (rows * cols)
    code = DTYPES[update.dtype]
    nbytes = lib.enc_orthogonalize_workspace_bytes(code, batch, rows, cols)
    ws = _workspace(nbytes, update.device)
    if lib.enc_orthogonalize(code, update.data_ptr(), out.data_ptr(), batch, rows, cols, steps, a, b, c, eps, _ptr(ws), nbytes,
                             _raw_stream(here)):
        _raise(lib, "orthogonalize")
    return out
