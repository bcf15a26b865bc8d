"""Host side of libenc_hip.so (include/enc_hip.h): the operators of an encoder layer around its attention op.  Checks,
allocation and the current stream are here, as ``ext.py`` has them for the attention op: outputs are new tensors on the
inputs' device, kernels are enqueued on torch's current HIP stream without synchronising, every error is a RuntimeError,
and there is no fallback -- a missing library, a CPU tensor or a failed launch raises.

Nothing is kept between calls: workspaces come from torch's caching allocator, so calls on several streams, and captured
graphs with their own memory pools, share none."""
import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "libenc_hip.so")
_lib = None

_I, _L, _Z, _P, _F = ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_float

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
            ("enc_gated_ffn_forward", [_I, _I, _P, _L] + [_P] * 4 + [_L] * 4 + [_P] * 3 + [_Z, _P], _I),
            ("enc_gated_ffn_backward", [_I, _I, _P, _L] + [_P] * 4 + [_L] * 5 + [_P] * 6 + [_Z, _P], _I)):
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


def _same(what, device, dtype, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise RuntimeError("%s: %s is on %s, not on %s" % (what, name, t.device, device))
        if t.dtype != dtype:
            raise RuntimeError("%s: %s has dtype %s, not %s" % (what, name, t.dtype, dtype))


def _shaped(what, **shapes):
    for name, (t, want) in shapes.items():
        if t is not None and tuple(t.shape) != want:
            raise RuntimeError("%s: %s has shape %s, not %s" % (what, name, tuple(t.shape), want))


def _rows(t):
    """(a 2-D view or copy of t with contiguous rows, elements from one row to the next)"""
    t = t.reshape(-1, t.shape[-1])
    if t.shape[0] <= 1:
        t = t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()
        return t, t.shape[1]
    if (t.stride(1) != 1 and t.shape[1] != 1) or t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, t.stride(0)


class _On:
    """The device of a call made current for its duration (launches and allocations go there), and its stream."""
    __slots__ = ("device", "guard")

    def __init__(self, device):
        self.device = device
        self.guard = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


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
    _same(what, x.device, x.dtype, w_in=w_in, b_in=b_in, w_out=w_out, b_out=b_out)
    _shaped(what, w_in=(w_in, (2 * hidden, width)), b_in=(b_in, (2 * hidden,)), w_out=(w_out, (out_width, hidden)),
            b_out=(b_out, (out_width,)))
    return hidden, out_width


def gated_ffn_forward(x, w_in, b_in, w_out, b_out, activation, keep):
    """-> (y [..., out_width], pre); pre: what the backward pass takes, or None unless `keep`."""
    hidden, out_width = check_gated_ffn(x, w_in, b_in, w_out, b_out, activation)
    if not x.is_cuda:
        raise RuntimeError("Not implemented on the CPU")
    lib = _load()
    with _On(x.device) as stream:
        rows, stride = _rows(x)
        w_in, w_out = w_in.contiguous(), w_out.contiguous()
        b_in, b_out = (None if b is None else b.contiguous() for b in (b_in, b_out))
        tokens, width = rows.shape
        code = DTYPES[x.dtype]
        y = torch.empty((*x.shape[:-1], out_width), dtype=x.dtype, device=x.device)
        pre = torch.empty((tokens, 2 * ((hidden + 7) // 8 * 8)), dtype=torch.float32, device=x.device) if keep else None
        nbytes = lib.enc_gated_ffn_forward_workspace_bytes(code, tokens, width, hidden, out_width)
        ws = _workspace(nbytes, x.device)
        rc = lib.enc_gated_ffn_forward(code, ACTIVATIONS[activation], rows.data_ptr(), stride, w_in.data_ptr(), _ptr(b_in),
                                       w_out.data_ptr(), _ptr(b_out), tokens, width, hidden, out_width, y.data_ptr(),
                                       _ptr(pre), _ptr(ws), nbytes, stream)
    if rc != 0:
        _raise(lib, "gated_feed_forward")
    return y, pre


def gated_ffn_backward(x, w_in, w_out, pre, grad, activation, needs):
    """-> (d_x, d_w_in, d_b_in, d_w_out, d_b_out), None where `needs` says False."""
    hidden, out_width = check_gated_ffn(x, w_in, None, w_out, None, activation)
    lib = _load()
    _same("gated_feed_forward backward", x.device, x.dtype, grad=grad)
    with _On(x.device) as stream:
        rows, stride = _rows(x)
        g, g_stride = _rows(grad)
        w_in, w_out = w_in.contiguous(), w_out.contiguous()
        tokens, width = rows.shape
        code = DTYPES[x.dtype]
        shapes = (tuple(x.shape), (2 * hidden, width), (2 * hidden,), (out_width, hidden), (out_width,))
        outs = [torch.empty(s, dtype=x.dtype, device=x.device) if n else None for s, n in zip(shapes, needs)]
        nbytes = lib.enc_gated_ffn_backward_workspace_bytes(code, tokens, width, hidden, out_width)
        ws = _workspace(nbytes, x.device)
        rc = lib.enc_gated_ffn_backward(code, ACTIVATIONS[activation], rows.data_ptr(), stride, w_in.data_ptr(),
                                        w_out.data_ptr(), pre.data_ptr(), g.data_ptr(), g_stride, tokens, width, hidden,
                                        out_width, *[_ptr(t) for t in outs], _ptr(ws), nbytes, stream)
    if rc != 0:
        _raise(lib, "gated_feed_forward backward")
    return outs
