"""Host side of libenc_hip.so (include/enc_hip.h), the operators of an encoder layer around its attention op, is the compiled
binding ``_enc_bind`` (csrc/enc_bind.cpp): checks, allocation and torch's current stream, as ``ext.py`` has them for the
attention op -- outputs are new tensors on the inputs' device, kernels are enqueued without synchronising, every error is a
RuntimeError, and there is no fallback: a missing library, a CPU tensor or a failed launch raises.

Nothing is kept between calls: workspaces come from torch's caching allocator, so calls on several streams, and captured
graphs with their own memory pools, share none."""
import importlib
import os

import torch

_bind = None

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
NORM_MAX_WIDTH = 16384          # ENC_NORM_MAX_WIDTH of the header


def bind():
    """The compiled binding (loaded after torch, so that all share one HIP runtime)."""
    global _bind
    if _bind is None:
        here = os.path.dirname(os.path.abspath(__file__))
        if not all(os.path.exists(os.path.join(here, f)) for f in ("libenc_hip.so", "_enc_bind.so")):
            raise RuntimeError("libenc_hip.so and its binding are not built: run `python -m instaorder_amd.build_ext` "
                               "(needs hipcc); there is no fallback implementation")
        _bind = importlib.import_module("._enc_bind", __package__)
    return _bind


def launch_count():
    """Kernel launches issued through the library so far (proof the HIP path ran)."""
    return int(bind().launch_count())
