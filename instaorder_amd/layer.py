"""Operators of an encoder layer around its attention op, on the kernels of libenc_hip.so (layer_ext.py):

    gated_feed_forward(x, w_in, b_in, w_out, b_out, activation)

GPU tensors always take the HIP kernels (errors propagate); CPU tensors take an elementary PyTorch path by explicit
device dispatch, as ``MSDeformAttn`` does."""
import torch
import torch.nn.functional as F
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import layer_ext

_ACT = {"silu": F.silu, "gelu": F.gelu, "sigmoid": torch.sigmoid, "relu": F.relu}


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class GatedFeedForwardFunction(Function):
    """Saves x, the two weights and the pre-activations in fp32 (8 bytes a hidden value, what a 16-bit eager block
    keeps in four tensors), so that the gradients are formed from unrounded values."""

    @staticmethod
    def forward(ctx, x, w_in, b_in, w_out, b_out, activation):
        y, pre = layer_ext.gated_ffn_forward(x, w_in, b_in, w_out, b_out, activation, True)
        ctx.activation = activation
        ctx.save_for_backward(x, w_in, w_out, pre)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, w_in, w_out, pre = ctx.saved_tensors
        return (*layer_ext.gated_ffn_backward(x, w_in, w_out, pre, grad, ctx.activation, ctx.needs_input_grad[:5]), None)


def gated_feed_forward(x, w_in, b_in, w_out, b_out, activation="silu"):
    """y = (a * act(b)) W_out^T + b_out with [a | b] = x W_in^T + b_in.

    x [..., width]; w_in [2 * hidden, width] (value rows first, then gate rows -- the order of ``F.glu``); w_out
    [out_width, hidden]; biases may be None.  activation: "silu", "gelu" (by the error function), "sigmoid", "relu".
    fp32, bf16 or fp16, one type for all; sums are fp32, h is rounded to the type once.  Differentiable once in all five
    tensors.  fp32: an Inf among the inputs gives NaN (its parts multiply zeros), a NaN stays one."""
    if not x.is_cuda:
        layer_ext.check_gated_ffn(x, w_in, b_in, w_out, b_out, activation)
        a, b = F.linear(x, w_in, b_in).chunk(2, -1)
        return F.linear(a * _ACT[activation](b), w_out, b_out)
    if _wants_grad(x, w_in, b_in, w_out, b_out):
        return GatedFeedForwardFunction.apply(x, w_in, b_in, w_out, b_out, activation)
    return layer_ext.gated_ffn_forward(x, w_in, b_in, w_out, b_out, activation, False)[0]
