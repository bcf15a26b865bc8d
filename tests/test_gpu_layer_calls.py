"""GPU tests of how the layer operators are called: derivatives of other kinds, broadcast gates, autocast, weights in 16 bits
with gradients out of their range, hooks; against the 64-bit forms of layer_reference.py where there are values to compare."""
import pytest
import torch

import layer_reference as R
from test_gpu_layer import FLOATS, ffn_inputs, gen, norm_inputs, rand

pytestmark = pytest.mark.gpu


def test_a_gradient_with_a_tangent_is_refused():
    """Forward over reverse: the kernels of the backward pass would drop it."""
    import torch.autograd.forward_ad as fwAD
    from instaorder_amd import gated_feed_forward, residual_norm
    args = [a.requires_grad_(True) for a in ffn_inputs(torch.float32, 5, 16, 8, 16, True)]
    for call in (lambda: gated_feed_forward(*args), lambda: residual_norm(args[0], args[0] * 2, outer="rms")[1]):
        y = call()
        with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, args[0], fwAD.make_dual(torch.ones_like(y), torch.ones_like(y)))
        dx, = torch.autograd.grad(call(), args[0], torch.ones_like(y))
        assert dx.isfinite().all()
