"""instaorder_amd -- MI355X-native multi-scale deformable attention (MSDA), the one native
hot path of SNU-VGILab/InstaOrder (Mask2Former's MSDeformAttnPixelDecoder encoder).

  csrc/msda_hip.hip   host side + the C ABI (include/msda_hip.h); kernels in csrc/msda_*.inc (gfx950 HIP)
  ext.py              host side of the extension boundary (checks, allocation, stream)
  functions.py        MSDeformAttnFunction (autograd wrapper) + the CPU-tensor PyTorch path
  modules.py          MSDeformAttn (the nn.Module that calls the op)
  encoder.py          the pixel decoder's MSDA encoder stack, detectron2-free
  pixel_decoder.py    MSDeformAttnPixelDecoder around it (input projections, FPN, mask features)
  layer_ext.py        host side of libenc_hip.so (include/enc_hip.h): operators of the layer around the op
  layer.py            gated_feed_forward, residual_norm: entry points and CPU paths
  layer_checks.py     their arguments' checks on the CPU
  optim.py            orthogonalize and the Muon optimiser for the stack's weight matrices
  synthetic.py        synthetic inputs of the encoder's shape (bench, tests)
"""
from .functions import MSDeformAttnFunction, ms_deform_attn_core_pytorch
from .layer import gated_feed_forward, residual_norm
from .modules import MSDeformAttn
from .optim import Muon, orthogonalize

__all__ = ["MSDeformAttnFunction", "MSDeformAttn", "ms_deform_attn_core_pytorch",
           "gated_feed_forward", "residual_norm",
           "Muon", "orthogonalize"]
