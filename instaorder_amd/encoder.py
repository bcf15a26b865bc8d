"""The MSDA encoder stack of Mask2Former's pixel decoder, without detectron2 -- the immediate
caller of the op.  Mirrors, with the same sub-module names (so
state-dict keys match), the reference's

  MSDeformAttnTransformerEncoderOnly / ...EncoderLayer / ...Encoder
      mask2former/modeling/pixel_decoder/msdeformattn.py:23-254
  PositionEmbeddingSine
      mask2former/modeling/transformer_decoder/position_encoding.py:12-56

Levels are passed LOW-RES FIRST, as MSDeformAttnPixelDecoder does (msdeformattn.py:440).
Parity: pinned.  MSDeformAttn by tests/golden/module_msdeformattn.npz; the stack by
tests/golden/encoder_{small,heads8,six_layers}.npz and position_encoding.npz -- outputs and input gradients of the
REFERENCE's own classes, which tests/golden/make_golden.py imports with name-only placeholders for the detectron2
symbols their module merely imports (nothing the encoder classes execute comes from a placeholder)."""
import copy
import math

import torch
import torch.nn.functional as F
from torch import nn
from torch.nn.init import normal_
from torch.nn.modules.module import _has_any_global_hook

from . import layer_ext
from .layer import ACTIVATIONS, autocast_dtype, gated_feed_forward, residual_norm
from .modules import MSDeformAttn


class PositionEmbeddingSine(nn.Module):
    def __init__(self, num_pos_feats=64, temperature=10000, normalize=False, scale=None):
        super().__init__()
        if scale is not None and normalize is False:
            raise ValueError("normalize should be True if scale is passed")
        self.num_pos_feats, self.temperature, self.normalize = num_pos_feats, temperature, normalize
        self.scale = 2 * math.pi if scale is None else scale

    def forward(self, x, mask=None):
        if mask is None:
            mask = torch.zeros((x.size(0), x.size(2), x.size(3)), device=x.device, dtype=torch.bool)
        keep = ~mask
        y_embed = keep.cumsum(1, dtype=torch.float32)
        x_embed = keep.cumsum(2, dtype=torch.float32)
        if self.normalize:
            eps = 1e-6
            y_embed = y_embed / (y_embed[:, -1:, :] + eps) * self.scale
            x_embed = x_embed / (x_embed[:, :, -1:] + eps) * self.scale
        dim_t = torch.arange(self.num_pos_feats, dtype=torch.float32, device=x.device)
        dim_t = self.temperature ** (2 * (dim_t // 2) / self.num_pos_feats)
        pos_x = x_embed[:, :, :, None] / dim_t
        pos_y = y_embed[:, :, :, None] / dim_t
        pos_x = torch.stack((pos_x[..., 0::2].sin(), pos_x[..., 1::2].cos()), dim=4).flatten(3)
        pos_y = torch.stack((pos_y[..., 0::2].sin(), pos_y[..., 1::2].cos()), dim=4).flatten(3)
        return torch.cat((pos_y, pos_x), dim=3).permute(0, 3, 1, 2)


# Activations of the feed-forward block that take a value and a gate: linear1 is twice as wide, its first half the value
# (the order of F.glu).  In the reference "glu" halves the hidden width under linear2 and cannot run; here it does.
GATED = {"glu": "sigmoid", "swiglu": "silu", "geglu": "gelu", "reglu": "relu"}


def _activation(name):
    return {"relu": F.relu, "gelu": F.gelu, **{k: ACTIVATIONS[v] for k, v in GATED.items()}}[name]


def _as_made(module, kind):
    """Does calling `module` do what `kind` does and nothing else?  Not for a subclass or a wrapper (an adapter, a
    parametrisation), a forward of its own, or one with hooks: those have to be called.  Nor under torch.jit.trace, which
    records torch's own operators and refuses the kernels."""
    return (type(module) is kind and "forward" not in module.__dict__ and not torch.jit.is_tracing()
            and not (module._forward_pre_hooks or module._forward_hooks or module._backward_pre_hooks
                     or module._backward_hooks or _has_any_global_hook()))


class MSDeformAttnTransformerEncoderLayer(nn.Module):
    gate, fused_norm = None, False      # of a layer that was pickled whole before it had them

    def __init__(self, d_model=256, d_ffn=1024, dropout=0.1, activation="relu", n_levels=4,
                 n_heads=8, n_points=4, use_adapters=False, adapter_dim=64, adapter_scale=0.1):
        super().__init__()
        self.self_attn = MSDeformAttn(d_model, n_levels, n_heads, n_points)
        self.dropout1 = nn.Dropout(dropout)
        self.norm1 = nn.LayerNorm(d_model)
        self.gate = GATED.get(activation)           # name of the gate's activation, None for a plain block
        self.linear1 = nn.Linear(d_model, 2 * d_ffn if self.gate else d_ffn)
        self.activation = _activation(activation)
        self.dropout2 = nn.Dropout(dropout)
        self.linear2 = nn.Linear(d_ffn, d_model)
        self.dropout3 = nn.Dropout(dropout)
        self.norm2 = nn.LayerNorm(d_model)
        # opt-in (not reference behaviour): src + block and its norm in one kernel (residual_norm).  Like the gated block's
        # kernels it takes the place of submodules that are as they were made; others (hooks, wrappers) are called.
        self.fused_norm = False
        self.use_adapters, self.adapter_scale = use_adapters, adapter_scale
        if use_adapters:        # InstaFormer's trainable adapters (msdeformattn.py:155-166)
            self.adapter = nn.Sequential(nn.Linear(d_model, adapter_dim), nn.ReLU(),
                                         nn.Linear(adapter_dim, d_model))
            nn.init.kaiming_normal_(self.adapter[0].weight)
            nn.init.zeros_(self.adapter[0].bias)
            nn.init.zeros_(self.adapter[2].weight)
            nn.init.zeros_(self.adapter[2].bias)

    @staticmethod
    def _one_type(*tensors):
        """Of one type that the layer operators take, or of any of them under autocast, which they follow."""
        return (all(t.dtype in layer_ext.DTYPES for t in tensors)
                and (len({t.dtype for t in tensors}) == 1 or autocast_dtype(tensors[0]) is not None))

    def _add_and_norm(self, src, block, norm):
        if (self.fused_norm and src.is_cuda and _as_made(norm, nn.LayerNorm) and norm.normalized_shape == src.shape[-1:]
                and self._one_type(src, block, *([] if norm.weight is None else [norm.weight]))
                and src.shape[-1] <= layer_ext.NORM_MAX_WIDTH):
            return residual_norm(src, block, outer="layer", outer_weight=norm.weight, outer_bias=norm.bias, eps=norm.eps,
                                 want_residual=False)[1]
        return norm(src + block)

    def _feed_forward(self, src):
        if not self.gate:
            return self.linear2(self.dropout2(self.activation(self.linear1(src))))
        made = (_as_made(self.linear1, nn.Linear) and _as_made(self.linear2, nn.Linear) and _as_made(self.dropout2, nn.Dropout)
                and self.activation is ACTIVATIONS[self.gate])
        dropping = self.dropout2.training and self.dropout2.p > 0        # dropout of h: inside the block, not in the kernels
        if not made or dropping or not self._one_type(src, self.linear1.weight):
            value, gate = self.linear1(src).chunk(2, -1)
            return self.linear2(self.dropout2(value * self.activation(gate)))
        return gated_feed_forward(src, self.linear1.weight, self.linear1.bias, self.linear2.weight, self.linear2.bias,
                                  self.gate)

    def forward(self, src, pos, reference_points, spatial_shapes, level_start_index, padding_mask=None):
        query = src if pos is None else src + pos
        src = self._add_and_norm(src, self.dropout1(self.self_attn(
            query, reference_points, src, spatial_shapes, level_start_index, padding_mask)), self.norm1)
        side = self.adapter(src) if self.use_adapters else None
        src = self._add_and_norm(src, self.dropout3(self._feed_forward(src)), self.norm2)
        if side is not None:
            src = src + self.adapter_scale * side
        return src


class MSDeformAttnTransformerEncoder(nn.Module):
    def __init__(self, encoder_layer, num_layers):
        super().__init__()
        self.layers = nn.ModuleList([copy.deepcopy(encoder_layer) for _ in range(num_layers)])
        self.num_layers = num_layers

    @staticmethod
    def get_reference_points(spatial_shapes, valid_ratios, device):
        """Pixel centres of every level, normalised by the valid extent, then expressed in every
        level's frame: [N, S, L, 2] (msdeformattn.py:215-229)."""
        refs = []
        for lvl, (h, w) in enumerate(spatial_shapes):
            h, w = int(h), int(w)
            ys, xs = torch.meshgrid(
                torch.linspace(0.5, h - 0.5, h, dtype=torch.float32, device=device),
                torch.linspace(0.5, w - 0.5, w, dtype=torch.float32, device=device), indexing="ij")
            ys = ys.reshape(-1)[None] / (valid_ratios[:, None, lvl, 1] * h)
            xs = xs.reshape(-1)[None] / (valid_ratios[:, None, lvl, 0] * w)
            refs.append(torch.stack((xs, ys), -1))
        return torch.cat(refs, 1)[:, :, None] * valid_ratios[:, None]

    def forward(self, src, spatial_shapes, level_start_index, valid_ratios, pos=None, padding_mask=None):
        reference_points = self.get_reference_points(spatial_shapes, valid_ratios, device=src.device)
        for layer in self.layers:
            src = layer(src, pos, reference_points, spatial_shapes, level_start_index, padding_mask)
        return src


class MSDeformAttnTransformerEncoderOnly(nn.Module):
    def __init__(self, d_model=256, nhead=8, num_encoder_layers=6, dim_feedforward=1024, dropout=0.1,
                 activation="relu", num_feature_levels=4, enc_n_points=4, use_adapters=False,
                 adapter_dim=64, adapter_scale=0.1):
        super().__init__()
        self.d_model, self.nhead = d_model, nhead
        layer = MSDeformAttnTransformerEncoderLayer(d_model, dim_feedforward, dropout, activation,
                                                    num_feature_levels, nhead, enc_n_points,
                                                    use_adapters, adapter_dim, adapter_scale)
        self.encoder = MSDeformAttnTransformerEncoder(layer, num_encoder_layers)
        self.level_embed = nn.Parameter(torch.Tensor(num_feature_levels, d_model))
        self._reset_parameters()

    def _reset_parameters(self):
        for p in self.parameters():
            if p.dim() > 1:
                nn.init.xavier_uniform_(p)
        for mod in self.modules():
            if isinstance(mod, MSDeformAttn):
                mod._reset_parameters()
        normal_(self.level_embed)

    @staticmethod
    def get_valid_ratio(mask):
        _, h, w = mask.shape
        valid_h = torch.sum(~mask[:, :, 0], 1).float() / h
        valid_w = torch.sum(~mask[:, 0, :], 1).float() / w
        return torch.stack([valid_w, valid_h], -1)

    def forward(self, srcs, pos_embeds):
        """srcs / pos_embeds: per level [N, C, H_l, W_l].  Returns (memory [N,S,C],
        spatial_shapes [L,2], level_start_index [L])  (msdeformattn.py:79-123)."""
        masks = [torch.zeros((x.size(0), x.size(2), x.size(3)), device=x.device, dtype=torch.bool)
                 for x in srcs]
        flat, flat_mask, flat_pos, shapes = [], [], [], []
        for lvl, (src, mask, pos) in enumerate(zip(srcs, masks, pos_embeds)):
            shapes.append(tuple(src.shape[2:]))
            flat.append(src.flatten(2).transpose(1, 2))
            flat_mask.append(mask.flatten(1))
            flat_pos.append(pos.flatten(2).transpose(1, 2) + self.level_embed[lvl].view(1, 1, -1))
        flat, flat_mask, flat_pos = torch.cat(flat, 1), torch.cat(flat_mask, 1), torch.cat(flat_pos, 1)
        spatial_shapes = torch.as_tensor(shapes, dtype=torch.long, device=flat.device)
        level_start_index = torch.cat((spatial_shapes.new_zeros((1,)),
                                       spatial_shapes.prod(1).cumsum(0)[:-1]))
        valid_ratios = torch.stack([self.get_valid_ratio(m) for m in masks], 1)
        memory = self.encoder(flat, spatial_shapes, level_start_index, valid_ratios, flat_pos, flat_mask)
        return memory, spatial_shapes, level_start_index
