"""Layer norm on the library's kernels: the normalisation in front of every block, behind the gate of the hybrid layer and
in front of the head (reference src/models/resnet_bk.py:243-244, src/models/phase7/hybrid_attention.py:55,143)."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _layer_ops as ops
from . import _lib

MAX_DIM = 16384   # BKCORE_LAYER_NORM_MAX_DIM


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of ``x`` over its last dimension (at most 16384 elements), in x's type; mean, centred variance and the
    gradients' sums in float32.  ``weight`` and ``bias``: (D,) in float32 or x's type, both of one type, or None."""
    what = "layer_norm"
    if x.dim() == 0:
        raise ValueError("bkcore: layer_norm needs at least one dimension")
    ops.need_device(x, weight, bias)
    ops.need_dtype(what, x)
    D = x.shape[-1]
    if not 1 <= D <= MAX_DIM:
        raise ValueError(f"bkcore: layer_norm normalises 1 to {MAX_DIM} elements, not {D}")
    for name, p in (("weight", weight), ("bias", bias)):
        ops.need_param(what, p, x)
        ops.need_shape(what, name, p, (D,))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("bkcore: layer_norm: weight and bias are of one type")
    if not eps >= 0.0:
        raise ValueError(f"bkcore: layer_norm: eps must not be negative, got {eps}")
    with ops.on_device(x.device):
        return _lib.load_native().layer_norm(x, weight, bias, float(eps), ops.wants_grad(x, weight, bias),
                                             ops.stream(x.device.index))


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension on the library's kernel (same parameters, same state_dict)."""

    def __init__(self, normalized_shape, *args, **kwargs):
        super().__init__(normalized_shape, *args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError("bkcore: LayerNorm normalises the last dimension only")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"bkcore: LayerNorm over {self.normalized_shape[0]} elements got {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps)
