"""Layer norm on the library's kernels: the normalisation in front of every block, behind the gate of the hybrid layer and
in front of the head (reference src/models/resnet_bk.py:243-244, src/models/phase7/hybrid_attention.py:55,143)."""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _layer_ops as ops
from . import _lib

MAX_DIM = 16384   # BKCORE_LAYER_NORM_MAX_DIM


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        L = _lib.load()
        D = x.shape[-1]
        x2 = ops.inner(x.reshape(-1, D))
        rows = x2.shape[0]
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty(2, rows, dtype=torch.float32, device=x.device) if keep else None
        param = ops.DTYPES[(w if w is not None else b if b is not None else x2).dtype]
        with torch.cuda.device(x.device):
            rc = L.bkcore_layer_norm(ops.ptr(x2), x2.stride(0), ops.DTYPES[x.dtype], ops.ptr(w), ops.ptr(b), param, eps,
                                     rows, D, ops.ptr(y), ops.ptr(stats), ops.stream())
        _lib.check(rc, "bkcore_layer_norm")
        if keep:
            ctx.save_for_backward(x2, w, stats)
            ctx.bk_bias = None if bias is None else bias.dtype
            ctx.bk_shape = x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        L = _lib.load()
        x2, w, stats = ctx.saved_tensors
        rows, D = x2.shape
        want = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        g2 = ops.inner(dy.reshape(-1, D))
        dx = torch.empty(rows, D, dtype=x2.dtype, device=x2.device)
        gp = torch.empty(2, D, dtype=torch.float32, device=x2.device) if want else None
        if want and rows == 0:
            gp.zero_()
        with torch.cuda.device(x2.device):
            nbytes = int(L.bkcore_layer_norm_backward_workspace_bytes(rows, D)) if want else 0
            ws = ops.scratch(nbytes, x2.device)
            rc = L.bkcore_layer_norm_backward(ops.ptr(g2), g2.stride(0), ops.ptr(x2), x2.stride(0), ops.DTYPES[x2.dtype],
                                              ops.ptr(w), ops.DTYPES[(x2 if w is None else w).dtype], ops.ptr(stats), rows,
                                              D, ops.ptr(dx), ops.ptr(gp), ops.ptr(ws), nbytes, ops.stream())
        _lib.check(rc, "bkcore_layer_norm_backward")
        dw = gp[0].to(w.dtype) if ctx.needs_input_grad[1] else None
        db = gp[1].to(ctx.bk_bias) if ctx.needs_input_grad[2] else None
        return dx.reshape(ctx.bk_shape) if ctx.needs_input_grad[0] else None, dw, db, None, None


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
    return _LayerNormFunction.apply(x, weight, bias, float(eps), ops.wants_grad(x, weight, bias))


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
