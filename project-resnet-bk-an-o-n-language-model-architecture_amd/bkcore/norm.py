"""Layer norm on the library's kernels: the normalisation in front of every block, behind the gate of the hybrid layer and
in front of the head (reference src/models/resnet_bk.py:243-244, src/models/phase7/hybrid_attention.py:55,143)."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _layer_ops as ops
from . import _lib

MAX_DIM = 16384   # BKCORE_LAYER_NORM_MAX_DIM


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        D = x.shape[-1]
        x2 = ops.inner(x if x.dim() == 2 else x.reshape(-1, D))
        rows = x2.shape[0]
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        dev = x.device
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        stats = torch.empty(2 * rows, dtype=torch.float32, device=dev) if keep else None
        p = w if w is not None else b if b is not None else x2
        with ops.on_device(dev):
            rc = _lib.load_held().bkcore_layer_norm(
                x2.data_ptr(), x2.stride(0), ops.DTYPES[x.dtype], ops.ptr(w), ops.ptr(b), ops.DTYPES[p.dtype], eps, rows, D,
                y.data_ptr(), ops.ptr(stats), ops.stream(dev.index))
        if rc:
            _lib.check(rc, "bkcore_layer_norm")
        if keep:
            ctx.save_for_backward(x2, w, stats)
            ctx.bk_bias = None if bias is None else bias.dtype
            ctx.bk_shape = x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        ops.once_only("layer_norm")
        x2, w, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        rows, D = x2.shape
        dev = x2.device
        g2 = ops.inner(dy if dy.dim() == 2 else dy.reshape(-1, D))
        dx = torch.empty(rows, D, dtype=x2.dtype, device=dev)
        L = _lib.load_held()
        gp = ws = None
        nbytes = 0
        if need_w or need_b:
            nbytes = L.bkcore_layer_norm_backward_workspace_bytes(rows, D)
            gp = torch.empty(2 * D, dtype=torch.float32, device=dev)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            if rows == 0:
                gp.zero_()
        with ops.on_device(dev):
            rc = L.bkcore_layer_norm_backward(
                g2.data_ptr(), g2.stride(0), x2.data_ptr(), x2.stride(0), ops.DTYPES[x2.dtype], ops.ptr(w),
                ops.DTYPES[(x2 if w is None else w).dtype], stats.data_ptr(), rows, D, dx.data_ptr(), ops.ptr(gp), ops.ptr(ws), nbytes,
                ops.stream(dev.index))
        if rc:
            _lib.check(rc, "bkcore_layer_norm_backward")
        return (dx.view(ctx.bk_shape) if need_x else None, gp[:D].to(w.dtype) if need_w else None,
                gp[D:].to(ctx.bk_bias) if need_b else None, None, None)


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
