"""The operators of a selective mixer: the short causal convolution and the selective state space scan, for prompts, for
training and for single tokens.  They stand beside ``fused_associative_scan``, the plain accumulation of the reference's
global path (src/models/phase1/ar_ssm_layer.py:517-525): here the decay and what enters the state depend on the input.

Channels are innermost: (B, L, C).  Positions at or behind ``lengths`` (B,) are padding of a right-padded batch: their
values do not matter, outputs and gradients there are zero, and a returned state is the one behind the last position inside."""
from __future__ import annotations

import torch

from . import _layer_ops as ops
from . import _lib

MAX_STATE = 64    # BKCORE_SCAN_MAX_STATE


def _activation(what: str, activation) -> int:
    if activation not in (None, "silu"):
        raise ValueError(f"bkcore: {what}: activation is None or 'silu', not {activation!r}")
    return int(activation == "silu")


def _conv_params(what, x, weight, bias):
    C = x.shape[-1]
    ops.need_device(x, weight, bias)
    ops.need_dtype(what, x)
    if weight.dim() != 2 or weight.shape[0] != C or not 2 <= weight.shape[1] <= 4:
        raise ValueError(f"bkcore: {what}: weight is ({C}, 2 to 4), got {tuple(weight.shape)}")
    ops.need_shape(what, "bias", bias, (C,))
    ops.need_param(what, weight, x)
    if bias is not None and bias.dtype != weight.dtype:
        raise TypeError(f"bkcore: {what}: weight and bias are of one type")
    return weight.shape[1]


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
                lengths: torch.Tensor | None = None, initial_state: torch.Tensor | None = None,
                return_state: bool = False):
    """Depthwise causal convolution ``y_t = act(bias + sum_k weight[:, k] x_{t-K+1+k})`` of x (B, L, C) with weight (C, K),
    K from 2 to 4; ``activation`` None or "silu".  ``initial_state`` (B, K-1, C): the inputs in front of the first
    position (zeros otherwise).  ``return_state``: also the last K-1 inputs of each sequence, to go on from."""
    what = "causal_conv"
    if x.dim() != 3:
        raise ValueError(f"bkcore: {what}: x is (B, L, C), got {tuple(x.shape)}")
    B, T, C = x.shape
    K = _conv_params(what, x, weight, bias)
    ops.need_device(x, initial_state)
    ops.need_dtype(what, x, initial_state)
    ops.need_shape(what, "initial_state", initial_state, (B, K - 1, C))
    silu = _activation(what, activation)
    n = ops.lengths_arg(what, lengths, x, B, T)
    keep = ops.wants_grad(x, weight, bias, initial_state)
    with ops.on_device(x.device):
        out = _lib.load_native().causal_conv(x, weight, bias, initial_state, n, silu, keep, bool(return_state),
                                             ops.stream(x.device.index))
    return tuple(out) if return_state else out[0]


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                     activation: str | None = None) -> torch.Tensor:
    """``causal_conv`` for one token of each sequence: x (B, C); ``state`` (B, K-1, C) contiguous, the last K-1 inputs, is
    moved on in place.  No gradient."""
    what = "causal_conv_step"
    if x.dim() != 2:
        raise ValueError(f"bkcore: {what}: x is (B, C), got {tuple(x.shape)}")
    K = _conv_params(what, x, weight, bias)
    B, C = x.shape
    ops.need_device(x, state)
    ops.need_state(what, "state", state, x, (B, K - 1, C), x.dtype)
    if not state.is_contiguous():
        raise ValueError(f"bkcore: {what}: state must be contiguous")
    silu = _activation(what, activation)
    ops.no_grad_through(what, x, weight, bias)
    with ops.on_device(x.device):
        return _lib.load_native().causal_conv_step(x, state, weight, bias, silu, ops.stream(x.device.index))


def _scan_params(what, x, A, D, delta_bias):
    """A (C, N) and the optional (C,) vectors, contiguous float32 (a cast is differentiable where they are trained)."""
    C = x.shape[-1]
    ops.need_device(x, A, D, delta_bias)
    if A.dim() != 2 or A.shape[0] != C or not 1 <= A.shape[1] <= MAX_STATE:
        raise ValueError(f"bkcore: {what}: A is ({C}, 1 to {MAX_STATE}), got {tuple(A.shape)}")
    out = []
    for name, p, shape in (("A", A, tuple(A.shape)), ("D", D, (C,)), ("delta_bias", delta_bias, (C,))):
        ops.need_shape(what, name, p, shape)
        ops.need_param(what, p, x)
        out.append(None if p is None else p.float())
    return out


def selective_scan(x: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: torch.Tensor | None = None, z: torch.Tensor | None = None, delta_bias: torch.Tensor | None = None,
                   delta_softplus: bool = False, lengths: torch.Tensor | None = None,
                   initial_state: torch.Tensor | None = None, return_state: bool = False):
    """The selective scan ``h_t = exp(d_t A) h_{t-1} + d_t x_t B_t``, ``y_t = (C_t . h_t + D x_t) silu(z_t)`` with
    ``d = delta + delta_bias``, through softplus if ``delta_softplus``.

    x, delta, z (B, L, C) and B, C (B, L, N), N <= 64, in one type; A (C, N), D and delta_bias (C,) in float32 or that
    type.  The state (B, C, N) is float32: ``initial_state`` to start from (zeros otherwise), ``return_state`` to get the
    one behind the last position.  All tensors get gradients, the states too."""
    what = "selective_scan"
    if x.dim() != 3:
        raise ValueError(f"bkcore: {what}: x is (B, L, C), got {tuple(x.shape)}")
    b, t, c = x.shape
    ops.need_device(x, delta, B, C, z, initial_state)
    ops.need_dtype(what, x, delta, B, C, z)
    A, D, delta_bias = _scan_params(what, x, A, D, delta_bias)
    n = A.shape[1]
    for name, m, shape in (("delta", delta, (b, t, c)), ("z", z, (b, t, c)), ("B", B, (b, t, n)), ("C", C, (b, t, n)),
                           ("initial_state", initial_state, (b, c, n))):
        ops.need_shape(what, name, m, shape)
    if initial_state is not None and initial_state.dtype != torch.float32:
        raise TypeError(f"bkcore: {what}: the state is float32, not {initial_state.dtype}")
    ln = ops.lengths_arg(what, lengths, x, b, t)
    keep = ops.wants_grad(x, delta, A, B, C, D, z, delta_bias, initial_state)
    with ops.on_device(x.device):
        out = _lib.load_native().selective_scan(x, delta, A, B, C, D, z, delta_bias, initial_state, ln,
                                                int(bool(delta_softplus)), keep, bool(return_state),
                                                ops.stream(x.device.index))
    return tuple(out) if return_state else out[0]


def selective_scan_step(x: torch.Tensor, state: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, D: torch.Tensor | None = None, z: torch.Tensor | None = None,
                        delta_bias: torch.Tensor | None = None, delta_softplus: bool = False) -> torch.Tensor:
    """``selective_scan`` for one token of each sequence: x, delta, z (B, C), B and C (B, N); ``state`` (B, C, N) float32,
    contiguous, is updated in place.  No gradient."""
    what = "selective_scan_step"
    if x.dim() != 2:
        raise ValueError(f"bkcore: {what}: x is (B, C), got {tuple(x.shape)}")
    b, c = x.shape
    ops.need_device(x, delta, B, C, z, state)
    ops.need_dtype(what, x, delta, B, C, z)
    ops.no_grad_through(what, x, delta, A, B, C, D, z, delta_bias)
    A, D, delta_bias = _scan_params(what, x, A, D, delta_bias)
    n = A.shape[1]
    for name, m, shape in (("delta", delta, (b, c)), ("z", z, (b, c)), ("B", B, (b, n)), ("C", C, (b, n))):
        ops.need_shape(what, name, m, shape)
    ops.need_state(what, "state", state, x, (b, c, n), torch.float32)
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError(f"bkcore: {what}: state must be contiguous and 16-byte aligned")
    with ops.on_device(x.device):
        return _lib.load_native().selective_scan_step(x, state, delta, A, B, C, D, z, delta_bias, int(bool(delta_softplus)),
                                                      ops.stream(x.device.index))
