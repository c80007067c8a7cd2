"""The operators of a selective mixer: the short causal convolution and the selective state space scan, for prompts, for
training and for single tokens.  They stand beside ``fused_associative_scan``, the plain accumulation of the reference's
global path (src/models/phase1/ar_ssm_layer.py:517-525): here the decay and what enters the state depend on the input.

Channels are innermost: (B, L, C).  Positions at or behind ``lengths`` (B,) are padding of a right-padded batch: they are
never read, outputs and gradients there are zero, and a returned state is the one behind the last position inside."""
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


class _CausalConvFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, keep, want_state):
        x = ops.inner(x)
        w = weight.contiguous()
        b = None if bias is None else bias.contiguous()
        st = None if state is None else state.contiguous()
        B, T, C = x.shape
        K = w.shape[1]
        dev = x.device
        y = torch.empty(B, T, C, dtype=x.dtype, device=dev)
        final = torch.empty(B, K - 1, C, dtype=x.dtype, device=dev) if want_state else None
        with ops.on_device(dev):
            rc = _lib.load_held().bkcore_causal_conv(
                x.data_ptr(), *ops.strides(x), ops.DTYPES[x.dtype], w.data_ptr(), ops.ptr(b), ops.DTYPES[w.dtype],
                ops.ptr(st), ops.ptr(lengths), B, T, C, K, silu, y.data_ptr(), ops.ptr(final), ops.stream(dev.index))
        if rc:
            _lib.check(rc, "bkcore_causal_conv")
        if keep:
            ctx.save_for_backward(x, w, b, st, lengths)
            ctx.bk_silu = silu
            ctx.set_materialize_grads(False)
        return (y, final) if want_state else y

    @staticmethod
    def backward(ctx, dy, dfinal=None):
        ops.once_only("causal_conv")
        x, w, b, st, lengths = ctx.saved_tensors
        need_x, need_w, need_b, need_st = ctx.needs_input_grad[:4]
        B, T, C = x.shape
        K = w.shape[1]
        dev = x.device
        dy = torch.zeros(B, T, C, dtype=x.dtype, device=dev) if dy is None else ops.inner(dy)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx = torch.empty(B, T, C, dtype=x.dtype, device=dev)
        dst = torch.empty_like(st) if st is not None and need_st else None
        L = _lib.load_held()
        gp = ws = None
        nbytes = 0
        if need_w or need_b:
            gp = torch.empty(C * (K + 1), dtype=torch.float32, device=dev)
            nbytes = L.bkcore_causal_conv_backward_workspace_bytes(B, T, C, K)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        if B == 0 or T == 0 or C == 0:       # nothing runs: no position, and the state passes through unchanged
            if gp is not None:
                gp.zero_()
            if dst is not None:
                dst.zero_() if dfinal is None else dst.copy_(dfinal)
        with ops.on_device(dev):
            rc = L.bkcore_causal_conv_backward(
                dy.data_ptr(), *ops.strides(dy), x.data_ptr(), *ops.strides(x), ops.DTYPES[x.dtype], w.data_ptr(), ops.ptr(b),
                ops.DTYPES[w.dtype], ops.ptr(st), ops.ptr(dfinal), ops.ptr(lengths), B, T, C, K, ctx.bk_silu, dx.data_ptr(),
                ops.ptr(gp), ops.ptr(dst), ops.ptr(ws), nbytes, ops.stream(dev.index))
        if rc:
            _lib.check(rc, "bkcore_causal_conv_backward")
        return (dx if need_x else None, gp[:C * K].view(C, K).to(w.dtype) if need_w else None,
                gp[C * K:].to(w.dtype) if need_b else None, dst, None, None, None, None)


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
    return _CausalConvFunction.apply(x, weight, bias, initial_state, n, silu, keep, bool(return_state))


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
    x = ops.inner(x)
    w = weight.contiguous()
    b = None if bias is None else bias.contiguous()
    dev = x.device
    y = torch.empty(B, C, dtype=x.dtype, device=dev)
    with ops.on_device(dev):
        rc = _lib.load_held().bkcore_causal_conv_step(
            x.data_ptr(), x.stride(0), ops.DTYPES[x.dtype], state.data_ptr(), w.data_ptr(), ops.ptr(b), ops.DTYPES[w.dtype],
            B, C, K, silu, y.data_ptr(), ops.stream(dev.index))
    if rc:
        _lib.check(rc, "bkcore_causal_conv_step")
    return y


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


class _SelectiveScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, A, Bm, Cm, D, z, bias, state, lengths, softplus, keep, want_state):
        x, delta, Bm, Cm, z = ops.inner(x), ops.inner(delta), ops.inner(Bm), ops.inner(Cm), ops.inner(z)
        A = A.contiguous()
        D, bias, state = (None if t is None else t.contiguous() for t in (D, bias, state))
        B, T, C = x.shape
        N = A.shape[1]
        dev = x.device
        L = _lib.load_held()
        y = torch.empty(B, T, C, dtype=x.dtype, device=dev)
        final = torch.empty(B, C, N, dtype=torch.float32, device=dev) if want_state else None
        if final is not None and T == 0:
            final.zero_() if state is None else final.copy_(state)
        ckpt = None
        if keep:
            ckpt = torch.empty(L.bkcore_selective_scan_checkpoint_bytes(B, T, C, N), dtype=torch.uint8, device=dev)
        nbytes = L.bkcore_selective_scan_workspace_bytes(B, T, C, N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        with ops.on_device(dev):
            rc = L.bkcore_selective_scan(
                x.data_ptr(), *ops.strides(x), delta.data_ptr(), *ops.strides(delta), A.data_ptr(), Bm.data_ptr(),
                *ops.strides(Bm), Cm.data_ptr(), *ops.strides(Cm), ops.ptr(D), ops.ptr(z), *ops.strides(z), ops.ptr(bias),
                softplus, ops.DTYPES[x.dtype], ops.ptr(lengths), ops.ptr(state), B, T, C, N, y.data_ptr(), ops.ptr(final),
                ops.ptr(ckpt), ops.ptr(ws), nbytes, ops.stream(dev.index))
        if rc:
            _lib.check(rc, "bkcore_selective_scan")
        if keep:
            ctx.save_for_backward(x, delta, A, Bm, Cm, D, z, bias, lengths, ckpt)
            ctx.bk_softplus = softplus
            ctx.set_materialize_grads(False)
        return (y, final) if want_state else y

    @staticmethod
    def backward(ctx, dy, dfinal=None):
        ops.once_only("selective_scan")
        x, delta, A, Bm, Cm, D, z, bias, lengths, ckpt = ctx.saved_tensors
        B, T, C = x.shape
        N = A.shape[1]
        dev, dt = x.device, x.dtype
        dy = torch.zeros(B, T, C, dtype=dt, device=dev) if dy is None else ops.inner(dy)
        dfinal = None if dfinal is None else dfinal.contiguous()
        dx = torch.empty(B, T, C, dtype=dt, device=dev)
        dd = torch.empty_like(dx)
        dz = None if z is None else torch.empty_like(dx)
        dB = torch.empty(B, T, N, dtype=dt, device=dev)
        dC = torch.empty_like(dB)
        gp = torch.empty(C * N + 2 * C, dtype=torch.float32, device=dev)
        dh0 = torch.empty(B, C, N, dtype=torch.float32, device=dev) if ctx.needs_input_grad[8] else None
        if B == 0 or T == 0 or C == 0:       # nothing runs: no position, and the state passes through unchanged
            for t in (gp, dB, dC):
                t.zero_()
            if dh0 is not None:
                dh0.zero_() if dfinal is None else dh0.copy_(dfinal)
        L = _lib.load_held()
        nbytes = L.bkcore_selective_scan_backward_workspace_bytes(B, T, C, N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        with ops.on_device(dev):
            rc = L.bkcore_selective_scan_backward(
                dy.data_ptr(), *ops.strides(dy), ops.ptr(dfinal), x.data_ptr(), *ops.strides(x), delta.data_ptr(),
                *ops.strides(delta), A.data_ptr(), Bm.data_ptr(), *ops.strides(Bm), Cm.data_ptr(), *ops.strides(Cm),
                ops.ptr(D), ops.ptr(z), *ops.strides(z), ops.ptr(bias), ctx.bk_softplus, ops.DTYPES[dt], ops.ptr(lengths),
                ckpt.data_ptr(), B, T, C, N, dx.data_ptr(), dd.data_ptr(), gp.data_ptr(), dB.data_ptr(), dC.data_ptr(),
                ops.ptr(dz), ops.ptr(dh0), ws.data_ptr(), nbytes, ops.stream(dev.index))
        if rc:
            _lib.check(rc, "bkcore_selective_scan_backward")
        grads = (dx, dd, gp[:C * N].view(C, N), dB, dC, gp[C * N:C * N + C], dz, gp[C * N + C:], dh0)
        return tuple(g if n else None for g, n in zip(grads, ctx.needs_input_grad)) + (None,) * 4


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
    return _SelectiveScanFunction.apply(x, delta, A, B, C, D, z, delta_bias, initial_state, ln, int(bool(delta_softplus)),
                                        keep, bool(return_state))


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
    code = ops.need_dtype(what, x, delta, B, C, z)
    ops.no_grad_through(what, x, delta, A, B, C, D, z, delta_bias)
    A, D, delta_bias = (None if t is None else t.contiguous() for t in _scan_params(what, x, A, D, delta_bias))
    n = A.shape[1]
    for name, m, shape in (("delta", delta, (b, c)), ("z", z, (b, c)), ("B", B, (b, n)), ("C", C, (b, n))):
        ops.need_shape(what, name, m, shape)
    ops.need_state(what, "state", state, x, (b, c, n), torch.float32)
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError(f"bkcore: {what}: state must be contiguous and 16-byte aligned")
    if A.data_ptr() % 16:
        A = A.clone()
    x, delta, B, C, z = ops.inner(x), ops.inner(delta), ops.inner(B), ops.inner(C), ops.inner(z)
    dev = x.device
    y = torch.empty(b, c, dtype=x.dtype, device=dev)
    with ops.on_device(dev):
        rc = _lib.load_held().bkcore_selective_scan_step(
            x.data_ptr(), x.stride(0), state.data_ptr(), delta.data_ptr(), delta.stride(0), A.data_ptr(), B.data_ptr(),
            B.stride(0), C.data_ptr(), C.stride(0), ops.ptr(D), ops.ptr(z), 0 if z is None else z.stride(0),
            ops.ptr(delta_bias), int(bool(delta_softplus)), code, b, c, n, y.data_ptr(), ops.stream(dev.index))
    if rc:
        _lib.check(rc, "bkcore_selective_scan_step")
    return y
