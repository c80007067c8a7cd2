"""Causal attention in a sliding window with sinks (a few first tokens that stay visible): the local mixing path of the
hybrid layer without its block borders (reference src/models/phase7/hybrid_attention.py:93-103), for training, for prompts
and, on a rolling key / value cache, for single tokens.

Query i of a sequence sees the keys j <= i with ``i - j < window`` or ``j < sinks``.  Positions at or behind ``lengths``
(B,) are padding of a right-padded batch: their values do not matter, outputs and gradients there are zero."""
from __future__ import annotations

import torch

from . import _layer_ops as ops
from . import _lib

MAX_HEAD_DIM = 128   # BKCORE_ATTENTION_MAX_HEAD_DIM
MAX_SINKS = 64       # BKCORE_ATTENTION_MAX_SINKS


def _window(what: str, window, sinks) -> tuple[int, int]:
    window, sinks = int(window), int(sinks)
    if window < 1:
        raise ValueError(f"bkcore: {what}: a window holds at least one position, got {window}")
    if not 0 <= sinks <= MAX_SINKS:
        raise ValueError(f"bkcore: {what}: 0 to {MAX_SINKS} sinks, got {sinks}")
    return window, sinks


def _heads(what: str, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, dims: int) -> int:
    """Checks q (B, H, ...), k and v (B, Hk, ...) and returns the type's code."""
    ops.need_device(q, k, v)
    code = ops.need_dtype(what, q, k, v)
    if q.dim() != dims or k.dim() != dims or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError(f"bkcore: {what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if q.shape[1] < 1 or k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"bkcore: {what}: {q.shape[1]} query heads are no multiple of {k.shape[1]} key heads")
    if not 1 <= q.shape[-1] <= MAX_HEAD_DIM:
        raise ValueError(f"bkcore: {what}: head dimensions 1 to {MAX_HEAD_DIM}, got {q.shape[-1]}")
    return code


def _scale(what: str, scale, D: int) -> float:
    scale = D ** -0.5 if scale is None else float(scale)
    if scale != scale:
        raise ValueError(f"bkcore: {what}: scale is not a number")
    return scale


def sliding_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int, sinks: int = 0,
                      scale: float | None = None, lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q (B, H, L, D) to k, v (B, Hk, L, D) of the same positions, H a multiple of Hk (neighbouring query heads
    share a key / value head), D <= 128, at most 64 sinks; ``scale`` defaults to D ** -0.5.  Heads and positions may have any
    strides (slices of one projection).  The result (B, H, L, D) has its heads inside a position in memory.

    Scores, softmax and sums are float32; probabilities and score gradients enter their products as two values of the
    operands' type, so results are as near as their own rounding.  A non-finite key or value inside a sequence may reach
    any row that works on the same tile of keys, not only those that see it, and leave NaN where the formula is infinite."""
    what = "sliding_attention"
    _heads(what, q, k, v, 4)
    B, H, T, D = q.shape
    window, sinks = _window(what, window, sinks)
    scale = _scale(what, scale, D)
    n = ops.lengths_arg(what, lengths, q, B, T)
    with ops.on_device(q.device):
        return _lib.load_native().sliding_attention(q, k, v, n, window, sinks, scale, ops.wants_grad(q, k, v),
                                                    ops.stream(q.device.index))


def _meet(distance: int, a: list, b: list) -> bool:
    """Whether an element of b, which begins `distance` behind a, is one of a's; (stride, size) of either's dimensions with
    strides descending.  Dimensions of equal stride are told apart exactly; where the largest strides left differ, views whose
    reaches meet count as meeting."""
    if not -sum(s * (n - 1) for s, n in b) <= distance <= sum(s * (n - 1) for s, n in a):
        return False
    if not a or not b or a[0][0] != b[0][0] or a[0][0] == 0:
        return True
    (stride, na), (_, nb) = a[0], b[0]
    a, b = a[1:], b[1:]
    least = -(-(-sum(s * (n - 1) for s, n in b) - distance) // stride)
    most = (sum(s * (n - 1) for s, n in a) - distance) // stride
    return any(_meet(distance + d * stride, a, b) for d in range(max(least, 1 - na), min(most, nb - 1) + 1))


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one type have memory in common."""
    if a.data_ptr() > b.data_ptr():
        a, b = b, a
    size, distance = a.element_size(), b.data_ptr() - a.data_ptr()
    if distance >= a.numel() * size and a.is_contiguous() or not (a.numel() and b.numel()):
        return False
    steps = [sorted(((t.stride(i), t.shape[i]) for i in range(t.dim()) if t.shape[i] > 1), reverse=True) for t in (a, b)]
    if distance % size:      # elements that straddle one another: by their reach
        return distance < (sum(s * (n - 1) for s, n in steps[0]) + 1) * size
    return _meet(distance // size, *steps)


def _cache(what: str, q: torch.Tensor, k: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, sinks: int) -> int:
    """Checks the caches (B, Hk, slots, D) and returns the number of slots."""
    ops.need_device(q, k_cache, v_cache)
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if c.dim() != 4 or c.shape[:2] != k.shape[:2] or c.shape[3] != k.shape[-1] or c.shape != k_cache.shape:
            raise ValueError(f"bkcore: {what}: {name} is (B, Hk, slots, D), got {tuple(c.shape)}")
        if c.shape[3] > 1 and c.stride(3) != 1:
            raise ValueError(f"bkcore: {what}: the last dimension of {name} must be contiguous")
        if not c.is_contiguous():
            reach = 1
            for stride, size in sorted((c.stride(i), c.shape[i]) for i in range(4) if c.shape[i] > 1):
                if stride < reach:
                    raise ValueError(f"bkcore: {what}: slots of {name} overlap")
                reach += stride * (size - 1)
        ops.need_state(what, name, c, q, tuple(c.shape), q.dtype)
    if _share(k_cache, v_cache):
        raise ValueError(f"bkcore: {what}: k_cache and v_cache share memory")
    if k_cache.shape[2] <= sinks:
        raise ValueError(f"bkcore: {what}: {k_cache.shape[2]} slots leave none behind {sinks} sinks")
    return k_cache.shape[2]


def sliding_cache_fill(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       lengths: torch.Tensor | None = None, sinks: int = 0) -> None:
    """Writes a prompt's keys and values (B, Hk, L, D) into rolling caches (B, Hk, slots, D): the first ``sinks`` positions
    and the last ``slots - sinks`` behind them.  Position p lives in slot p for p < sinks and in slot
    ``sinks + (p - sinks) % (slots - sinks)`` behind; slots of no position stay as they were.  k and v lie outside the
    caches."""
    what = "sliding_cache_fill"
    _heads(what, k, k, v, 4)
    _, sinks = _window(what, 1, sinks)
    ops.no_grad_through(what, k, v)
    _cache(what, k, k, k_cache, v_cache, sinks)
    if any(_share(t, c) for t in (k, v) for c in (k_cache, v_cache)):
        raise ValueError(f"bkcore: {what}: k or v shares memory with a cache, whose slots are written in no order")
    n = ops.lengths_arg(what, lengths, k, k.shape[0], k.shape[2])
    with ops.on_device(k.device):
        _lib.load_native().sliding_cache_fill(k, v, k_cache, v_cache, n, sinks, ops.stream(k.device.index))


def sliding_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           positions: torch.Tensor, window: int, sinks: int = 0,
                           scale: float | None = None) -> torch.Tensor:
    """``sliding_attention`` for one token of each sequence: q (B, H, D), k and v (B, Hk, D) of the token at ``positions``
    (B,), which are written into the rolling caches (see ``sliding_cache_fill``; at least ``window + sinks`` slots) in place.
    A negative position, or one from 2**31 on, leaves its sequence alone: output zero, cache as it was.  No gradient."""
    what = "sliding_attention_step"
    _heads(what, q, k, v, 3)
    window, sinks = _window(what, window, sinks)
    ops.no_grad_through(what, q, k, v)
    cap = _cache(what, q, k, k_cache, v_cache, sinks)
    if cap < window + sinks:
        raise ValueError(f"bkcore: {what}: a window of {window} and {sinks} sinks need {window + sinks} slots, got {cap}")
    scale = _scale(what, scale, q.shape[-1])
    ops.need_shape(what, "positions", positions, (q.shape[0],))
    ops.need_device(q, positions)
    if positions.dtype == torch.int64:
        positions = positions.clamp(-1, 2 ** 31).to(torch.int32)      # 2**31 becomes the lowest int32: left alone too
    elif positions.dtype != torch.int32:
        raise TypeError(f"bkcore: {what}: positions are int32 or int64, not {positions.dtype}")
    with ops.on_device(q.device):
        return _lib.load_native().sliding_attention_step(q, k, v, k_cache, v_cache, positions, window, sinks, scale,
                                                         ops.stream(q.device.index))
