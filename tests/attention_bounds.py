"""How near sliding-window attention comes to the rounding of its results, and the same computed with one of the two-value
operands or the output's remainder left out."""
import math

import torch

from mixer_reference import d64

# Probabilities and score gradients are two values of the operands' type: off by half a step of half a step (float16: a step
# of a step, its conversion cuts), 2^-16 in bfloat16 and 2^-20 in float16; so is delta.  Float32 sums and exponentials are worth
# about 2^-20.  Over n <= 900 terms of random sign that is at most sqrt(n) of the result's size, 2^-11 and 2^-15; rounding the
# result is worth 0.42 half steps on the average, 2^-9.3 and 2^-12.3.  Squares add: sqrt(1 + 2^-3.4 / 2) - 1 = 0.05 if every term
# were at its worst and of one sign; being uniform and of both they are a third of that at most, squared a ninth: 0.006.
NEAR = 1.02


def rounding_ratio(got, want):
    """|got - want| over |want rounded to got's type - want|, 2-norms."""
    want = want.double()
    return float((d64(got) - want).norm() / (want.to(got.dtype).double() - want).norm())


def emulate(q, k, v, do, window, sinks, scale, dtype, once=()):
    """o, dq, dk, dv of one head in 64 bits with the roundings of the kernels; `once`: which of "p", "ds", "delta" are rounded
    to the operands' type only once."""
    def two(x):
        hi = x.to(dtype).double()
        return hi + (x - hi).to(dtype).double()
    n = q.shape[0]
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    see = (j <= i) & ((i - j < window) | (j < sinks))
    p = torch.softmax((q @ k.t() * scale).masked_fill(~see, -math.inf), -1)
    pr = p.to(dtype).double() if "p" in once else two(p)
    o = pr @ v
    seen = o.to(dtype).double() if "delta" in once else two(o)
    ds = p * (do @ v.t() - (do * seen).sum(-1, keepdim=True))
    ds = ds.to(dtype).double() if "ds" in once else two(ds)
    return [t.to(dtype) for t in (o, ds @ k * scale, ds.t() @ q * scale, pr.t() @ do)]
