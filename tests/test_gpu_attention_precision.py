"""What sliding-window attention promises beyond the rounding of its operands' type."""
import pytest
import torch

from attention_bounds import NEAR, rounding_ratio
from mixer_reference import assert_within, attention, d64
from test_gpu_attention import BF16, F16, F32, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def train(q, k, v, do, window, sinks, lengths=None):
    import bkcore
    ls = [t.detach().requires_grad_() for t in (q, k, v)]
    o = bkcore.sliding_attention(*ls, window, sinks, lengths=lengths)
    return (o.detach(), *torch.autograd.grad(o, ls, do))


# a row that sees one key has that key's value as its output and no score gradient at all
@pytest.mark.parametrize("B,H,Hk,L,D,window,sinks", [(2, 4, 2, 1, 64, 7, 0), (3, 2, 2, 1, 20, 5, 4), (2, 8, 4, 200, 32, 1, 0),
                                                     (6, 32, 16, 300, 128, 1, 0), (1, 5, 1, 70, 73, 1, 0), (9, 32, 32, 1, 128, 30, 16)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_of_one_key_have_no_score_gradient(B, H, Hk, L, D, window, sinks, dtype):
    q, k, v, do = (t.cuda() for t in inputs(B, H, Hk, L, D, dtype, seed=L + D))
    o, dq, dk, dv = train(q, k, v, do, window, sinks)
    assert torch.equal(o, v.repeat_interleave(H // Hk, 1))
    assert (dq == 0).all() and (dk == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_first_rows_have_no_score_gradient(dtype):
    q, k, v, do = (t.cuda() for t in inputs(2, 4, 2, 150, 64, dtype, seed=1))
    do[:, :, 1:] = 0
    o, dq, dk, dv = train(q, k, v, do, 40, 3)
    assert (dq == 0).all() and (dk == 0).all()
    # p is the exponential of a score less itself: |score| stays below 8, its product's rounding is worth 8 ln2 2^-24, the
    # exponential 2^-23
    g = do[:, :, 0].cpu().double().view(2, 2, 2, 64)
    assert_within(dv[:, :, 0], g.sum(2), 2.0 ** -21 * g.abs().sum(2))


# lengths with and without a part of the sinks behind the first keys, shared heads, a batch that takes 128 rows a workgroup
@pytest.mark.parametrize("B,H,Hk,L,D,window,sinks", [(1, 2, 1, 257, 32, 31, 33), (2, 2, 2, 400, 128, 8, 64), (1, 4, 4, 150, 64, 40, 3),
                                                     (1, 2, 1, 900, 64, 300, 4), (6, 16, 16, 300, 128, 150, 4), (1, 3, 3, 300, 73, 60, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_results_are_as_near_as_their_rounding(B, H, Hk, L, D, window, sinks, dtype):
    q, k, v, do = inputs(B, H, Hk, L, D, dtype, seed=L)
    got = train(*(t.cuda() for t in (q, k, v, do)), window, sinks)
    r = attention(*d64(q, k, v), window, sinks, D ** -0.5, 0.0, None, d64(do))
    for t, n in zip(got, ("o", "dq", "dk", "dv")):
        assert rounding_ratio(t, r[n]) <= NEAR, n


@pytest.mark.parametrize("B,H,Hk,D,window,sinks", [(4, 8, 2, 64, 400, 4), (16, 16, 16, 128, 30, 2), (1, 5, 1, 73, 800, 0)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_single_tokens_are_as_near_as_their_rounding(B, H, Hk, D, window, sinks, dtype):
    """At the last position that fills the cache every slot is visible, in any order."""
    import bkcore
    slots = window + sinks
    q, k, v, _ = inputs(B, H, Hk, slots, D, dtype, seed=D)
    kc, vc = k.cuda(), v.cuda()
    pos = torch.full((B,), slots - 1, dtype=torch.int32, device="cuda")
    got = bkcore.sliding_attention_step(q[:, :, -1].cuda(), k[:, :, -1].cuda(), v[:, :, -1].cuda(), kc, vc, pos, window, sinks)
    K, V = (t.double().repeat_interleave(H // Hk, 1) for t in (k, v))
    p = torch.softmax((K @ q[:, :, -1, :, None].double())[..., 0] * D ** -0.5, -1)
    assert rounding_ratio(got, (p[..., None] * V).sum(2)) <= NEAR


# float16 gradients over its whole range: score gradients far below its smallest steps and beyond its largest value, values so
# small that the output is kept in whole steps of 2^-24, rows of very different size in one sequence
ANY_SIZE = [(1024, 64, 512, 0, 1, 1, 1e-4), (1024, 64, 512, 4, 1, 1, 1e-4), (300, 64, 4, 0, 0.05, 1, 1e4), (300, 128, 4, 0, 0.02, 1, 1e4),
            (900, 32, 8, 40, 0.02, 1, 1e4), (300, 64, 40, 3, 1, 1e-3, 1e2), (300, 64, 40, 3, 1, 1e-5, 1e4),
            (200, 128, 30, 2, 0.1, 1e3, 1e-2), (300, 20, 60, 2, 1, 1, 1e-4)]


@pytest.mark.parametrize("B,H,Hk,L,D,window,sinks,qk,vs,dos",
                         [(1, 4, 1, *c) for c in ANY_SIZE] + [(6, 16, 16, *c) for c in ANY_SIZE if c[0] <= 300])
def test_float16_gradients_of_any_size(B, H, Hk, L, D, window, sinks, qk, vs, dos):
    q, k, v, do = (t.float() for t in inputs(B, H, Hk, L, D, F32, seed=D + L))
    q, k, v, do = (qk * q).half(), (qk * k).half(), (vs * v).half(), (dos * do).half()
    got = train(*(t.cuda() for t in (q, k, v, do)), window, sinks)
    r = attention(*d64(q, k, v), window, sinks, D ** -0.5, 0.0, None, d64(do))
    for t, n in zip(got, ("o", "dq", "dk", "dv")):
        want = r[n]                                     # where the definition is beyond float16's largest value, so is the result
        border = (want.abs() / 65520 - 1).abs() < 2.0 ** -11
        over = torch.isinf(want.half())
        assert torch.equal(torch.isinf(t.cpu())[~border], over[~border]) and not torch.isnan(t).any(), n
        fine = ~over & ~border
        assert rounding_ratio(t.cpu()[fine], want[fine]) <= NEAR, n


def test_float16_gradients_of_rows_of_any_size():
    """Each row's dout at its own power of two: dq is held row by row, dk and dv by the sizes of what reaches a key."""
    q, k, v, do = inputs(2, 4, 2, 300, 64, F32, seed=3)
    g = torch.Generator().manual_seed(4)
    size = 2.0 ** torch.randint(-12, 12, (2, 4, 300, 1), generator=g)
    q, k, v, do = q.half(), k.half(), v.half(), (size * do).half()
    got = train(*(t.cuda() for t in (q, k, v, do)), 40, 3)
    r = attention(*d64(q, k, v), 40, 3, 0.125, 0.0, None, d64(do))
    for t, n in zip(got, ("o", "dq", "dk", "dv")):
        assert rounding_ratio(t, r[n]) <= NEAR, n
    dq, want = d64(got[1]), r["dq"]
    off, least = (dq - want).norm(dim=-1), (want.half().double() - want).norm(dim=-1)
    assert (off <= 2 * least + 2.0 ** -24).all()        # of a row's 64 roundings one or two fall to the other side
