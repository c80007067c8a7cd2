"""Sliding-window attention on batches large enough for the kernels of 128 rows a workgroup, against the 64-bit definition."""
import pytest
import torch

from mixer_reference import assert_within, attention, d64, half_step
from test_gpu_attention import BF16, F16, F32, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def workgroups(B, heads, L):
    return B * heads * ((L + 127) // 128)


# windows inside a tile and beyond it; sinks with a rest behind the wide key tile, without one, and none
@pytest.mark.parametrize("H,Hk,D,window,sinks", [(16, 16, 32, 37, 4), (32, 16, 64, 8, 40), (16, 16, 128, 150, 0), (16, 16, 128, 8, 40),
                                                 (16, 16, 128, 500, 4), (16, 16, 20, 37, 4), (16, 16, 100, 70, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_wide_tiles(H, Hk, D, window, sinks, dtype):
    import bkcore
    B, L, lens = 6, 300, [300, 0, 129, 128, 257, 64]
    assert workgroups(B, Hk, L) >= 256              # both the queries' and the keys' kernels take 128 rows from here on
    q, k, v, do = inputs(B, H, Hk, L, D, dtype, seed=D + window)
    for i, n in enumerate(lens):
        for t in (q, k, v, do):
            t[i, :, n:] = float("nan")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ls = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = bkcore.sliding_attention(*ls, window, sinks, lengths=n)
    o.backward(do.cuda())
    r = attention(*d64(q, k, v), window, sinks, D ** -0.5, half_step(dtype), lens, d64(do))
    assert_within(o, r["o"], r["eo"], "o")
    for t, name in zip(ls, ("dq", "dk", "dv")):
        assert_within(t.grad, r[name], r["e" + name], name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_wide_queries_over_narrow_keys(dtype):
    """Shared heads: 128 queries a workgroup, 64 keys."""
    import bkcore
    B, H, Hk, L, D = 2, 64, 4, 300, 64
    assert workgroups(B, H, L) >= 256 > workgroups(B, Hk, L)
    q, k, v, do = inputs(B, H, Hk, L, D, dtype, seed=1)
    ls = [t.cuda().requires_grad_() for t in (q, k, v)]
    o = bkcore.sliding_attention(*ls, 90, 5)
    o.backward(do.cuda())
    r = attention(*d64(q, k, v), 90, 5, D ** -0.5, half_step(dtype), None, d64(do))
    assert_within(o, r["o"], r["eo"], "o")
    for t, name in zip(ls, ("dq", "dk", "dv")):
        assert_within(t.grad, r[name], r["e" + name], name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_wide_and_narrow_tiles_agree(dtype):
    """The same sequence alone and in a batch that takes the wide tiles: equal outputs (a row's sums run in the same order)."""
    import bkcore
    q, k, v, _ = inputs(1, 16, 16, 300, 64, dtype, seed=2)
    alone = bkcore.sliding_attention(q.cuda(), k.cuda(), v.cuda(), 100, 4)
    many = bkcore.sliding_attention(*(t.cuda().expand(6, -1, -1, -1).contiguous() for t in (q, k, v)), 100, 4)
    for b in range(6):
        assert torch.equal(many[b], alone[0])
