"""What sliding-window attention promises beyond the rounding of its operands' type."""
import pytest
import torch

from mixer_reference import assert_within
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
