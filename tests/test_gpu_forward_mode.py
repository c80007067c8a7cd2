"""Forward-mode tangents: the operators have no such derivative and say so, whichever operand carries one."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def rn(*shape):
    return torch.randn(*shape, device="cuda")


def pos():
    return torch.zeros(2, dtype=torch.int32, device="cuda")


CALLS = {
    "layer_norm": lambda: [rn(2, 8), rn(8), rn(8)],
    "causal_conv": lambda: [rn(2, 5, 8), rn(8, 4), rn(8)],
    "causal_conv_step": lambda: [rn(2, 8), rn(2, 3, 8), rn(8, 4), rn(8)],
    "selective_scan": lambda: [rn(2, 5, 8), rn(2, 5, 8), rn(8, 4), rn(2, 5, 4), rn(2, 5, 4), rn(8), rn(2, 5, 8), rn(8)],
    "selective_scan_step": lambda: [rn(2, 8), rn(2, 8, 4), rn(2, 8), rn(8, 4), rn(2, 4), rn(2, 4), rn(8), rn(2, 8), rn(8)],
    "sliding_attention": lambda: [rn(2, 4, 5, 16), rn(2, 2, 5, 16), rn(2, 2, 5, 16)],
    "sliding_attention_step": lambda: [rn(2, 4, 16), rn(2, 2, 16), rn(2, 2, 16), rn(2, 2, 10, 16), rn(2, 2, 10, 16)],
    "sliding_cache_fill": lambda: [rn(2, 2, 5, 16), rn(2, 2, 5, 16), rn(2, 2, 10, 16), rn(2, 2, 10, 16)],
}
MORE = {"sliding_attention": lambda: (4,), "sliding_attention_step": lambda: (pos(), 8, 2)}


@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name):
    import bkcore
    call, more = getattr(bkcore, name), MORE.get(name, lambda: ())()
    count = len(CALLS[name]())
    call(*CALLS[name](), *more)
    for i in range(count):
        with forward_ad.dual_level():
            args = CALLS[name]()
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            kept = [forward_ad.unpack_dual(a).primal.clone() for a in args]
            with pytest.raises(RuntimeError):
                call(*args, *more)
            if name.endswith(("_step", "_fill")):       # refused before anything was written
                for a, k in zip(args, kept):
                    assert torch.equal(forward_ad.unpack_dual(a).primal, k)
