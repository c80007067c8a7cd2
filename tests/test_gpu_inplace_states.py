"""Buffers that the single-token calls update in place, next to gradients that still need them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def rn(*shape):
    return torch.randn(*shape, device="cuda")


def conv_step(state):
    import bkcore
    bkcore.causal_conv_step(rn(2, 8), state, rn(8, 4))


def scan_step(state):
    import bkcore
    bkcore.selective_scan_step(rn(2, 8), state, rn(2, 8), rn(8, 4), rn(2, 4), rn(2, 4))


def attention_step(caches):
    import bkcore
    bkcore.sliding_attention_step(rn(2, 4, 16), rn(2, 2, 16), rn(2, 2, 16), *caches, torch.zeros(2, dtype=torch.int32, device="cuda"), 8, 2)


def cache_fill(caches):
    import bkcore
    bkcore.sliding_cache_fill(rn(2, 2, 5, 16), rn(2, 2, 5, 16), *caches, None, 2)


def test_every_call_counts_as_a_change_of_what_it_writes():
    conv, scan, caches = rn(2, 3, 8), rn(2, 8, 4), (rn(2, 2, 10, 16), rn(2, 2, 10, 16))
    for call, arg, tensors in ((conv_step, conv, [conv]), (scan_step, scan, [scan]), (attention_step, caches, caches),
                               (cache_fill, caches, caches)):
        before = [t._version for t in tensors]
        view = [t[:1] for t in tensors]
        call(arg)
        for t, v, b in zip(tensors, view, before):
            assert t._version > b and v._version == t._version, call.__name__


def test_a_state_that_moved_on_is_noticed_by_the_convolutions_backward():
    import bkcore
    state, w = rn(2, 3, 8), rn(8, 4).requires_grad_()
    y = bkcore.causal_conv(rn(2, 5, 8), w, initial_state=state)
    with torch.no_grad():
        conv_step(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_state_that_moved_on_is_noticed_by_another_operation():
    state, w = rn(2, 8, 4), rn(2, 8, 4).requires_grad_()
    y = (state * w).sum()
    scan_step(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("call", [attention_step, cache_fill])
@pytest.mark.parametrize("which", [0, 1])
def test_caches_that_moved_on_are_noticed_by_the_attentions_backward(call, which):
    import bkcore
    caches = (rn(2, 2, 10, 16), rn(2, 2, 10, 16))
    q, other = rn(2, 4, 10, 16).requires_grad_(), rn(2, 2, 10, 16)
    kv = [other, other.clone()]
    kv[which] = caches[which]
    o = bkcore.sliding_attention(q, *kv, 4)
    with torch.no_grad():
        call(caches)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_inference_tensors_are_updated_too():
    import bkcore
    with torch.inference_mode():
        state = torch.zeros(2, 3, 8, device="cuda")
        x = rn(2, 8)
        bkcore.causal_conv_step(x, state, rn(8, 4))
        assert torch.equal(state[:, 2], x)
        caches = (torch.zeros(2, 2, 10, 16, device="cuda"), torch.zeros(2, 2, 10, 16, device="cuda"))
        attention_step(caches)
        assert (caches[0][:, :, 0] != 0).all()


@pytest.mark.parametrize("outside", [-1, -2 ** 31, -2 ** 32, -2 ** 33 + 1, -2 ** 63, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 63 - 1])
def test_positions_outside_int32_leave_their_sequence_alone(outside):
    """Their low 32 bits are positions that the cache has."""
    import bkcore
    q, k, v = rn(2, 4, 16), rn(2, 2, 16), rn(2, 2, 16)
    kc, vc = rn(2, 2, 10, 16), rn(2, 2, 10, 16)
    k0, v0 = kc.clone(), vc.clone()
    o = bkcore.sliding_attention_step(q, k, v, kc, vc, torch.tensor([outside, 0], device="cuda"), 8, 2)
    assert (o[0] == 0).all() and torch.equal(kc[0], k0[0]) and torch.equal(vc[0], v0[0])
    assert torch.equal(o[1], v[1].repeat_interleave(2, 0)) and torch.equal(kc[1, :, 0], k[1])
