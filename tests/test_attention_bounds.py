"""The bound that the attention's precision is tested with holds for two-value operands and does not for single ones."""
import pytest
import torch

from attention_bounds import NEAR, emulate, rounding_ratio
from mixer_reference import attention, d64


@pytest.mark.parametrize("L,D,window,sinks", [(257, 32, 31, 33), (400, 128, 8, 64), (150, 64, 40, 3), (900, 64, 300, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_bound_tells_one_rounding_from_two(L, D, window, sinks, dtype):
    g = torch.Generator().manual_seed(L)
    q, k, v, do = (torch.randn(1, 1, L, D, generator=g).to(dtype) for _ in range(4))
    r = attention(*d64(q, k, v), window, sinks, D ** -0.5, 0.0, None, d64(do))

    def far(*once):
        got = emulate(*(t[0, 0] for t in d64(q, k, v, do)), window, sinks, D ** -0.5, dtype, once)
        return [n for t, n in zip(got, ("o", "dq", "dk", "dv")) if rounding_ratio(t, r[n][0, 0]) > NEAR]
    assert far() == []
    assert far("p") == ["o", "dq", "dk", "dv"]       # dq and dk through delta
    assert far("ds") == ["dq", "dk"]
    assert far("delta") == ["dq", "dk"]
