"""The selective scan where states grow (d A > 0) and a chunk's factor is beyond float32, against the 64-bit definition."""
import pytest
import torch

from mixer_reference import assert_within, d64, scan
from test_gpu_selective import GRADS, NAMES, leaf, scan_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("L", [130, 512, 1023])
@pytest.mark.parametrize("N", [4, 16, 20])
def test_states_that_stay_zero_through_growing_chunks(L, N):
    """Inputs at the last three positions only: every state in front of them is zero, whatever the factors."""
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import bkcore
    v = scan_inputs(1, L, 6, N, torch.float32, seed=L + N)
    v["delta"], v["A"] = torch.ones_like(v["delta"]), 1.5 - v["A"]     # factors of e^2 to e^4 a position, e^128 and more a chunk
    v["x"][:, :-3] = 0
    v["dy"][:, 3:] = 0                                                # the adjoint's state is zero behind the third position
    names = [n for n in NAMES if n not in ("bias", "h0")]
    ls = {n: leaf(v[n]) for n in names}
    y, hT = bkcore.selective_scan(ls["x"], ls["delta"], ls["A"], ls["Bm"], ls["Cm"], ls["D"], ls["z"], return_state=True)
    y.backward(v["dy"].cuda())
    a = {n: d64(v[n]) for n in names}
    r = scan(a["x"], a["delta"], a["A"], a["Bm"], a["Cm"], a["D"], a["z"], None, False, None, None, d64(v["dy"]))
    assert_within(y, r["y"], r["ey"], "y")
    assert_within(hT, r["hT"], r["ehT"], "hT")
    for n, gn in zip(NAMES, GRADS):
        if n in ls:
            assert_within(ls[n].grad, r[gn], r["e" + gn], gn)
