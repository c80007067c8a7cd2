"""The C entry points of the mixing layer's operators refuse bad arguments before any launch (no GPU needed)."""
import ctypes

import pytest

OK, EINVAL, EWS = 0, -1, -4
p = ctypes.c_void_p(256)       # never dereferenced: every call here returns before a launch


@pytest.fixture(scope="module")
def L():
    from bkcore import _lib
    return _lib.load()


def test_layer_norm(L):
    def fwd(x=p, dt=0, pd=0, eps=1e-5, rows=4, D=8, y=p):
        return L.bkcore_layer_norm(x, D, dt, p, p, pd, eps, rows, D, y, None, None)
    assert fwd(rows=0) == OK
    assert fwd(x=None) == EINVAL and fwd(y=None) == EINVAL
    assert fwd(dt=3) == EINVAL and fwd(dt=1, pd=2) == EINVAL and fwd(eps=-1.0) == EINVAL and fwd(eps=float("nan")) == EINVAL
    assert fwd(D=0) == EINVAL and fwd(D=16385) == EINVAL and fwd(rows=-1) == EINVAL

    def bwd(ws, n, gp=p):
        return L.bkcore_layer_norm_backward(p, 8, p, 8, 0, p, 0, p, 4, 8, p, gp, ws, n, None)
    need = L.bkcore_layer_norm_backward_workspace_bytes(4, 8)
    assert need == 2 * 8 * 4
    assert bwd(None, need) == EWS and bwd(p, need - 1) == EWS
    assert L.bkcore_layer_norm_backward(None, 8, p, 8, 0, p, 0, p, 4, 8, p, None, None, 0, None) == EINVAL


def test_causal_conv(L):
    def fwd(dt=0, pd=0, B=1, T=4, C=8, K=4, x=p, w=p):
        return L.bkcore_causal_conv(x, 32, 8, dt, w, None, pd, None, None, B, T, C, K, 0, p, None, None)
    assert fwd(B=0) == OK and fwd(T=0) == OK and fwd(C=0) == OK
    assert fwd(K=1) == EINVAL and fwd(K=5) == EINVAL and fwd(dt=3) == EINVAL and fwd(dt=1, pd=2) == EINVAL
    assert fwd(x=None) == EINVAL and fwd(w=None) == EINVAL and fwd(B=-1) == EINVAL

    def bwd(ws, n):
        return L.bkcore_causal_conv_backward(p, 32, 8, p, 32, 8, 0, p, p, 0, None, None, None, 1, 4, 8, 4, 1, p, p, None, ws, n,
                                             None)
    need = L.bkcore_causal_conv_backward_workspace_bytes(1, 4, 8, 4)
    assert need == 5 * 8 * 4
    assert bwd(None, 0) == EWS and bwd(p, need - 1) == EWS
    assert L.bkcore_causal_conv_step(p, 8, 0, None, p, p, 0, 2, 8, 4, 0, p, None) == EINVAL
    assert L.bkcore_causal_conv_step(p, 8, 0, p, p, p, 0, 0, 8, 4, 0, p, None) == OK


def test_selective_scan(L):
    def fwd(B=1, T=16, C=8, N=16, dt=0, x=p, ws=None, n=0):
        return L.bkcore_selective_scan(x, 1, 1, p, 1, 1, p, p, 1, 1, p, 1, 1, None, None, 0, 0, None, 1, dt, None, None, B, T, C,
                                       N, p, None, None, ws, n, None)
    assert fwd(B=0) == OK and fwd(T=0) == OK and fwd(C=0) == OK
    assert fwd(N=0) == EINVAL and fwd(N=65) == EINVAL and fwd(dt=3) == EINVAL and fwd(x=None) == EINVAL
    need = L.bkcore_selective_scan_workspace_bytes(1, 4096, 8, 16)          # few channels: chunks, with their end states
    assert need > 0 and need % (8 * 17 * 4) == 0
    assert fwd(T=4096) == EWS and fwd(T=4096, ws=p, n=need - 1) == EWS
    assert L.bkcore_selective_scan_workspace_bytes(64, 2048, 4096, 16) == 0  # channels enough: one pass
    assert L.bkcore_selective_scan_checkpoint_bytes(2, 17, 8, 16) == 2 * 2 * 8 * 16 * 4
    assert L.bkcore_selective_scan_backward_workspace_bytes(1, 16, 8, 16) > 0
    assert L.bkcore_selective_scan_step(p, 8, None, p, 8, p, p, 16, p, 16, None, None, 0, None, 1, 0, 2, 8, 16, p, None) == EINVAL
    odd = ctypes.c_void_p(260)
    assert L.bkcore_selective_scan_step(p, 8, odd, p, 8, p, p, 16, p, 16, None, None, 0, None, 1, 0, 2, 8, 16, p, None) == EINVAL


def test_operators_refuse_cpu_tensors():
    import torch

    import bkcore
    x = torch.zeros(2, 4, 8)
    for call in (lambda: bkcore.layer_norm(x), lambda: bkcore.causal_conv(x, torch.zeros(8, 4)),
                 lambda: bkcore.causal_conv_step(x[0], x, torch.zeros(8, 4)),
                 lambda: bkcore.selective_scan(x, x, torch.zeros(8, 4), x[..., :4], x[..., :4])):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


def test_sliding_attention(L):
    def fwd(dt=1, B=1, H=4, Hk=2, T=8, D=16, W=4, S=1, scale=0.25, q=p, out=p):
        return L.bkcore_sliding_attention(q, 1, 1, 1, p, 1, 1, 1, p, 1, 1, 1, dt, None, B, H, Hk, T, D, W, S, scale, out, None, None,
                                          None)
    assert fwd(B=0) == OK and fwd(T=0) == OK
    for bad in (dict(dt=3), dict(H=3), dict(Hk=0), dict(D=0), dict(D=129), dict(W=0), dict(S=-1), dict(S=65),
                dict(scale=float("nan")), dict(B=-1), dict(q=None), dict(out=None)):
        assert fwd(**bad) == EINVAL, bad

    def bwd(ws, n, T=2000, lse=p):
        return L.bkcore_sliding_attention_backward(p, 1, 1, 1, p, 1, 1, 1, p, 1, 1, 1, p, 1, 1, 1, p, None, lse, 1, None, 1, 4, 2, T, 16,
                                                   8, 2, 0.25, p, p, p, ws, n, None)
    need = L.bkcore_sliding_attention_backward_workspace_bytes(1, 4, 2, 2000, 16, 8, 2)
    assert need > 4 * 2000 * 4                              # delta, and the sinks' partial sums of a long rest
    assert L.bkcore_sliding_attention_backward_workspace_bytes(1, 4, 2, 2000, 16, 8, 0) == 4 * 2000 * 4
    assert bwd(None, 0) == EWS and bwd(p, need - 1) == EWS and bwd(p, need, lse=None) == EINVAL

    def step(cap=10, W=8, S=2, ws=None, n=0, pos=p):
        return L.bkcore_sliding_attention_step(p, 1, 1, p, 1, 1, p, 1, 1, p, 1, 1, 16, p, 1, 1, 16, pos, 1, 1, 4, 2, cap, 16, W, S,
                                               0.25, p, ws, n, None)
    assert step(cap=9) == EINVAL and step(pos=None) == EINVAL and step(W=0) == EINVAL
    need = L.bkcore_sliding_attention_step_workspace_bytes(1, 4, 2, 5000, 16, 4096, 4)
    assert need > 0 and step(cap=5000, W=4096, S=4) == EWS and step(cap=5000, W=4096, S=4, ws=p, n=need - 1) == EWS
    assert L.bkcore_sliding_attention_step_workspace_bytes(1, 4, 2, 10, 16, 8, 2) == 0

    def fill(cap=10, S=2, D=16, k=p):
        return L.bkcore_sliding_cache_fill(k, 1, 1, 1, p, 1, 1, 1, p, 1, 1, 16, p, 1, 1, 16, None, 1, 1, 2, 8, cap, D, S, None)
    assert fill(cap=2) == EINVAL and fill(D=129) == EINVAL and fill(k=None) == EINVAL
