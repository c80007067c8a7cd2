"""The short causal convolution and the selective scan on the GPU against their 64-bit definitions."""
import pytest
import torch

from mixer_reference import assert_within, conv, d64, directional, scan

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def leaf(t):
    return None if t is None else t.cuda().requires_grad_()


# ---------------------------------------------------------------------------------------------------------- convolution

def conv_inputs(B, L, C, K, dtype, seed=0, params=F32):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    return (rn(B, L, C).to(dtype), (rn(C, K) * K ** -0.5).to(params), (0.2 * rn(C)).to(params), rn(B, K - 1, C).to(dtype),
            rn(B, L, C).to(dtype), rn(B, K - 1, C).to(dtype))


def check_conv(x, w, b, st, dy, df, act, lens=None):
    import bkcore
    ls = [leaf(t) for t in (x, w, b, st)]
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    y, fin = bkcore.causal_conv(ls[0], ls[1], ls[2], act, n, ls[3], return_state=True)
    torch.autograd.backward([y, fin], [dy.cuda(), df.cuda()])
    r = conv(*d64(x, w, b), act == "silu", lens, d64(st), d64(dy), d64(df))
    assert y.dtype == x.dtype and fin.dtype == x.dtype
    assert_within(y, r["y"], r["ey"], "y")
    assert torch.equal(fin.double().cpu(), r["final"])
    assert_within(ls[0].grad, r["dx"], r["edx"], "dx")
    assert_within(ls[1].grad, r["dw"], r["edw"], "dw")
    if b is not None:
        assert_within(ls[2].grad, r["db"], r["edb"], "db")
    if st is not None:
        assert_within(ls[3].grad, r["dstate"], r["edstate"], "dstate")


@pytest.mark.parametrize("B,L,C,K", [(1, 1, 1, 2), (2, 2, 3, 4), (1, 16, 8, 3), (3, 17, 16, 4), (2, 33, 40, 2), (1, 255, 5, 4),
                                     (2, 257, 264, 4), (1, 513, 24, 3)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", [None, "silu"])
def test_conv_shapes(B, L, C, K, dtype, act):
    check_conv(*conv_inputs(B, L, C, K, dtype, seed=L * C + K), act)


@pytest.mark.parametrize("K", [2, 3, 4])
def test_conv_lengths(K):
    lens = [0, 1, 2, 31, 32, 64, 300, -5]          # beyond the batch's length and below zero count as the nearest of the two
    x, w, b, st, dy, df = conv_inputs(8, 64, 16, K, BF16, seed=K)
    for i, n in enumerate(lens):                    # padding is not read
        x[i, max(n, 0):] = float("nan")
        dy[i, max(n, 0):] = float("inf")
    x[6], dy[6] = conv_inputs(1, 64, 16, K, BF16, seed=77)[0][0], 1.0
    check_conv(x, w, b, st, dy, df, "silu", lens)
    check_conv(x, w, None, None, dy, df, None, lens)


def test_conv_parameters_of_the_inputs_type_and_int64_lengths():
    import bkcore
    x, w, b, st, dy, df = conv_inputs(2, 20, 32, 4, F16, params=F16)
    check_conv(x, w, b, st, dy, df, "silu")
    n = torch.tensor([5, 1 << 40], device="cuda")
    y = bkcore.causal_conv(x.cuda(), w.cuda(), b.cuda(), None, n)
    r = conv(*d64(x, w, b), False, [5, 20])
    assert_within(y, r["y"], r["ey"])


def test_conv_strided_input_and_gradient():
    import bkcore
    x, w, b, st, dy, df = conv_inputs(3, 40, 24, 4, BF16)
    r = conv(*d64(x, w, b), True, None, None, d64(dy))
    both = torch.full((3, 40, 60), float("nan"), dtype=BF16, device="cuda")
    for off in (0, 8, 3):                            # aligned and unaligned slices of a wider projection
        both[..., off:off + 24] = x.cuda()
        xs = both[..., off:off + 24].detach().requires_grad_()
        y = bkcore.causal_conv(xs, w.cuda(), b.cuda(), "silu")
        dys = torch.empty(40, 3, 24, dtype=BF16, device="cuda").transpose(0, 1)
        dys.copy_(dy)
        y.backward(dys)
        assert_within(y, r["y"], r["ey"])
        assert_within(xs.grad, r["dx"], r["edx"])
    xc = x.cuda().transpose(1, 2).contiguous().transpose(1, 2)      # channels not innermost: copied
    assert_within(bkcore.causal_conv(xc, w.cuda(), b.cuda(), "silu"), r["y"], r["ey"])


@pytest.mark.parametrize("B,C,K,dtype", [(1, 1, 2, F32), (3, 17, 4, BF16), (5, 64, 3, F16), (64, 256, 4, BF16)])
def test_conv_steps_continue_a_prompt(B, C, K, dtype):
    import bkcore
    L, P = 9, 5
    x, w, b, _, _, _ = conv_inputs(B, L, C, K, dtype, seed=C)
    whole = bkcore.causal_conv(x.cuda(), w.cuda(), b.cuda(), "silu")
    y, state = bkcore.causal_conv(x[:, :P].cuda(), w.cuda(), b.cuda(), "silu", return_state=True)
    assert torch.equal(y, whole[:, :P])
    for t in range(P, L):
        yt = bkcore.causal_conv_step(x[:, t].cuda(), state, w.cuda(), b.cuda(), "silu")
        assert torch.equal(yt, whole[:, t])          # the same operations in the same order
    assert torch.equal(state.cpu(), x[:, L - K + 1:])


def test_conv_gradient_against_differences():
    import bkcore
    x, w, b, st, dy, df = conv_inputs(2, 11, 6, 4, F32, seed=5)
    ls = [leaf(t) for t in (x, w, b, st)]
    y, fin = bkcore.causal_conv(ls[0], ls[1], ls[2], "silu", None, ls[3], return_state=True)
    torch.autograd.backward([y, fin], [dy.cuda(), df.cuda()])

    def f(x, w, b, st):
        r = conv(x, w, b, True, None, st)
        return (r["y"] * d64(dy)).sum() + (r["final"] * d64(df)).sum()
    for i in range(4):
        got, fd, size = directional(f, list(d64(x, w, b, st)), [t.grad for t in ls], i, seed=i)
        assert abs(got - fd) <= 1e-5 * size + 1e-6


def test_conv_empty_and_refusals():
    import bkcore
    x, w, b, st, dy, df = (t.cuda() for t in conv_inputs(2, 6, 8, 4, BF16))
    s = st.clone().requires_grad_()
    wl = w.clone().requires_grad_()
    y, fin = bkcore.causal_conv(x[:, :0], wl, b, None, None, s, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(fin, st)
    fin.backward(df)
    assert torch.equal(s.grad, df) and (wl.grad == 0).all()
    with pytest.raises(ValueError):
        bkcore.causal_conv(x[0], w, b)
    with pytest.raises(ValueError):
        bkcore.causal_conv(x, w[:, :1], b)
    with pytest.raises(ValueError):
        bkcore.causal_conv(x, torch.cat([w, w[:, :1]], 1), b)
    with pytest.raises(ValueError):
        bkcore.causal_conv(x, w, b, "gelu")
    with pytest.raises(ValueError):
        bkcore.causal_conv(x, w, b[:7])
    with pytest.raises(ValueError):
        bkcore.causal_conv(x, w, b, initial_state=st[:, :2])
    with pytest.raises(TypeError):
        bkcore.causal_conv(x, w, b, initial_state=st.float())
    with pytest.raises(TypeError):
        bkcore.causal_conv(x, w.half(), b.half())
    with pytest.raises(TypeError):
        bkcore.causal_conv(x, w, b, lengths=torch.zeros(2, device="cuda"))
    with pytest.raises(RuntimeError, match="ROCm device"):
        bkcore.causal_conv(x, w, b, lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no gradient"):
        bkcore.causal_conv_step(x[:, 0], st, w.requires_grad_(), b)
    with torch.no_grad():
        with pytest.raises(ValueError):
            bkcore.causal_conv_step(x[:, 0], st.transpose(1, 2).contiguous().transpose(1, 2), w, b)
        with pytest.raises(ValueError):
            bkcore.causal_conv_step(x[:, 0], st[:, 1:], w, b)


# ------------------------------------------------------------------------------------------------------- selective scan

def scan_inputs(B, L, C, N, dtype, seed=0, step=0.1):
    """d is spread around `step`, so states forget over some tens of positions."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    bias = torch.log(torch.expm1(torch.full((C,), step) * torch.exp(0.5 * rn(C))))
    return dict(x=rn(B, L, C).to(dtype), delta=(0.5 * rn(B, L, C)).to(dtype), A=-(0.5 + 2 * torch.rand(C, N, generator=g)),
                Bm=rn(B, L, N).to(dtype), Cm=rn(B, L, N).to(dtype), D=rn(C), z=rn(B, L, C).to(dtype), bias=bias,
                h0=rn(B, C, N), dy=rn(B, L, C).to(dtype), dhT=rn(B, C, N))


NAMES = ("x", "delta", "A", "Bm", "Cm", "D", "z", "bias", "h0")
GRADS = ("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "dbias", "dh0")


def check_scan(v, lens=None, softplus=True, without=()):
    import bkcore
    ls = {k: None if k in without else leaf(v[k]) for k in NAMES}
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    y, hT = bkcore.selective_scan(ls["x"], ls["delta"], ls["A"], ls["Bm"], ls["Cm"], ls["D"], ls["z"], ls["bias"], softplus,
                                  n, ls["h0"], return_state=True)
    torch.autograd.backward([y, hT], [v["dy"].cuda(), v["dhT"].cuda()])
    a = {k: None if k in without else d64(v[k]) for k in NAMES}
    r = scan(a["x"], a["delta"], a["A"], a["Bm"], a["Cm"], a["D"], a["z"], a["bias"], softplus, lens, a["h0"],
             d64(v["dy"]), d64(v["dhT"]))
    assert y.dtype == v["x"].dtype and hT.dtype == F32
    assert_within(y, r["y"], r["ey"], "y")
    assert_within(hT, r["hT"], r["ehT"], "hT")
    for k, gk in zip(NAMES, GRADS):
        if ls[k] is not None:
            assert_within(ls[k].grad, r[gk], r["e" + gk], gk)


@pytest.mark.parametrize("B,L,C,N", [(1, 1, 1, 1), (2, 3, 5, 4), (1, 16, 64, 16), (2, 17, 65, 16), (1, 33, 16, 7),
                                     (2, 40, 33, 32), (1, 50, 20, 17), (1, 31, 17, 64), (2, 20, 9, 33), (3, 64, 130, 16)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scan_shapes(B, L, C, N, dtype):
    check_scan(scan_inputs(B, L, C, N, dtype, seed=L + C + N))


@pytest.mark.parametrize("L", [127, 128, 129, 400, 1023])       # few channels: the time axis is cut into chunks
@pytest.mark.parametrize("N", [4, 16, 20])
def test_scan_in_chunks(L, N):
    check_scan(scan_inputs(1, L, 6, N, F32, seed=L + N))


def test_scan_lengths_leave_padding_unread():
    lens = [0, 1, 15, 16, 17, 100, 128, 500, -3]
    v = scan_inputs(9, 130, 5, 16, BF16, seed=2)
    for i, n in enumerate(lens):
        for k in ("x", "delta", "z", "Bm", "Cm", "dy"):
            v[k][i, max(n, 0):] = float("nan") if k != "delta" else float("inf")
    check_scan(v, lens)


@pytest.mark.parametrize("without", [("D",), ("z",), ("bias",), ("h0",), ("D", "z", "bias", "h0")])
def test_scan_optional_operands(without):
    v = scan_inputs(2, 45, 12, 16, F32, seed=4)
    v["delta"] = v["delta"].abs() * 0.3
    check_scan(v, without=without)
    if "bias" in without:
        check_scan(v, softplus=False, without=without)


def test_scan_steps_of_every_size():
    # softplus from 1e-6 (its argument far below zero) to 30 (above the switch at 20), decays from 1 to 0
    v = scan_inputs(1, 64, 8, 16, F32, seed=6)
    v["bias"] = torch.tensor([-14.0, -8.0, -3.0, 0.0, 2.0, 8.0, 19.5, 25.0])
    check_scan(v)


def test_scan_strided_operands():
    import bkcore
    v = scan_inputs(2, 37, 24, 16, BF16, seed=8)
    r = scan(*d64(v["x"], v["delta"], v["A"], v["Bm"], v["Cm"], v["D"], v["z"], v["bias"]), True, None, None, d64(v["dy"]))
    xz = torch.cat([v["x"], v["z"]], -1).cuda()
    bc = torch.cat([torch.zeros(2, 37, 3, dtype=BF16), v["Bm"], v["Cm"]], -1).cuda()      # unaligned slices of a projection
    ls = [xz[..., :24].detach().requires_grad_(), v["delta"].cuda().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(),
          bc[..., 3:19].detach().requires_grad_(), bc[..., 19:].detach().requires_grad_(), xz[..., 24:].detach().requires_grad_()]
    y = bkcore.selective_scan(ls[0], ls[1], v["A"].cuda(), ls[2], ls[3], v["D"].cuda(), ls[4], v["bias"].cuda(), True)
    y.backward(v["dy"].cuda())
    assert_within(y, r["y"], r["ey"])
    for t, k in zip(ls, ("dx", "ddelta", "dB", "dC", "dz")):
        assert_within(t.grad, r[k], r["e" + k], k)


def test_scan_parameters_in_sixteen_bits():
    import bkcore
    v = scan_inputs(1, 20, 8, 16, BF16)
    A, D, bias = (v[k].to(BF16) for k in ("A", "D", "bias"))
    Al = A.cuda().requires_grad_()
    y = bkcore.selective_scan(v["x"].cuda(), v["delta"].cuda(), Al, v["Bm"].cuda(), v["Cm"].cuda(), D.cuda(), None,
                              bias.cuda(), True)
    y.backward(v["dy"].cuda())
    r = scan(*d64(v["x"], v["delta"], A, v["Bm"], v["Cm"], D), None, d64(bias), True, None, None, d64(v["dy"]))
    assert_within(y, r["y"], r["ey"])
    assert Al.grad.dtype == BF16
    assert_within(Al.grad, r["dA"], r["edA"])


@pytest.mark.parametrize("B,C,N,dtype", [(1, 1, 1, F32), (3, 7, 16, BF16), (2, 33, 20, F16), (4, 70, 64, BF16), (2, 5, 6, F32)])
def test_scan_steps_continue_a_prompt(B, C, N, dtype):
    import bkcore
    L, P = 12, 7
    v = scan_inputs(B, L, C, N, dtype, seed=C + N)
    r = scan(*d64(v["x"], v["delta"], v["A"], v["Bm"], v["Cm"], v["D"], v["z"], v["bias"]), True)
    dev = {k: t.cuda() for k, t in v.items()}
    y, state = bkcore.selective_scan(dev["x"][:, :P], dev["delta"][:, :P], dev["A"], dev["Bm"][:, :P], dev["Cm"][:, :P],
                                     dev["D"], dev["z"][:, :P], dev["bias"], True, return_state=True)
    assert_within(y, r["y"][:, :P], r["ey"][:, :P])
    for t in range(P, L):
        yt = bkcore.selective_scan_step(dev["x"][:, t], state, dev["delta"][:, t], dev["A"], dev["Bm"][:, t],
                                        dev["Cm"][:, t], dev["D"], dev["z"][:, t], dev["bias"], True)
        assert_within(yt, r["y"][:, t], r["ey"][:, t], f"token {t}")
    assert_within(state, r["hT"], r["ehT"], "state")


def test_scan_gradient_against_differences():
    import bkcore
    v = scan_inputs(2, 19, 5, 6, F32, seed=12)
    ls = [leaf(v[k]) for k in NAMES]
    y, hT = bkcore.selective_scan(*ls[:8], True, None, ls[8], return_state=True)
    torch.autograd.backward([y, hT], [v["dy"].cuda(), v["dhT"].cuda()])

    def f(x, delta, A, Bm, Cm, D, z, bias, h0):
        r = scan(x, delta, A, Bm, Cm, D, z, bias, True, None, h0)
        return (r["y"] * d64(v["dy"])).sum() + (r["hT"] * d64(v["dhT"])).sum()
    for i in range(9):
        got, fd, size = directional(f, [d64(v[k]) for k in NAMES], [t.grad for t in ls], i, seed=i)
        assert abs(got - fd) <= 5e-5 * size + 1e-6


def test_scan_repeats_and_replays_from_a_graph():
    import bkcore
    v = {k: t.cuda() for k, t in scan_inputs(2, 300, 40, 16, BF16, seed=1).items()}

    def step():
        ls = [v[k].detach().requires_grad_() for k in NAMES[:8]]
        y = bkcore.selective_scan(*ls, True)
        return (y, *torch.autograd.grad(y, ls, v["dy"]))
    first = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        for a, t in zip(step(), first):
            assert torch.equal(a, t)
        graph.replay()
        torch.cuda.synchronize()
        for a, t in zip(held, first):
            assert torch.equal(a, t)
    v["x"].mul_(-0.5)
    graph.replay()
    for a, t in zip(held, step()):
        assert torch.equal(a, t)


def test_scan_empty_and_refusals():
    import bkcore
    v = {k: t.cuda() for k, t in scan_inputs(2, 6, 8, 16, BF16).items()}
    op = [v[k] for k in NAMES[:8]]
    h0 = v["h0"].clone().requires_grad_()
    y, hT = bkcore.selective_scan(*(t[:, :0] if k in ("x", "delta", "Bm", "Cm", "z") else t for k, t in zip(NAMES, op)), True,
                                  None, h0, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(hT, v["h0"])
    hT.backward(v["dhT"])
    assert torch.equal(h0.grad, v["dhT"])

    def call(**kw):
        a = dict(zip(NAMES, op), h0=None, lengths=None)
        a.update(kw)
        return bkcore.selective_scan(a["x"], a["delta"], a["A"], a["Bm"], a["Cm"], a["D"], a["z"], a["bias"], True,
                                     a["lengths"], a["h0"])
    for bad in (dict(delta=v["delta"][:, :5]), dict(A=v["A"][:7]), dict(Bm=v["Bm"][..., :15]), dict(D=v["D"][:3]),
                dict(z=v["z"][:1]), dict(A=torch.zeros(8, 65, device="cuda")), dict(x=v["x"][0]),
                dict(h0=v["h0"][:, :4]), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(delta=v["delta"].float()), dict(Cm=v["Cm"].half()), dict(A=v["A"].double()), dict(h0=v["h0"].half())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(z=v["z"].cpu())
    step = [t[:, 0] if k in ("x", "delta", "Bm", "Cm", "z") else t for k, t in zip(NAMES, op)]
    with pytest.raises(TypeError):
        bkcore.selective_scan_step(step[0], v["h0"].half(), *step[1:], True)
    with pytest.raises(ValueError):
        bkcore.selective_scan_step(step[0], v["h0"].transpose(1, 2), *step[1:], True)
    with pytest.raises(RuntimeError, match="no gradient"):
        bkcore.selective_scan_step(step[0].clone().requires_grad_(), v["h0"], *step[1:], True)
