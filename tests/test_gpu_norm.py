"""Layer norm on the GPU against its 64-bit definition: forward, backward, odd widths, strides, refusals."""
import pytest
import torch

from mixer_reference import assert_within, d64, directional, norm

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def make(rows, D, dtype, seed=0, params="f32", shift=0.5):
    g = torch.Generator().manual_seed(seed)
    p = torch.float32 if params == "f32" else dtype
    x = (1.5 * torch.randn(rows, D, generator=g) + shift).to(dtype)
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(p)
    b = (0.3 * torch.randn(D, generator=g)).to(p)
    dy = torch.randn(rows, D, generator=g).to(dtype)
    return x, w, b, dy


def check(x, w, b, dy, eps=1e-5, view=lambda t: t):
    import bkcore
    leaves = [None if t is None else view(t.cuda()).detach().requires_grad_() for t in (x, w, b)]
    if w is not None:
        leaves[1] = w.cuda().requires_grad_()
    if b is not None:
        leaves[2] = b.cuda().requires_grad_()
    y = bkcore.layer_norm(*leaves, eps=eps)
    y.backward(view(dy.cuda()))
    ref = norm(*d64(x, w, b), eps, d64(dy))
    assert y.dtype == x.dtype
    assert_within(y, *ref[0], "y")
    assert_within(leaves[0].grad, *ref[1], "dx")
    if w is not None:
        assert leaves[1].grad.dtype == w.dtype
        assert_within(leaves[1].grad, *ref[2], "dw")
    if b is not None:
        assert_within(leaves[2].grad, *ref[3], "db")


# widths on both sides of every variant's border, odd ones and one that breaks 16-byte alignment
@pytest.mark.parametrize("D", [1, 2, 7, 64, 255, 256, 512, 513, 1000, 1024, 1025, 2048, 2056, 4096, 4097, 8192, 8200, 16384])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_widths(D, dtype):
    check(*make(5, D, dtype, seed=D))


@pytest.mark.parametrize("rows", [1, 3, 4, 17, 2048, 4099])
def test_rows(rows):
    check(*make(rows, 96, torch.float32, seed=rows))
    check(*make(rows, 96, torch.bfloat16, seed=rows, params="own"))


@pytest.mark.parametrize("which", ["weight", "bias", "neither"])
def test_without_parameters(which):
    x, w, b, dy = make(6, 130, torch.float16)
    check(x, None if which != "weight" else w, None if which != "bias" else b, dy)


def test_large_mean_keeps_the_centred_variance():
    # mean 1000 times the spread: E[x^2] - mean^2 in float32 would lose every digit of the variance
    check(*make(8, 300, torch.float32, shift=1500.0))


@pytest.mark.parametrize("D", [48, 51])
def test_strided_rows_and_more_dimensions(D):
    import bkcore
    x, w, b, dy = make(12, D, torch.bfloat16, seed=3)
    wide = torch.zeros(12, D + 5, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:2 + D] = x.cuda()                       # rows neither contiguous nor aligned
    ref = norm(*d64(x, w, b), 1e-5, d64(dy))
    xs = wide[:, 2:2 + D].detach().requires_grad_()
    y = bkcore.layer_norm(xs, w.cuda(), b.cuda())
    y.backward(dy.cuda())
    assert_within(y, *ref[0], "y")
    assert_within(xs.grad, *ref[1], "dx")
    x3 = x.view(3, 4, D).cuda().transpose(0, 1).detach().requires_grad_()   # rows in another order
    y3 = bkcore.layer_norm(x3, w.cuda(), b.cuda())
    assert y3.shape == (4, 3, D)
    assert_within(y3.transpose(0, 1).reshape(12, D), *ref[0], "y of a transposed view")
    y3.sum().backward()                                # an expanded gradient
    assert x3.grad.shape == x3.shape
    xt = x.t().contiguous().t().cuda()                 # the last dimension strided
    assert_within(bkcore.layer_norm(xt, w.cuda(), b.cuda()), *ref[0], "y of a column-major input")


def test_gradient_against_differences():
    import bkcore
    x, w, b, dy = make(7, 33, torch.float32, seed=9)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    bkcore.layer_norm(*leaves).backward(dy.cuda())

    def f(x, w, b):
        return (norm(x, w, b, 1e-5)[0] * d64(dy)).sum()
    args = list(d64(x, w, b))
    for i in range(3):
        got, fd, size = directional(f, args, [t.grad for t in leaves], i, seed=i)
        assert abs(got - fd) <= 1e-5 * size + 1e-6     # 100 float32 half steps of the terms, 1e-6 of the difference quotient


def test_a_row_with_nan_or_infinity_stays_alone():
    import bkcore
    x, w, b, dy = make(9, 200, torch.float32)
    x[2, 5] = float("nan")
    x[6, 7] = float("inf")
    ref = norm(*d64(x, w, b), 1e-5)
    y = bkcore.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    keep = [i for i in range(9) if i not in (2, 6)]
    assert_within(y[keep], ref[0][keep], ref[1][keep])
    assert torch.isnan(y[2]).all() and torch.isnan(y[6]).all()


def test_constant_rows_and_no_rows():
    import bkcore
    x = torch.full((4, 64), 3.25, device="cuda", requires_grad=True)
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.full((64,), 0.5, device="cuda", requires_grad=True)
    y = bkcore.layer_norm(x, w, b)
    assert (y == 0.5).all()
    y.sum().backward()
    assert torch.isfinite(x.grad).all() and (w.grad == 0).all() and (b.grad == 4).all()
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    w.grad = None
    z = bkcore.layer_norm(e, w)
    assert z.shape == (0, 64)
    z.sum().backward()
    assert (w.grad == 0).all() and e.grad.shape == (0, 64)


def test_results_repeat_and_replay_from_a_graph():
    import bkcore
    x, w, b, dy = (t.cuda() for t in make(3000, 256, torch.bfloat16))

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = bkcore.layer_norm(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))
    first = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        for a, t in zip(step(), first):
            assert torch.equal(a, t)
        graph.replay()
        torch.cuda.synchronize()
        for a, t in zip(held, first):
            assert torch.equal(a, t)
    x.mul_(0.5)
    graph.replay()
    for a, t in zip(held, step()):
        assert torch.equal(a, t)


def test_module_has_the_tensor_librarys_parameters():
    import bkcore
    ref = torch.nn.LayerNorm(40, eps=1e-4).cuda()
    with torch.no_grad():
        ref.weight.normal_()
        ref.bias.normal_()
    own = bkcore.LayerNorm(40, eps=1e-4).cuda()
    own.load_state_dict(ref.state_dict())
    x = torch.randn(3, 5, 40, device="cuda")
    want = norm(*d64(x, ref.weight, ref.bias), 1e-4)
    assert_within(own(x), *want)
    assert bkcore.LayerNorm(40, bias=False).cuda()(x).shape == x.shape
    with pytest.raises(ValueError):
        own(x[..., :39])
    with pytest.raises(ValueError):
        bkcore.LayerNorm((4, 40))


def test_refusals():
    import bkcore
    x = torch.zeros(2, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    with pytest.raises(RuntimeError, match="ROCm device"):
        bkcore.layer_norm(x, w.cpu())
    with pytest.raises(TypeError):
        bkcore.layer_norm(x.double())
    with pytest.raises(TypeError):
        bkcore.layer_norm(x, w.half())
    with pytest.raises(TypeError):
        bkcore.layer_norm(x.half(), w.half(), w)
    with pytest.raises(ValueError):
        bkcore.layer_norm(x, w[:7])
    with pytest.raises(ValueError):
        bkcore.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        bkcore.layer_norm(torch.zeros(2, 16385, device="cuda"))
    with pytest.raises(ValueError):
        bkcore.layer_norm(torch.zeros(2, 0, device="cuda"))
    with pytest.raises(ValueError):
        bkcore.layer_norm(torch.zeros((), device="cuda"))
