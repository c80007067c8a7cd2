"""Sliding-window attention with sinks on the GPU against its 64-bit definition: training, prompts, single tokens."""
import pytest
import torch

from mixer_reference import assert_within, attention, d64, directional, half_step

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def inputs(B, H, Hk, L, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype)
    return rn(B, H, L, D), rn(B, Hk, L, D), rn(B, Hk, L, D), rn(B, H, L, D)


def check(q, k, v, do, window, sinks, lens=None, scale=None, place=lambda t: t.cuda()):
    import bkcore
    ls = [place(t).detach().requires_grad_() for t in (q, k, v)]
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    o = bkcore.sliding_attention(*ls, window, sinks, scale=scale, lengths=n)
    o.backward(place(do))
    s = q.shape[-1] ** -0.5 if scale is None else scale
    r = attention(*d64(q, k, v), window, sinks, s, half_step(q.dtype), lens, d64(do))
    assert o.dtype == q.dtype
    assert_within(o, r["o"], r["eo"], "o")
    for t, name in zip(ls, ("dq", "dk", "dv")):
        assert_within(t.grad, r[name], r["e" + name], name)


# lengths around the tiles of 16, 32, 64 and 128; windows of one, inside a tile, across tiles, beyond the length
@pytest.mark.parametrize("L,window,sinks", [(1, 1, 0), (2, 5, 1), (15, 4, 2), (16, 16, 0), (33, 7, 3), (64, 1, 1), (65, 64, 64),
                                            (100, 33, 17), (128, 128, 0), (129, 20, 5), (200, 500, 4), (257, 31, 33),
                                            (300, 3, 64), (385, 1, 0), (400, 65, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_lengths_windows_sinks(L, window, sinks, dtype):
    check(*inputs(2, 2, 2, L, 32, dtype, seed=L), window, sinks)


@pytest.mark.parametrize("D", [1, 3, 8, 24, 31, 32, 40, 64, 65, 80, 94, 96, 128])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_head_dimensions(D, dtype):
    check(*inputs(1, 2, 1, 150, D, dtype, seed=D), 40, 3)


@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 1), (6, 2), (5, 5), (10, 2), (20, 1)])
def test_shared_heads(H, Hk):
    check(*inputs(2, H, Hk, 140, 64, BF16, seed=H), 50, 4)


@pytest.mark.parametrize("L,window,sinks,D", [(1500, 40, 5, 64), (1100, 100, 40, 32), (900, 8, 64, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_rest_behind_the_sinks(L, window, sinks, D, dtype):
    check(*inputs(1, 2, 1, L, D, dtype, seed=L), window, sinks)


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F32, 32), (F16, 20)])
def test_lengths_leave_padding_unread(dtype, D):
    lens = [0, 1, 63, 64, 65, 130, 300, 999, -4]
    q, k, v, do = inputs(9, 2, 1, 300, D, dtype, seed=3)
    for i, n in enumerate(lens):
        for t in (q, k, v, do):
            t[i, :, max(n, 0):] = float("nan")
    check(q, k, v, do, 37, 4, lens)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides(dtype):
    q, k, v, do = inputs(2, 4, 2, 90, 32, dtype, seed=5)
    # heads inside a position; a slice of a wider projection at an aligned and at an unaligned place; d not innermost
    check(q, k, v, do, 20, 2, place=lambda t: t.cuda().transpose(1, 2).contiguous().transpose(1, 2))

    def sliced(off):
        def f(t):
            wide = torch.full((*t.shape[:3], 48), float("nan"), dtype=t.dtype, device="cuda")
            wide[..., off:off + 32] = t.cuda()
            return wide[..., off:off + 32]
        return f
    check(q, k, v, do, 20, 2, place=sliced(8))
    check(q, k, v, do, 20, 2, place=sliced(3))
    check(q, k, v, do, 20, 2, place=lambda t: t.cuda().transpose(2, 3).contiguous().transpose(2, 3))
    check(q, q[:1].expand(2, -1, -1, -1)[:, :2], v, do, 20, 2, place=lambda t: t.cuda())


def test_an_expanded_gradient_and_one_fused_projection():
    import bkcore
    q, k, v, _ = inputs(2, 2, 2, 70, 16, F32, seed=6)
    qkv = torch.stack([q, k, v]).permute(1, 3, 0, 2, 4).contiguous().cuda().requires_grad_()     # (B, L, 3, H, D)
    a, b, c = qkv.permute(2, 0, 3, 1, 4)
    o = bkcore.sliding_attention(a, b, c, 9, 1)
    o.sum().backward()
    r = attention(*d64(q, k, v), 9, 1, 0.25, half_step(F32), None, torch.ones_like(q).double())
    for i, name in enumerate(("dq", "dk", "dv")):
        assert_within(qkv.grad[:, :, i].transpose(1, 2), r[name], r["e" + name], name)


def test_large_scores_and_scale():
    q, k, v, do = inputs(1, 2, 2, 130, 64, F32, seed=7)
    check(30 * q, 30 * k, v, do, 50, 3)              # scores in the thousands: the maximum is what keeps them finite
    check(q, k, v, do, 50, 3, scale=0.0)
    check(q, k, v, do, 50, 3, scale=-0.7)


def test_gradient_against_differences():
    import bkcore
    q, k, v, do = inputs(1, 4, 2, 40, 8, F32, seed=8)
    ls = [t.cuda().requires_grad_() for t in (q, k, v)]
    bkcore.sliding_attention(*ls, 11, 2).backward(do.cuda())

    def f(q, k, v):
        return (attention(q, k, v, 11, 2, 8 ** -0.5, 0.0)["o"] * d64(do)).sum()
    for i in range(3):
        got, fd, size = directional(f, list(d64(q, k, v)), [t.grad for t in ls], i, seed=i)
        assert abs(got - fd) <= 1e-5 * size + 1e-6


def test_repeats_and_replays_from_a_graph():
    import bkcore
    q, k, v, do = (t.cuda() for t in inputs(2, 4, 2, 700, 64, BF16, seed=9))

    def step():
        ls = [t.detach().requires_grad_() for t in (q, k, v)]
        o = bkcore.sliding_attention(*ls, 64, 4)
        return (o, *torch.autograd.grad(o, ls, do))
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
    q.mul_(0.5)
    graph.replay()
    for a, t in zip(held, step()):
        assert torch.equal(a, t)


# --------------------------------------------------------------------------------------------------------- single tokens

@pytest.mark.parametrize("B,H,Hk,D,window,sinks,spare", [(1, 1, 1, 32, 1, 0, 0), (2, 4, 2, 64, 5, 2, 0), (3, 8, 8, 32, 16, 4, 3),
                                                        (2, 20, 1, 128, 30, 1, 0), (1, 6, 2, 20, 300, 64, 0),
                                                        (2, 34, 2, 40, 140, 3, 7)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_steps_continue_a_prompt(B, H, Hk, D, window, sinks, spare, dtype):
    """Prompts of unequal lengths fill the cache, tokens follow; the outputs are those of the whole sequences."""
    import bkcore
    L, P = 60 if window < 100 else 420, [17, 3, 0, 40][:B] if window < 100 else [390, 2][:B]
    q, k, v, _ = inputs(B, H, Hk, L, D, dtype, seed=B + H)
    r = attention(*d64(q, k, v), window, sinks, D ** -0.5, half_step(dtype))
    cap = window + sinks + spare
    kc, vc = (torch.full((B, Hk, cap, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    n = torch.tensor(P, dtype=torch.int32, device="cuda")
    most = max(P)
    if most:
        bkcore.sliding_cache_fill(k[:, :, :most].cuda(), v[:, :, :most].cuda(), kc, vc, n, sinks)
    dev = [t.cuda() for t in (q, k, v)]
    rows = torch.arange(B)
    for step in range(20):
        at = torch.tensor([p + step for p in P])
        pos = at.to("cuda", torch.int64 if step % 2 else torch.int32)
        qt, kt, vt = (t[rows.cuda(), :, at.cuda()] for t in dev)
        o = bkcore.sliding_attention_step(qt, kt, vt, kc, vc, pos, window, sinks)
        assert_within(o, r["o"][rows, :, at], r["eo"][rows, :, at], f"token {step}")
    # what the caches hold: the last position of every slot, and the fill value where none came
    for b in range(B):
        want = {}
        for p in range(P[b] + 20):
            want[p if p < sinks else sinks + (p - sinks) % (cap - sinks)] = p
        for c, src in ((kc, k), (vc, v)):
            for slot in range(cap):
                exp = src[b, :, want[slot]] if slot in want else torch.full((Hk, D), 7.0, dtype=dtype)
                assert torch.equal(c[b, :, slot].cpu(), exp), (b, slot)


def test_inactive_sequences_are_left_alone():
    import bkcore
    q, k, v, _ = (t[:, :, 0].cuda() for t in inputs(3, 4, 2, 1, 64, BF16))
    kc, vc = (torch.randn(3, 2, 40, 64, device="cuda").to(BF16) for _ in range(2))
    k0, v0 = kc.clone(), vc.clone()
    o = bkcore.sliding_attention_step(q, k, v, kc, vc, torch.tensor([-1, 0, -7], device="cuda"), 36, 4)
    assert (o[0] == 0).all() and (o[2] == 0).all()
    assert torch.equal(o[1], v[1].repeat_interleave(2, 0))       # the first token sees itself alone
    for c, c0, new in ((kc, k0, k), (vc, v0, v)):
        c0[1, :, 0] = new[1]
        assert torch.equal(c, c0)


def test_caches_with_strides_and_nan_in_unused_slots():
    import bkcore
    B, H, Hk, D, W, S = 2, 4, 2, 32, 24, 4
    q, k, v, _ = inputs(B, H, Hk, 10, D, BF16, seed=11)
    r = attention(*d64(q, k, v), W, S, D ** -0.5, half_step(BF16))
    store = torch.full((B, W + S, 2, Hk, D + 8), float("nan"), dtype=BF16, device="cuda")       # slots outside, heads inside
    kc, vc = (store[:, :, i, :, :D].transpose(1, 2) for i in range(2))
    for t in range(10):
        pos = torch.full((B,), t, dtype=torch.int32, device="cuda")
        o = bkcore.sliding_attention_step(*(x[:, :, t].cuda() for x in (q, k, v)), kc, vc, pos, W, S)
        assert_within(o, r["o"][:, :, t], r["eo"][:, :, t], f"token {t}")
    assert torch.isnan(store[..., D:]).all()


def test_step_replays_from_a_graph_with_moving_positions():
    import bkcore
    B, H, Hk, D, W, S = 2, 8, 2, 64, 700, 4
    q, k, v, _ = (t.cuda() for t in inputs(B, H, Hk, 40, D, BF16, seed=12))
    kc, vc = (torch.zeros(B, Hk, W + S, D, dtype=BF16, device="cuda") for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    qt, kt, vt = (t[:, :, 0].clone() for t in (q, k, v))
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bkcore.sliding_attention_step(qt, kt, vt, kc, vc, pos, W, S)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = bkcore.sliding_attention_step(qt, kt, vt, kc, vc, pos, W, S)
    for t in range(40):
        for dst, src in ((qt, q), (kt, k), (vt, v)):
            dst.copy_(src[:, :, t])
        pos.fill_(t)
        graph.replay()
        eager = bkcore.sliding_attention_step(qt, kt, vt, want_k, want_v, pos, W, S)
        assert torch.equal(held, eager) and torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_empty_and_refusals():
    import bkcore
    q, k, v, do = (t.cuda() for t in inputs(2, 4, 2, 8, 16, BF16))
    e = q[:, :, :0].requires_grad_()
    o = bkcore.sliding_attention(e, k[:, :, :0], v[:, :, :0], 4)
    assert o.shape == (2, 4, 0, 16)
    o.sum().backward()
    assert bkcore.sliding_attention(q[:0], k[:0], v[:0], 4).shape == (0, 4, 8, 16)
    call = bkcore.sliding_attention
    for bad in ((q, k[:, :, :7], v), (q, k, v[:, :1]), (q[:1], k, v), (q[:, :3], k, v), (q[0], k[0], v[0]),
                (q[..., :8], k, v)):
        with pytest.raises(ValueError):
            call(*bad, 4)
    with pytest.raises(ValueError):
        call(q, k, v, 0)
    with pytest.raises(ValueError):
        call(q, k, v, 4, 65)
    with pytest.raises(ValueError):
        call(q, k, v, 4, -1)
    with pytest.raises(ValueError):
        call(q, k, v, 4, scale=float("nan"))
    with pytest.raises(ValueError):
        call(*(torch.zeros(1, 1, 4, 129, device="cuda") for _ in range(3)), 4)
    with pytest.raises(TypeError):
        call(q, k.float(), v, 4)
    with pytest.raises(TypeError):
        call(q.double(), k.double(), v.double(), 4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(q, k.cpu(), v, 4)
    g = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(call(g, k, v, 4).float().sum(), g, create_graph=True)
    qs, ks, vs = q[:, :, 0], k[:, :, 0], v[:, :, 0]
    kc = torch.zeros(2, 2, 12, 16, dtype=BF16, device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    step = bkcore.sliding_attention_step
    for bad in ((kc[:, :, :5], kc, pos, 4, 2), (kc, kc, pos, 12, 1), (kc[:, :1], kc[:, :1], pos, 4, 2),
                (kc, kc, pos[:1], 4, 2), (kc[..., :8], kc[..., :8], pos, 4, 2), (kc, kc, pos, 0, 2),
                (kc[:, :, :1].expand(-1, -1, 12, -1), kc, pos, 4, 2), (kc.transpose(2, 3), kc.transpose(2, 3), pos, 4, 2)):
        with pytest.raises(ValueError):
            step(qs, ks, vs, *bad)
    with pytest.raises(TypeError):
        step(qs, ks, vs, kc.float(), kc.float(), pos, 4, 2)
    with pytest.raises(TypeError):
        step(qs, ks, vs, kc, kc.clone(), pos.float(), 4, 2)
    with pytest.raises(RuntimeError, match="ROCm device"):
        step(qs, ks, vs, kc, kc.clone(), pos.cpu(), 4, 2)
    with pytest.raises(RuntimeError, match="no gradient"):
        step(qs.clone().requires_grad_(), ks, vs, kc, kc.clone(), pos, 4, 2)
    with pytest.raises(ValueError):
        bkcore.sliding_cache_fill(k, v, kc[:, :, :4], kc[:, :, :4], None, 4)
    with pytest.raises(TypeError):
        bkcore.sliding_cache_fill(k, v, kc.float(), kc.float())


def test_caches_that_share_memory_are_refused():
    import bkcore
    q, k, v, _ = (t.cuda() for t in inputs(2, 4, 2, 8, 16, BF16))
    qs, ks, vs = q[:, :, 0], k[:, :, 0], v[:, :, 0]
    kc, vc = (torch.zeros(2, 2, 12, 16, dtype=BF16, device="cuda") for _ in range(2))
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    shared = (kc[:1].expand(2, -1, -1, -1), kc[:, :1].expand(-1, 2, -1, -1),
              kc.view(-1).as_strided((2, 2, 12, 16), (200, 192, 16, 1)))
    for a, b in [(kc, kc)] + [(c, vc) for c in shared] + [(vc, c) for c in shared]:
        with pytest.raises(ValueError):
            bkcore.sliding_attention_step(qs, ks, vs, a, b, pos, 4, 2)
        with pytest.raises(ValueError):
            bkcore.sliding_cache_fill(k, v, a, b)
    both = torch.zeros(2, 12, 2, 2, 16, dtype=BF16, device="cuda")       # keys and values side by side in a slot
    a, b = both.permute(3, 0, 2, 1, 4)
    got = bkcore.sliding_attention_step(qs, ks, vs, a, b, pos, 4, 2)
    assert torch.equal(got, vs.repeat_interleave(2, 1)) and torch.equal(a[:, :, 0], ks) and torch.equal(b[:, :, 0], vs)


@pytest.mark.parametrize("position", [2 ** 31 - 2, 2 ** 31 - 1])
def test_step_at_the_last_positions(position):
    """Two slots behind two sinks: the token itself and the one in front of it, next to the sinks."""
    import bkcore
    q, k, v, _ = (t.cuda() for t in inputs(1, 2, 2, 4, 16, torch.float32))
    kc, vc = (torch.empty(1, 2, 4, 16, device="cuda") for _ in range(2))
    at = [0, 1, 2 + (position - 3) % 2, 2 + (position - 2) % 2]
    kc[:, :, at], vc[:, :, at] = k, v
    kc[:, :, at[3]], vc[:, :, at[3]] = float("nan"), float("nan")
    pos = torch.tensor([position], dtype=torch.int64, device="cuda")
    got = bkcore.sliding_attention_step(q[:, :, 3], k[:, :, 3], v[:, :, 3], kc, vc, pos, 2, 2)
    want = attention(*d64(q, k, v), 4, 0, 16 ** -0.5, half_step(torch.float32))
    assert_within(got, want["o"][:, :, 3], want["eo"][:, :, 3])
    assert torch.equal(kc[:, :, at], k) and torch.equal(vc[:, :, at], v)
