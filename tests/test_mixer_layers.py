"""The layer operators where the package uses them: the hybrid layer's sliding and selective paths, the kernel layer norm,
the small LM built of them, prompts followed by single tokens."""
import pytest
import torch
import torch.nn.functional as F


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def test_default_layers_keep_their_state_dicts():
    from bkcore.layers import BKHybridLayer
    from bkcore.lm import SmallResNetBKLM
    old = {"v_proj.weight", "v_proj.bias", "output_proj.weight", "output_proj.bias", "bk_scale", "gamma", "epsilon_param",
           "h0_diag_base", "h0_sub_base", "h0_super_base", "hybrid_attn.gate_sensitivity", "hybrid_attn.layer_norm.weight",
           "hybrid_attn.layer_norm.bias", "local_qkv.weight", "local_out.weight", "global_in.weight", "global_out.weight",
           "global_out.bias"}
    assert set(BKHybridLayer(32, 16, num_heads=4).state_dict()) == old
    new = set(BKHybridLayer(32, 16, num_heads=4, local="sliding", sinks=2, norm="kernel").state_dict())
    assert new == old                                            # the same parameters, other operators
    sel = set(BKHybridLayer(32, 16, num_heads=4, global_path="selective").state_dict())
    assert {k for k in sel if k.startswith("selective.")} == {"selective." + n for n in (
        "in_proj.weight", "conv_weight", "conv_bias", "x_proj.weight", "dt_proj.weight", "dt_proj.bias", "A_log", "D",
        "out_proj.weight")}
    a = SmallResNetBKLM(50, 16, 1, 8)
    b = SmallResNetBKLM(50, 16, 1, 8, norm="kernel")
    assert list(a.state_dict()) == list(b.state_dict())


def test_refusals():
    from bkcore.layers import BKHybridLayer
    from bkcore.lm import SmallResNetBKLM
    for kw in (dict(local="ring"), dict(global_path="max"), dict(norm="rms"), dict(sinks=2)):
        with pytest.raises(ValueError):
            BKHybridLayer(32, 16, num_heads=4, **kw)
    with pytest.raises(ValueError):
        SmallResNetBKLM(50, 16, 1, 8, local="sliding")           # without hybrid=True there is no local path
    with pytest.raises(ValueError):
        BKHybridLayer(32, 16, num_heads=4).new_local_cache(1, "cpu")


def plain_sliding(layer, x):
    B, N, D = x.shape
    q, k, v = layer._heads(x)
    i, j = torch.arange(N, device=x.device)[:, None], torch.arange(N, device=x.device)[None]
    see = (j <= i) & ((i - j < layer.window) | (j < layer.sinks))
    p = torch.softmax((q @ k.transpose(-1, -2).contiguous() * (D // layer.num_heads) ** -0.5).masked_fill(~see, float("-inf")), -1)
    return layer.local_out((p @ v).transpose(1, 2).reshape(B, N, D))


def plain_selective(m, x):
    v, z = m.in_proj(x).chunk(2, -1)
    K = m.conv_width
    u = F.silu(F.conv1d(F.pad(v.transpose(1, 2), (K - 1, 0)), m.conv_weight[:, None], m.conv_bias, groups=m.d_inner)).transpose(1, 2)
    delta, B, C = m._projections(u)
    d = F.softplus(delta + m.dt_proj.bias)
    A = -torch.exp(m.A_log)
    h, ys = torch.zeros(x.shape[0], m.d_inner, m.d_state, dtype=x.dtype, device=x.device), []
    for t in range(x.shape[1]):
        h = torch.exp(d[:, t, :, None] * A) * h + (d[:, t] * u[:, t])[..., None] * B[:, t, None]
        ys.append((h * C[:, t, None]).sum(-1) + m.D * u[:, t])
    return m.out_proj(torch.stack(ys, 1) * F.silu(z))


def close(got, want, what, tol):
    """Largest difference against the largest value: the chains behind these are float32 against float64, some hundred
    roundings of 2^-24 each."""
    got, want = got.detach().double().cpu(), want.detach().cpu()
    err = float((got - want).abs().max() / want.abs().max().clamp_min(1e-30))
    assert err <= tol, (what, err)


@pytest.mark.gpu
def test_selective_mixer_and_its_gradients():
    need_gpu()
    import bkcore
    torch.manual_seed(0)
    m = bkcore.SelectiveMixer(24, d_inner=40, d_state=8).cuda()
    ref = bkcore.SelectiveMixer(24, d_inner=40, d_state=8).double()
    ref.load_state_dict(m.state_dict())
    x = torch.randn(2, 70, 24)
    g = torch.randn(2, 70, 24)
    xr, xg = x.double().requires_grad_(), x.cuda().requires_grad_()
    want, got = plain_selective(ref, xr), m(xg)
    want.backward(g.double())
    got.backward(g.cuda())
    close(got, want, "y", 300 * 2.0 ** -24)
    close(xg.grad, xr.grad, "dx", 1000 * 2.0 ** -24)
    for (n, p), (_, r) in zip(m.named_parameters(), ref.named_parameters()):
        close(p.grad, r.grad, n, 2000 * 2.0 ** -24)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(8, 2), (200, 0)])
def test_sliding_local_path_and_its_gradients(window, sinks):
    need_gpu()
    from bkcore.layers import BKHybridLayer
    torch.manual_seed(1)
    m = BKHybridLayer(64, 90, num_heads=4, window=window, local="sliding", sinks=sinks).cuda()
    ref = BKHybridLayer(64, 90, num_heads=4, window=window, local="sliding", sinks=sinks).double()
    ref.load_state_dict(m.state_dict())
    x, g = torch.randn(2, 90, 64), torch.randn(2, 90, 64)
    xr, xg = x.double().requires_grad_(), x.cuda().requires_grad_()
    want, got = plain_sliding(ref, xr), m.local_path(xg)
    want.backward(g.double())
    got.backward(g.cuda())
    close(got, want, "y", 300 * 2.0 ** -24)
    close(xg.grad, xr.grad, "dx", 1000 * 2.0 ** -24)
    for n in ("local_qkv", "local_out"):
        close(getattr(m, n).weight.grad, getattr(ref, n).weight.grad, n, 2000 * 2.0 ** -24)


@pytest.mark.gpu
def test_prompts_then_single_tokens_through_both_paths():
    """A padded batch of prompts, then tokens one at a time: what the whole sequences give."""
    need_gpu()
    from bkcore.layers import BKHybridLayer
    torch.manual_seed(2)
    B, N, D, lens = 3, 40, 64, [17, 30, 5]
    m = BKHybridLayer(D, N, num_heads=4, window=12, local="sliding", sinks=3, global_path="selective").cuda()
    x = torch.randn(B, N, D, device="cuda")
    with torch.no_grad():
        local, glob = m.local_path(x), m.selective(x)
        P = max(lens)
        n = torch.tensor(lens, device="cuda")
        cache = m.new_local_cache(B, "cuda")
        lp = m.local_prefill(x[:, :P], cache, n)
        gp, state = m.selective(x[:, :P], n, m.selective.new_state(B, "cuda"), return_state=True)
        for b, k in enumerate(lens):
            close(lp[b, :k], local[b, :k].double(), "local prompt", 300 * 2.0 ** -24)
            close(gp[b, :k], glob[b, :k].double(), "global prompt", 300 * 2.0 ** -24)
        rows = torch.arange(B, device="cuda")
        for t in range(10):
            at = n + t
            lo = m.local_step(x[rows, at], cache, at)
            go = m.selective.step(x[rows, at], state)
            close(lo, local[rows, at].double(), f"local token {t}", 300 * 2.0 ** -24)
            close(go, glob[rows, at].double(), f"global token {t}", 300 * 2.0 ** -24)


def lm(kernels, **kw):
    from bkcore.lm import SmallResNetBKLM
    torch.manual_seed(3)
    extra = dict(norm="kernel", local="sliding", sinks=2, global_path="selective") if kernels else {}
    return SmallResNetBKLM(101, 64, 2, 48, hybrid=True, **extra, **kw).cuda()


@pytest.mark.gpu
def test_kernel_norm_gives_the_tensor_librarys_gradients():
    need_gpu()
    from bkcore.lm import SmallResNetBKLM
    grads = []
    for norm in ("torch", "kernel"):
        torch.manual_seed(4)
        m = SmallResNetBKLM(101, 64, 2, 48, norm=norm).cuda()
        g = torch.Generator(device="cuda").manual_seed(5)
        tok, tgt = (torch.randint(0, 101, (3, 48), device="cuda", generator=g) for _ in range(2))
        F.cross_entropy(m(tok).flatten(0, 1), tgt.flatten()).backward()
        grads.append({n: p.grad for n, p in m.named_parameters() if p.grad is not None})
    assert set(grads[0]) == set(grads[1])
    for n in grads[0]:
        if "bk_layer.v_proj" not in n:        # that gradient passes through bfloat16 operands: last-bit inputs move whole steps
            close(grads[1][n], grads[0][n].double(), n, 1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [False, True])
def test_lm_of_kernels_trains_and_replays_from_a_graph(autocast):
    """Two layers of all operators together: gradients finite and present everywhere, the captured step equal to the eager one."""
    need_gpu()
    from bkcore.lm import training_step
    g = torch.Generator(device="cuda").manual_seed(6)
    tok, tgt = (torch.randint(0, 101, (3, 48), device="cuda", generator=g) for _ in range(2))

    def run(capture):
        m = lm(True)
        opt = torch.optim.SGD(m.parameters(), lr=0.05)

        def step():
            with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
                return training_step(m, opt, tok, tgt)
        if capture:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
        else:
            step()
        unused = ("output_proj", "bk_scale", "gamma", "epsilon_param")    # off the hybrid path; z gets no gradient
        for n, p in m.named_parameters():
            if not any(u in n.split(".") for u in unused):
                assert p.grad is not None and torch.isfinite(p.grad).all(), n
        if capture:
            opt.zero_grad(set_to_none=True)
            for blk in m.blocks:
                blk.bk_layer.last_g_ii = None      # it holds the warm-up's autograd graph, whose leaves the capture shares
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                loss = step()
            losses = []
            for _ in range(3):
                graph.replay()
                torch.cuda.synchronize()
                losses.append(float(loss))
        else:
            losses = [float(step()) for _ in range(3)]
        return losses, [p.detach().clone() for p in m.parameters()]
    eager, captured = run(False), run(True)
    for a, b in zip(eager[1], captured[1]):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-5)   # library products may take other kernels under capture


@pytest.mark.gpu
def test_calls_on_two_streams_at_once_do_not_meet():
    """Every operator, forward and backward, on two streams with data of their own: the results of the calls alone."""
    need_gpu()
    import bkcore

    def data(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
        return dict(x=rn(2, 900, 96), w=rn(96), cw=rn(96, 4), A=-rn(96, 16).abs(), B=rn(2, 900, 16), C=rn(2, 900, 16),
                    q=rn(2, 6, 900, 32), k=rn(2, 3, 900, 32), v=rn(2, 3, 900, 32))

    def work(d):
        t = {n: v.detach().requires_grad_() for n, v in d.items()}
        y = bkcore.layer_norm(t["x"], t["w"])
        u = bkcore.causal_conv(y, t["cw"], None, "silu")
        s = bkcore.selective_scan(u, 0.1 * y, t["A"], t["B"], t["C"], delta_softplus=True)
        o = bkcore.sliding_attention(t["q"], t["k"], t["v"], 40, 4)
        grads = torch.autograd.grad([s.sum() + (o * o).sum()], list(t.values()))
        return [s.detach(), o.detach(), *grads]
    inputs = [data(1), data(2)]
    alone = [work(d) for d in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    both = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                both[i] = work(inputs[i])
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_changed_inputs_are_noticed_by_the_backward():
    need_gpu()
    import bkcore
    x = torch.randn(4, 32, device="cuda", requires_grad=True)
    h = x * 1.0
    y = bkcore.layer_norm(h)
    h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
