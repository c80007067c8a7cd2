"""The operators of the hybrid mixing layer as workloads: sliding-window attention with sinks, the short causal
convolution, the selective state space scan and layer norm, each in a plain form (elementary tensor operations in 32 bits,
rounded once at the end) and as the calls a user makes of ``bkcore``.

``listed()`` gives the cases, ``draw(rng)`` further ones of the same ranges, ``prepare(case, seed)`` what a program has in
hand before the call, ``run(state)`` one pass, ``work(case)`` the bytes and operations the pass cannot do without, and
``exact(case, seed)`` the same outputs from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _bkcore():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "project-resnet-bk-an-o-n-language-model-architecture_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import bkcore
    return bkcore


# ----------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # the small LM's blocks (batch 8, 256 positions, width 256) in training: launches dominate
        dict(name="norm_small_train_f32", op="norm", rows=2048, dim=256, dtype="f32", train=True),
        # pre-norm of a larger model's training step
        dict(name="norm_train_bf16", op="norm", rows=16384, dim=2048, dtype="bf16", train=True),
        # a serving batch with an odd width, forward only
        dict(name="norm_odd_f16", op="norm", rows=4099, dim=1537, dtype="f16", train=False),
        # the convolution in front of the scan, training; x is a slice of the wider input projection
        dict(name="conv_train_bf16", op="conv", batch=8, length=2048, dim=1024, width=4, act="silu", dtype="bf16",
             ragged=False, train=True),
        # the same for one token of each sequence of a serving batch: latency
        dict(name="conv_step_bf16", op="conv_step", batch=64, dim=1024, width=4, act="silu", dtype="bf16"),
        # training pass of the selective mixer
        dict(name="scan_train_bf16", op="scan", batch=4, length=2048, dim=1024, state=16, dtype="bf16", ragged=False,
             train=True),
        # one long prompt: few channels, a long axis; the state is kept for the tokens that follow
        dict(name="scan_prompt_f32", op="scan", batch=1, length=8191, dim=512, state=16, dtype="f32", ragged=False,
             train=False),
        # one token of each sequence of a serving batch
        dict(name="scan_step_bf16", op="scan_step", batch=256, dim=2048, state=16, dtype="bf16"),
        # local path of the small LM: 8 heads of 32, windows of 32, training in 32 bits
        dict(name="attn_small_train_f32", op="attn", batch=8, heads=8, kv_heads=8, length=256, dim=32, window=32, sinks=4,
             dtype="f32", ragged=False, train=True),
        # long-context training with shared key/value heads
        dict(name="attn_long_train_bf16", op="attn", batch=2, heads=16, kv_heads=4, length=8192, dim=128, window=1024,
             sinks=4, dtype="bf16", ragged=False, train=True),
        # prompts of unequal lengths in one padded batch
        dict(name="attn_prompt_ragged_f16", op="attn", batch=4, heads=8, kv_heads=8, length=3001, dim=64, window=500,
             sinks=3, dtype="f16", ragged=True, train=False),
        # one token of each sequence of a serving batch: the rolling cache is read once
        dict(name="attn_step_bf16", op="attn_step", batch=64, heads=32, kv_heads=8, dim=128, window=4096, sinks=4,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        op = rng.choice(["norm", "conv", "conv_step", "scan", "scan_step", "attn", "attn", "attn_step"])
        if op == "norm":
            case = dict(op=op, rows=_log(rng, 1, 65536), dim=_log(rng, 1, 8192), dtype=dtype, train=rng.random() < 0.6)
        elif op == "conv":
            case = dict(op=op, batch=_log(rng, 1, 16), length=_log(rng, 1, 8192), dim=_log(rng, 1, 4096),
                        width=rng.randint(2, 4), act=rng.choice(["silu", "none"]), dtype=dtype,
                        ragged=rng.random() < 0.4, train=rng.random() < 0.6)
        elif op == "conv_step":
            case = dict(op=op, batch=_log(rng, 1, 512), dim=_log(rng, 1, 4096), width=rng.randint(2, 4),
                        act=rng.choice(["silu", "none"]), dtype=dtype)
        elif op == "scan":
            case = dict(op=op, batch=_log(rng, 1, 8), length=_log(rng, 1, 16384), dim=_log(rng, 1, 4096),
                        state=rng.choice([16, 16, _log(rng, 1, 64)]), dtype=dtype, ragged=rng.random() < 0.4,
                        train=rng.random() < 0.6)
            if case["batch"] * case["length"] * case["dim"] * case["state"] > 4 * 2048 * 1024 * 16:
                continue
        elif op == "scan_step":
            case = dict(op=op, batch=_log(rng, 1, 512), dim=_log(rng, 1, 4096), state=rng.choice([16, _log(rng, 1, 64)]),
                        dtype=dtype)
            if case["batch"] * case["dim"] * case["state"] > 1 << 25:
                continue
        else:
            kv = rng.choice([1, 2, 4, 8])
            dim = rng.choice([32, 64, 128, rng.randint(1, 16) * 8, rng.randint(1, 128)])
            case = dict(op=op, batch=_log(rng, 1, 8), heads=kv * rng.choice([1, 1, 2, 4, 5]), kv_heads=kv,
                        length=_log(rng, 1, 8192), dim=dim, window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 16, 64]),
                        dtype=dtype, ragged=rng.random() < 0.4, train=rng.random() < 0.6)
            if op == "attn_step":
                case = {k: case[k] for k in ("op", "batch", "heads", "kv_heads", "dim", "window", "sinks", "dtype")}
                case["batch"] = _log(rng, 1, 64)
            elif case["dtype"] == "f32":       # a quarter of the length: 32-bit products run at a small part of the rate
                case["length"] = max(1, case["length"] // 4)
        big = [work(c) for c in listed()]
        w = work(case)
        if w["bytes"] <= max(b["bytes"] for b in big) and w["flops"] <= max(b["flops"] for b in big):
            return case


def _lengths(case):
    """Lengths of a padded batch, from the case alone: the first sequence fills it, the others fall off unevenly."""
    B, L = case["batch"], case["length"]
    return [max(0, L - (b * (L + 3)) // (B + 1)) if case.get("ragged") else L for b in range(B)]


def _positions(case):
    """Position of each sequence's new token: from an early one to well past the window."""
    span = case["window"] + case["sinks"]
    return [max(0, span + 17 * b - (span // 2 if b % 4 == 3 else 0)) for b in range(case["batch"])]


def _visible_pairs(L, W, S):
    """sum over i < L of the number of keys that query i sees"""
    total = 0
    for i in range(L):
        lo = max(0, i - W + 1)
        total += i - lo + 1 + min(S, lo)
    return total


def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    if op == "norm":
        n = case["rows"] * case["dim"]
        by, fl = 2 * e * n + 8 * case["dim"], 8 * n
        if case["train"]:                     # the forward's read and write; x and dy once more, dx
            by += 3 * e * n + 8 * case["dim"]
            fl += 14 * n
    elif op == "conv":
        n = sum(_lengths(case)) * case["dim"]
        by, fl = 2 * e * n, (2 * case["width"] + 5) * n
        if case["train"]:
            by += 3 * e * n
            fl += (6 * case["width"] + 10) * n
    elif op == "conv_step":
        n = case["batch"] * case["dim"]
        by, fl = e * n * (2 + 2 * (case["width"] - 1)), (2 * case["width"] + 5) * n
    elif op == "scan":
        n, N = sum(_lengths(case)) * case["dim"], case["state"]
        bc = sum(_lengths(case)) * 2 * N * e
        by, fl = 4 * e * n + bc, 7 * N * n
        if case["train"]:                     # x, delta, z, dy in; dx, ddelta, dz out; B, C in, dB, dC out
            by += 7 * e * n + 2 * bc
            fl += 16 * N * n
    elif op == "scan_step":
        n, N = case["batch"] * case["dim"], case["state"]
        by, fl = 8 * N * n + 4 * e * n, 7 * N * n
    elif op == "attn":
        D, lens = case["dim"], _lengths(case)
        pairs = case["heads"] * sum(_visible_pairs(l, case["window"], case["sinks"]) for l in lens)
        rows = sum(lens) * D * e
        by, fl = rows * (2 * case["heads"] + 2 * case["kv_heads"]), 4 * pairs * D
        if case["train"]:                     # q, k, v, o, do in; dq, dk, dv out; five products
            by += rows * (4 * case["heads"] + 4 * case["kv_heads"])
            fl += 10 * pairs * D
    else:
        keys = sum(min(p + 1, case["window"] + min(case["sinks"], max(0, p + 1 - case["window"]))) for p in _positions(case))
        by = e * case["dim"] * (2 * keys * case["kv_heads"] + 2 * case["batch"] * (case["heads"] + case["kv_heads"]))
        fl = 4 * keys * case["heads"] * case["dim"]
    return {"bytes": int(by), "flops": int(fl)}


# ------------------------------------------------------------------------------------------------------------ the inputs

def prepare(case, seed):
    dt = _DTYPE[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rn(*shape, dtype=dt, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    def ru(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case=case)
    op = case["op"]
    if op == "norm":
        R, D = case["rows"], case["dim"]
        s.update(x=rn(R, D, scale=1.5, shift=0.3), weight=rn(D, dtype=torch.float32, scale=0.1, shift=1.0),
                 bias=rn(D, dtype=torch.float32, scale=0.1))
        if case["train"]:
            s["dy"] = rn(R, D)
    elif op in ("conv", "conv_step"):
        B, C, K = case["batch"], case["dim"], case["width"]
        s.update(weight=rn(C, K, dtype=torch.float32, scale=K ** -0.5), bias=rn(C, dtype=torch.float32, scale=0.1))
        if op == "conv_step":
            s.update(x=rn(B, C), state=rn(B, K - 1, C))
        else:
            L = case["length"]
            s["x"] = rn(B, L, 2 * C)[..., :C]                       # the first half of the input projection's output
            s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None
            if case["train"]:
                s["dy"] = rn(B, L, C)
    elif op in ("scan", "scan_step"):
        B, C, N = case["batch"], case["dim"], case["state"]
        n = torch.arange(1, N + 1, device="cuda", dtype=torch.float32)
        step = torch.exp(ru(C) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        s.update(A=-(n * torch.exp(0.1 * torch.randn(C, N, generator=g, device="cuda"))).contiguous(),
                 D=rn(C, dtype=torch.float32, scale=0.1, shift=1.0),
                 delta_bias=step + torch.log(-torch.expm1(-step)))  # softplus of it is the step
        lead = (B,) if op == "scan_step" else (B, case["length"])
        s.update(x=rn(*lead, C), delta=rn(*lead, C, scale=0.5), z=rn(*lead, C))
        bc = rn(*lead, 2 * N)                                       # one projection gives both
        s.update(B=bc[..., :N], C=bc[..., N:])
        if op == "scan_step":
            s["state"] = rn(B, C, N, dtype=torch.float32, scale=0.3)
        else:
            s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None
            if case["train"]:
                s["dy"] = rn(B, case["length"], C)
    else:
        B, H, Hk, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        if op == "attn":                                            # heads lie inside a position, as a projection leaves them
            L = case["length"]
            q, k, v = rn(B, L, H, D), rn(B, L, Hk, D), rn(B, L, Hk, D)
            s.update(q=q.transpose(1, 2), k=k.transpose(1, 2), v=v.transpose(1, 2))
            s["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32) if case["ragged"] else None
            if case["train"]:
                s["do"] = rn(B, L, H, D).transpose(1, 2)
        else:
            cap = case["window"] + case["sinks"]
            s.update(q=rn(B, H, D), k=rn(B, Hk, D), v=rn(B, Hk, D), k_cache=rn(B, Hk, cap, D), v_cache=rn(B, Hk, cap, D),
                     positions=torch.tensor(_positions(case), device="cuda", dtype=torch.int32))
    return s


# ------------------------------------------------------------------------------------------------------ plain form

def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20))))


def _row_mask(s, L):
    """(B, L) truth values of the positions inside each sequence, or None"""
    if s.get("lengths") is None:
        return None
    return torch.arange(L, device="cuda")[None] < s["lengths"][:, None]


def _plain_norm(s, eps=1e-5):
    x = s["x"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * rstd
    y = (xh * s["weight"] + s["bias"]).to(s["x"].dtype)
    if "dy" not in s:
        return y
    dy = s["dy"].float()
    gw = dy * s["weight"]
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xh).sum(0), dy.sum(0)


def _plain_conv(s):
    case, w = s["case"], s["weight"]
    K, dt = case["width"], s["x"].dtype
    if case["op"] == "conv_step":
        window = torch.cat([s["state"], s["x"][:, None]], 1)
        pre = (window.float() * w.t()[None]).sum(1) + s["bias"]
        y = pre * torch.sigmoid(pre) if case["act"] == "silu" else pre
        s["state"].copy_(window[:, 1:])
        return y.to(dt), s["state"]
    x = s["x"].float()
    L = x.shape[1]
    inside = _row_mask(s, L)
    if inside is not None:
        x = torch.where(inside[..., None], x, 0.0)
    xp = torch.cat([x.new_zeros(x.shape[0], K - 1, x.shape[2]), x], 1)
    pre = s["bias"].expand_as(x)
    for k in range(K):
        pre = pre + w[:, k] * xp[:, k:k + L]
    sig = torch.sigmoid(pre)
    y = pre * sig if case["act"] == "silu" else pre
    if inside is not None:
        y = torch.where(inside[..., None], y, 0.0)
    if "dy" not in s:
        return y.to(dt)
    g = s["dy"].float()
    if inside is not None:
        g = torch.where(inside[..., None], g, 0.0)
    if case["act"] == "silu":
        g = g * (sig * (1 + pre * (1 - sig)))
    gp = torch.cat([g, g.new_zeros(g.shape[0], K - 1, g.shape[2])], 1)
    dx = torch.zeros_like(x)
    dw = torch.empty_like(w)
    for k in range(K):
        dx = dx + w[:, k] * gp[:, K - 1 - k:K - 1 - k + L]
        dw[:, k] = (g * xp[:, k:k + L]).sum((0, 1))
    if inside is not None:
        dx = torch.where(inside[..., None], dx, 0.0)
    return y.to(dt), dx.to(dt), dw, g.sum((0, 1))


def _doubling(a, u):
    """h_t = a_t h_{t-1} + u_t along dimension 1 from h = 0, in ceil(log2 L) passes"""
    L, step = a.shape[1], 1
    while step < L:
        u = torch.cat([u[:, :step], u[:, step:] + a[:, step:] * u[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return u


def _plain_scan(s):
    x, z, A = s["x"].float(), s["z"].float(), s["A"]
    pre = s["delta"].float() + s["delta_bias"]
    d = _softplus(pre)
    Bm, Cm = s["B"].float(), s["C"].float()
    dt = s["x"].dtype
    sz = torch.sigmoid(z)
    if s["case"]["op"] == "scan_step":
        h = torch.exp(d[..., None] * A) * s["state"] + (d * x)[..., None] * Bm[:, None, :]
        y = ((h * Cm[:, None, :]).sum(-1) + s["D"] * x) * (z * sz)
        s["state"].copy_(h)
        return y.to(dt), s["state"]
    inside = _row_mask(s, x.shape[1])
    if inside is not None:
        m = inside[..., None]
        x, z, sz, d = (torch.where(m, t, 0.0) for t in (x, z, sz, d))
    a = torch.exp(d[..., None] * A)                                         # (B, L, C, N)
    h = _doubling(a, (d * x)[..., None] * Bm[:, :, None, :])
    yp = (h * Cm[:, :, None, :]).sum(-1) + s["D"] * x
    y = (yp * (z * sz)).to(dt)
    if "dy" not in s:
        return y, h[:, -1].contiguous()
    dy = s["dy"].float()
    if inside is not None:
        dy = torch.where(m, dy, 0.0)
    u = dy * (z * sz)
    dz = dy * yp * (sz * (1 + z * (1 - sz)))
    # the adjoint state runs the other way: g_t = C_t u_t + a_{t+1} g_{t+1}
    a_next = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    gr = _doubling(a_next.flip(1), (u[..., None] * Cm[:, :, None, :]).flip(1)).flip(1)
    h_prev = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    e = gr * h_prev * a                                                     # dL / d(exponent)
    gB = (gr * Bm[:, :, None, :]).sum(-1)
    dx = d * gB + s["D"] * u
    dd = (x * gB + (e * A).sum(-1)) * torch.sigmoid(pre)
    if inside is not None:
        dx, dd, dz = (torch.where(m, t, 0.0) for t in (dx, dd, dz))
    dA = (e * d[..., None]).sum((0, 1))
    dB = (gr * (d * x)[..., None]).sum(2)
    dC = (h * u[..., None]).sum(2)
    return (y, dx.to(dt), dd.to(dt), dA, dB.to(dt), dC.to(dt), (u * x).sum((0, 1)), dz.to(dt), dd.sum((0, 1)))


def _plain_attn(s):
    case = s["case"]
    W, S, D = case["window"], case["sinks"], case["dim"]
    B, H, L, _ = s["q"].shape
    Hk = case["kv_heads"]
    G, scale, dt = H // Hk, D ** -0.5, s["q"].dtype
    q = s["q"].float().reshape(B, Hk, G, L, D)
    k, v = s["k"].float()[:, :, None], s["v"].float()[:, :, None]
    inside = _row_mask(s, L)
    if inside is not None:
        k, v = (torch.where(inside[:, None, None, :, None], t, 0.0) for t in (k, v))
    train = "do" in s
    out = torch.empty_like(q)
    if train:
        do = s["do"].float().reshape(B, Hk, G, L, D)
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    step = 512
    for i0 in range(0, L, step):
        i1 = min(L, i0 + step)
        lo = max(0, i0 - W + 1)
        cols = torch.cat([torch.arange(0, min(S, lo), device="cuda"), torch.arange(lo, i1, device="cuda")])
        i, j = torch.arange(i0, i1, device="cuda")[:, None], cols[None]
        see = ((j <= i) & ((i - j < W) | (j < S)))[None, None, None]
        if inside is not None:
            see = see & inside[:, None, None, i0:i1, None] & inside[:, cols][:, None, None, None, :]
        kb, vb = k[:, :, :, cols], v[:, :, :, cols]
        sc = torch.matmul(q[:, :, :, i0:i1], kb.transpose(-1, -2).contiguous()) * scale
        sc = torch.where(see, sc, -math.inf)
        mx = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(torch.isinf(mx), 0.0, mx))
        den = p.sum(-1, keepdim=True)
        p = p / torch.where(den == 0, 1.0, den)
        o = torch.matmul(p, vb)
        out[:, :, :, i0:i1] = o
        if train:
            dob = do[:, :, :, i0:i1]
            if inside is not None:
                dob = torch.where(inside[:, None, None, i0:i1, None], dob, 0.0)
            dp = torch.matmul(dob, vb.transpose(-1, -2).contiguous())
            ds = p * (dp - (dob * o).sum(-1, keepdim=True)) * scale
            dq[:, :, :, i0:i1] = torch.matmul(ds, kb)
            dk[:, :, :, cols] += torch.matmul(ds.transpose(-1, -2).contiguous(), q[:, :, :, i0:i1]).sum(2, keepdim=True)
            dv[:, :, :, cols] += torch.matmul(p.transpose(-1, -2).contiguous(), dob).sum(2, keepdim=True)
    out = out.reshape(B, H, L, D).to(dt)
    if not train:
        return out
    return out, dq.reshape(B, H, L, D).to(dt), dk[:, :, 0].to(dt), dv[:, :, 0].to(dt)


def _slots(p, S, cap):
    """Where the rolling cache keeps position p: sinks in front, the rest in turn behind them."""
    return torch.where(p < S, p, S + (p - S) % max(1, cap - S))


def _plain_attn_step(s):
    case = s["case"]
    W, S, D = case["window"], case["sinks"], case["dim"]
    B, H, _ = s["q"].shape
    Hk, cap = case["kv_heads"], s["k_cache"].shape[2]
    pos = s["positions"].long()
    b = torch.arange(B, device="cuda")
    slot = _slots(pos, S, cap)
    s["k_cache"][b, :, slot] = s["k"]
    s["v_cache"][b, :, slot] = s["v"]
    # the position that each slot holds: the latest one that maps there
    t = torch.arange(cap, device="cuda")[None]
    ring = max(1, cap - S)
    held = torch.where(t < S, t, pos[:, None] - (pos[:, None] - S - (t - S)) % ring)
    see = (held >= torch.where(t < S, 0, S)) & (held <= pos[:, None]) & ((pos[:, None] - held < W) | (held < S))
    q = s["q"].float().reshape(B, Hk, H // Hk, D)
    sc = torch.matmul(q, s["k_cache"].float().transpose(-1, -2).contiguous()) * D ** -0.5
    sc = torch.where(see[:, None, None], sc, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, s["v_cache"].float()).reshape(B, H, D).to(s["q"].dtype)
    return o, s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------- the framework's calls

def _leaves(s, names):
    return [s[n].detach().requires_grad_() for n in names]


def _own(s):
    bk = _bkcore()
    case = s["case"]
    op = case["op"]
    if op == "norm":
        if not case["train"]:
            return bk.layer_norm(s["x"], s["weight"], s["bias"])
        leaves = _leaves(s, ("x", "weight", "bias"))
        y = bk.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if op in ("conv", "conv_step"):
        act = None if case["act"] == "none" else case["act"]
        if op == "conv_step":
            return bk.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation=act), s["state"]
        if not case["train"]:
            return bk.causal_conv(s["x"], s["weight"], s["bias"], activation=act, lengths=s["lengths"])
        leaves = _leaves(s, ("x", "weight", "bias"))
        y = bk.causal_conv(*leaves, activation=act, lengths=s["lengths"])
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if op == "scan_step":
        y = bk.selective_scan_step(s["x"], s["state"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"],
                                   s["delta_bias"], delta_softplus=True)
        return y, s["state"]
    if op == "scan":
        names = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias")
        if not case["train"]:
            return bk.selective_scan(*(s[n] for n in names), delta_softplus=True, lengths=s["lengths"], return_state=True)
        leaves = _leaves(s, names)
        y = bk.selective_scan(*leaves, delta_softplus=True, lengths=s["lengths"])
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if op == "attn_step":
        o = bk.sliding_attention_step(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], case["window"],
                                      case["sinks"])
        return o, s["k_cache"], s["v_cache"]
    if not case["train"]:
        return bk.sliding_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"], lengths=s["lengths"])
    leaves = _leaves(s, ("q", "k", "v"))
    o = bk.sliding_attention(*leaves, case["window"], case["sinks"], lengths=s["lengths"])
    return (o.detach(), *torch.autograd.grad(o, leaves, s["do"]))


_PLAIN = {"norm": _plain_norm, "conv": _plain_conv, "conv_step": _plain_conv, "scan": _plain_scan,
          "scan_step": _plain_scan, "attn": _plain_attn, "attn_step": _plain_attn_step}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    d64 = {k: (t.double() if torch.is_tensor(t) and t.is_floating_point() else t) for k, t in s.items()}
    with torch.no_grad():
        return {"norm": _exact_norm, "conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan,
                "scan_step": _exact_scan_step, "attn": _exact_attn, "attn_step": _exact_attn_step}[case["op"]](case, d64)


def _exact_norm(case, s, eps=1e-5):
    var, mean = torch.var_mean(s["x"], -1, correction=0, keepdim=True)
    sd = torch.sqrt(var + eps)
    xh = (s["x"] - mean) / sd
    y = xh * s["weight"] + s["bias"]
    if not case["train"]:
        return y
    n = case["dim"]
    g = s["dy"] * s["weight"]
    dx = (n * g - g.sum(-1, keepdim=True) - xh * (g * xh).sum(-1, keepdim=True)) / (n * sd)
    return y, dx, torch.einsum("rd,rd->d", s["dy"], xh), s["dy"].sum(0)


def _act64(case, pre):
    """activation and its derivative"""
    if case["act"] == "none":
        return pre, torch.ones_like(pre)
    sg = 1 / (1 + torch.exp(-pre))
    return pre * sg, sg + pre * sg * (1 - sg)


def _exact_conv_step(case, s):
    hist = torch.cat([s["state"], s["x"][:, None]], 1)
    pre = torch.einsum("bkc,ck->bc", hist, s["weight"]) + s["bias"]
    return _act64(case, pre)[0], hist[:, 1:].contiguous()


def _exact_conv(case, s):
    B, L, C = s["x"].shape
    K = case["width"]
    y, dx = torch.zeros(2, B, L, C, device="cuda", dtype=torch.float64)
    dw, db = torch.zeros_like(s["weight"]), torch.zeros_like(s["bias"])
    for b, n in enumerate(_lengths(case)):                   # each sequence alone, without its padding
        if n == 0:
            continue
        xs = torch.cat([torch.zeros(K - 1, C, device="cuda", dtype=torch.float64), s["x"][b, :n]])
        taps = xs.unfold(0, K, 1)                            # (n, C, K)
        pre = (taps * s["weight"]).sum(-1) + s["bias"]
        out, der = _act64(case, pre)
        y[b, :n] = out
        if case["train"]:
            g = s["dy"][b, :n] * der
            dw += (taps * g[..., None]).sum(0)
            db += g.sum(0)
            back = torch.zeros(n + K - 1, C, device="cuda", dtype=torch.float64)
            for k in range(K):
                back[k:k + n] += g * s["weight"][:, k]
            dx[b, :n] = back[K - 1:]
    return (y, dx, dw, db) if case["train"] else y


def _exact_scan_step(case, s):
    d = torch.nn.functional.softplus(s["delta"] + s["delta_bias"], threshold=40)
    h = s["state"] * torch.exp(torch.einsum("bc,cn->bcn", d, s["A"])) + torch.einsum("bc,bn->bcn", d * s["x"], s["B"])
    y = torch.einsum("bcn,bn->bc", h, s["C"]) + s["x"] * s["D"]
    return y * torch.nn.functional.silu(s["z"]), h


def _exact_scan(case, s):
    B, L, C = s["x"].shape
    N = case["state"]
    if B * L * C * N > 1 << 28:
        return None
    lens = torch.tensor(_lengths(case), device="cuda")
    pre = s["delta"] + s["delta_bias"]
    d = torch.nn.functional.softplus(pre, threshold=40)
    act = torch.nn.functional.silu(s["z"])
    train = case["train"]
    h = torch.zeros(B, C, N, device="cuda", dtype=torch.float64)
    hs = torch.empty(L, B, C, N, device="cuda", dtype=torch.float64) if train else None
    yp = torch.zeros(B, L, C, device="cuda", dtype=torch.float64)
    for t in range(L):                                       # one position after the other
        live = (t < lens)[:, None, None]
        if train:
            hs[t] = h
        nxt = torch.exp(d[:, t, :, None] * s["A"]) * h + (d[:, t] * s["x"][:, t])[..., None] * s["B"][:, t, None]
        h = torch.where(live, nxt, h)
        yp[:, t] = torch.where(live[..., 0], (h * s["C"][:, t, None]).sum(-1) + s["D"] * s["x"][:, t], 0.0)
    y = yp * torch.where((torch.arange(L, device="cuda")[None] < lens[:, None])[..., None], act, 0.0)
    if not train:
        return y, h
    dx, dd, dz = torch.zeros(3, B, L, C, device="cuda", dtype=torch.float64)
    dB, dC = torch.zeros(2, B, L, N, device="cuda", dtype=torch.float64)
    dA, dD, dbias = torch.zeros_like(s["A"]), torch.zeros_like(s["D"]), torch.zeros_like(s["D"])
    g = torch.zeros_like(h)
    for t in range(L - 1, -1, -1):
        live = (t < lens)[:, None]
        xt, dt_, dyt = s["x"][:, t], d[:, t], torch.where(live, s["dy"][:, t], 0.0)
        sg = torch.sigmoid(s["z"][:, t])
        u = dyt * act[:, t]
        dz[:, t] = dyt * yp[:, t] * (sg + act[:, t] * (1 - sg))
        g = g + u[..., None] * s["C"][:, t, None]
        a = torch.exp(dt_[..., None] * s["A"])
        hn = a * hs[t] + (dt_ * xt)[..., None] * s["B"][:, t, None]
        dC[:, t] = (u[..., None] * hn).sum(1)
        gl = torch.where(live[..., None], g, 0.0)
        dB[:, t] = (gl * (dt_ * xt)[..., None]).sum(1)
        gb = (gl * s["B"][:, t, None]).sum(-1)
        ex = gl * a * hs[t]
        dA += (ex * dt_[..., None]).sum(0)
        dx[:, t] = gb * dt_ + s["D"] * u
        dd[:, t] = (gb * xt + (ex * s["A"]).sum(-1)) * torch.sigmoid(pre[:, t])
        dD += (u * xt).sum(0)
        dbias += dd[:, t].sum(0)
        g = torch.where(live[..., None], g * a, g)
    return y, dx, dd, dA, dB, dC, dD, dz, dbias


def _exact_attn(case, s):
    B, H, L, D = s["q"].shape
    if B * H * L * L > 1 << 33:
        return None
    G = H // case["kv_heads"]
    out, dq = torch.zeros(2, B, H, L, D, device="cuda", dtype=torch.float64)
    dk, dv = torch.zeros(2, B, case["kv_heads"], L, D, device="cuda", dtype=torch.float64)
    for b, n in enumerate(_lengths(case)):
        i = torch.arange(n, device="cuda")
        gap = i[:, None] - i[None]
        hide = (gap < 0) | ((gap >= case["window"]) & (i[None] >= case["sinks"]))
        for h in range(H if n else 0):
            q, k, v = s["q"][b, h, :n].contiguous(), s["k"][b, h // G, :n].contiguous(), s["v"][b, h // G, :n].contiguous()
            p = torch.softmax((q @ k.t().contiguous() / math.sqrt(D)).masked_fill(hide, -math.inf), -1)
            out[b, h, :n] = p @ v
            if case["train"]:
                do = s["do"][b, h, :n].contiguous()
                dp = do @ v.t().contiguous()
                ds = p * (dp - (dp * p).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[b, h, :n] = ds @ k
                dk[b, h // G, :n] += ds.t().contiguous() @ q
                dv[b, h // G, :n] += p.t().contiguous() @ do
    return (out, dq, dk, dv) if case["train"] else out


def _exact_attn_step(case, s):
    B, H, D = s["q"].shape
    W, S, cap = case["window"], case["sinks"], s["k_cache"].shape[2]
    G = H // case["kv_heads"]
    out = torch.zeros_like(s["q"])
    kc, vc = s["k_cache"].clone(), s["v_cache"].clone()
    for b, p in enumerate(_positions(case)):
        def slot(j):
            return j if j < S else S + (j - S) % (cap - S)
        kc[b, :, slot(p)], vc[b, :, slot(p)] = s["k"][b], s["v"][b]
        first = max(0, p - W + 1)
        seen = torch.tensor([slot(j) for j in list(range(min(S, first))) + list(range(first, p + 1))], device="cuda")
        for h in range(H):
            w = torch.softmax(kc[b, h // G, seen] @ s["q"][b, h] / math.sqrt(D), 0)
            out[b, h] = w @ vc[b, h // G, seen]
    return out, kc, vc
