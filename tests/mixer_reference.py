"""Plain 64-bit CPU implementations of the mixing layer's operators, with the error bounds the tests use.

u32 = 2^-24 is half a step of float32.  A bound ``E`` is the float32 error of a computed value; a value stored in type T
is off by at most  E + half a step of T (relative to the value) -- ``assert_within`` adds that rounding."""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, err, what=""):
    """|got - want| <= err + half a step of got's type at the computed value; non-finite values in the same places."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    u = 0.0 if got.dtype == torch.float32 else half_step(got.dtype)   # float32: the last rounding is part of err
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 1e-37        # below the normal range steps are absolute
    g = got.detach().double().cpu()
    want, err = want.double(), torch.as_tensor(err, dtype=torch.float64).expand_as(want)
    bad = torch.isnan(g) != torch.isnan(want)
    assert not bad.any(), f"{what}: NaN in other places, first {bad.nonzero()[0].tolist()}"
    ok = torch.isnan(want) | (g == want) | ((g - want).abs() <= err + u * (want.abs() + err) + tiny)
    if not ok.all():
        i = tuple((~ok).nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} beyond the bound; at {i}: got {float(g[i]):.9g}, "
                             f"want {float(want[i]):.9g}, bound {float((err + u * want.abs())[i]):.3g}")


def d64(*ts):
    out = [None if t is None else t.detach().double().cpu() for t in ts]
    return out[0] if len(out) == 1 else out


# ------------------------------------------------------------------------------------------------------------ layer norm

def norm(x, w, b, eps, dy=None):
    """y, dx, dw, db (the last three None without dy) and their bounds.

    mean: at most 32 elements a thread and ten levels of a tree, so 48 u32 of mean |x|; m = mean|x| rstd is what that is worth
    in units of xh.  var: 50 u32 and twice the mean's part; rstd: half of it and its own two roundings."""
    D = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * rstd
    m = x.abs().mean(-1, keepdim=True) * rstd
    dxh = U32 * (xh.abs() * (30 + 50 * m) + 50 * m + 2)
    W = torch.ones(D, dtype=torch.float64) if w is None else w
    B = torch.zeros(D, dtype=torch.float64) if b is None else b
    y = xh * W + B
    out = [(y, W.abs() * dxh + 3 * U32 * (xh.abs() * W.abs() + B.abs()))]
    if dy is None:
        return out[0]
    g = dy * W
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    size = rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + (1 + xh.abs()) * (g.abs() * (1 + xh.abs())).mean(-1, keepdim=True))
    out.append((dx, U32 * (120 + 120 * m) * size))
    rows = x.shape[:-1].numel()
    depth = 60 + rows / 4          # additions a column's sum goes through: a wave's rows, the joins (at most all rows / 4)
    s = tuple(range(x.dim() - 1))
    out.append(((dy * xh).sum(s), (dy.abs() * (dxh + depth * U32 * xh.abs())).sum(s)))
    out.append((dy.sum(s), depth * U32 * dy.abs().sum(s)))
    return out


# --------------------------------------------------------------------------------------------------------- convolution

def conv(x, w, b, silu, lens=None, state=None, dy=None, dfinal=None):
    """dict of values and bounds: y, final, and with dy: dx, dw, db, dstate."""
    B, L, C = x.shape
    K = w.shape[1]
    lens = [L] * B if lens is None else [min(max(int(n), 0), L) for n in lens]
    bias = torch.zeros(C, dtype=torch.float64) if b is None else b
    st = torch.zeros(B, K - 1, C, dtype=torch.float64) if state is None else state
    r = {k: torch.zeros(B, L, C, dtype=torch.float64) for k in ("y", "ey", "dx", "edx")}
    r["final"] = torch.zeros(B, K - 1, C, dtype=torch.float64)
    for k, like in (("dw", w), ("edw", w), ("db", bias), ("edb", bias), ("dstate", st), ("edstate", st)):
        r[k] = torch.zeros_like(like)
    for i, n in enumerate(lens):
        xs = torch.cat([st[i], x[i, :n]])                       # (K - 1 + n, C)
        r["final"][i] = xs[n:]
        full = torch.zeros(K - 1 + n, C, dtype=torch.float64)
        efull = torch.zeros_like(full)
        for t in range(n):
            taps = xs[t:t + K]                                  # (K, C)
            pre = (w.t() * taps).sum(0) + bias
            mag = (w.t() * taps).abs().sum(0) + bias.abs()
            sg = torch.sigmoid(pre)
            # sigmoid by exp2 and a reciprocal, one step each, and the argument's rounding: 8 u32 of silu and 2 u32 more
            y = pre * sg if silu else pre
            epre = (K + 2) * U32 * mag
            r["y"][i, t] = y
            r["ey"][i, t] = 1.1 * epre + (U32 * (8 * y.abs() + 2) if silu else 0)
            if dy is not None:
                der = sg * (1 + pre * (1 - sg)) if silu else torch.ones_like(pre)
                g = dy[i, t] * der
                eg = dy[i, t].abs() * ((0.5 * epre + 12 * U32) if silu else 0)
                for k in range(K):
                    full[t + k] += w[:, k] * g
                    efull[t + k] += w[:, k].abs() * (eg + (K + 2) * U32 * g.abs())
                    r["dw"][:, k] += g * taps[k]
                    r["edw"][:, k] += taps[k].abs() * (eg + U32 * g.abs() * (60 + B * L / 8))
                r["db"] += g
                r["edb"] += eg + U32 * g.abs() * (60 + B * L / 8)
        if dfinal is not None:
            full[n:] += dfinal[i]
            efull[n:] += 2 * U32 * (dfinal[i].abs() + full[n:].abs())
        r["dstate"][i], r["edstate"][i] = full[:K - 1], efull[:K - 1]
        r["dx"][i, :n], r["edx"][i, :n] = full[K - 1:], efull[K - 1:]
    return r


# ------------------------------------------------------------------------------------------------------- selective scan

def scan(x, delta, A, Bm, Cm, D=None, z=None, bias=None, softplus=False, lens=None, h0=None, dy=None, dhT=None):
    """dict of values (y, hT and with dy: dx, ddelta, dA, dB, dC, dD, dz, dbias, dh0) and of bounds (e + name).

    Beside each value its magnitude is formed: the same formula with absolute values.  The decay is a product rounded
    twice and an exponential (at most 4 + 10 |d A| half steps, softplus included); the effect of one step's error dies out
    with the decay, so at most `memory` = min(L, 1 / (1 - largest decay)) of them add up.  64 more cover the fold of the
    chunks (the sum of d enters as s exp(-s) <= 0.37 of its own error) and the sum over states."""
    Bn, L, C = x.shape
    N = A.shape[1]
    lens = [L] * Bn if lens is None else [min(max(int(n), 0), L) for n in lens]
    pre = delta if bias is None else delta + bias
    d = torch.nn.functional.softplus(pre, threshold=30) if softplus else pre
    sk = torch.zeros(C, dtype=torch.float64) if D is None else D
    r = {k: torch.zeros_like(x) for k in ("y", "dx", "ddelta", "dz", "ey", "edx", "eddelta", "edz")}
    for k in ("dB", "dC", "edB", "edC"):
        r[k] = torch.zeros(Bn, L, N, dtype=torch.float64)
    for k in ("dA", "edA"):
        r[k] = torch.zeros_like(A)
    for k in ("dD", "edD", "dbias", "edbias"):
        r[k] = torch.zeros(C, dtype=torch.float64)
    for k in ("hT", "ehT", "dh0", "edh0"):
        r[k] = torch.zeros(Bn, C, N, dtype=torch.float64)
    for i, n in enumerate(lens):
        h = torch.zeros(C, N, dtype=torch.float64) if h0 is None else h0[i].clone()
        H = h.abs()
        a = torch.exp(d[i, :n, :, None] * A)
        worst = float(a.max()) if n else 0.0
        memory = min(n, 1.0 / (1.0 - worst)) if worst < 1 else n
        kappa = U32 * (64 + memory * (8 + 10 * float((d[i, :n, :, None] * A).abs().max() if n else 0)))
        hs, Hs = [h], [H]
        for t in range(n):
            h = a[t] * h + (d[i, t] * x[i, t])[:, None] * Bm[i, t]
            H = a[t] * H + (d[i, t] * x[i, t]).abs()[:, None] * Bm[i, t].abs()
            hs.append(h)
            Hs.append(H)
        r["hT"][i], r["ehT"][i] = h, kappa * H
        g = torch.zeros(C, N, dtype=torch.float64) if dhT is None else dhT[i].clone()
        G = g.abs()
        for t in range(n - 1, -1, -1):
            gate = torch.ones(C, dtype=torch.float64) if z is None else z[i, t] * torch.sigmoid(z[i, t])
            yp = (hs[t + 1] * Cm[i, t]).sum(-1) + sk * x[i, t]
            Yp = (Hs[t + 1] * Cm[i, t].abs()).sum(-1) + (sk * x[i, t]).abs()
            ug = U32 * 12 * (gate.abs() + 1) if z is not None else torch.zeros(C, dtype=torch.float64)
            r["y"][i, t] = yp * gate
            r["ey"][i, t] = kappa * Yp * gate.abs() + Yp * ug
            if dy is None:
                continue
            u = dy[i, t] * gate
            U = u.abs() + dy[i, t].abs() * ug / kappa       # the gate's own error, in units of kappa
            if z is not None:
                sg = torch.sigmoid(z[i, t])
                der = sg * (1 + z[i, t] * (1 - sg))
                r["dz"][i, t] = dy[i, t] * yp * der
                r["edz"][i, t] = dy[i, t].abs() * Yp * (kappa * der.abs() + 16 * U32)
            g = g + u[:, None] * Cm[i, t]
            G = G + U[:, None] * Cm[i, t].abs()
            dx_ = d[i, t] * x[i, t]
            many = U32 * (C + 60)                            # additions over the channels
            r["dC"][i, t] = (u[:, None] * hs[t + 1]).sum(0)
            r["edC"][i, t] = ((2 * kappa + many) * U[:, None] * Hs[t + 1]).sum(0)
            r["dB"][i, t] = (g * dx_[:, None]).sum(0)
            r["edB"][i, t] = ((2 * kappa + many) * G * dx_.abs()[:, None]).sum(0)
            gb, GB = (g * Bm[i, t]).sum(-1), (G * Bm[i, t].abs()).sum(-1)
            e, E = g * a[t] * hs[t], G * a[t] * Hs[t]
            sig = torch.sigmoid(pre[i, t]) if softplus else torch.ones(C, dtype=torch.float64)
            r["dx"][i, t] = d[i, t] * gb + sk * u
            r["edx"][i, t] = 2 * kappa * (d[i, t].abs() * GB + sk.abs() * U)
            dd = (x[i, t] * gb + (e * A).sum(-1)) * sig
            DD = (x[i, t].abs() * GB + (E * A.abs()).sum(-1)) * sig
            r["ddelta"][i, t], r["eddelta"][i, t] = dd, 3 * kappa * DD
            far = U32 * (L * Bn / 8 + 60)                    # additions over the positions
            r["dA"] += e * d[i, t][:, None]
            r["edA"] += (3 * kappa + far) * E * d[i, t].abs()[:, None]
            r["dD"] += u * x[i, t]
            r["edD"] += (kappa + far) * U * x[i, t].abs()
            r["dbias"] += dd
            r["edbias"] += (3 * kappa + far) * DD
            g, G = g * a[t], G * a[t]
        r["dh0"][i], r["edh0"][i] = g, 2 * kappa * G
    return r


def directional(f, args, grads, index, seed, step=1e-6):
    """<gradient, v> by the given gradient and by a central difference of the 64-bit f along a random direction v of
    argument `index`, with the size of the terms."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(args[index].shape, generator=g, dtype=torch.float64)
    plus, minus = list(args), list(args)
    plus[index], minus[index] = args[index] + step * v, args[index] - step * v
    fd = float((f(*plus) - f(*minus)) / (2 * step))
    gd = d64(grads[index])
    return float((gd * v).sum()), fd, float((gd * v).abs().sum())


# ------------------------------------------------------------------------------------------------------------ attention

def attention(q, k, v, window, sinks, scale, u, lens=None, do=None):
    """dict of values (o and with do: dq, dk, dv) and bounds (e + name); u is half a step of the operands' type.

    Scores: D products in float32, 2 D u32 of sum |q_i k_j|, plus the base-2 exponential (4 u32 and the scaled score's own
    rounding): ep is what that is worth relative to a probability.  Probabilities and score gradients are rounded to the
    operands' type before the second products (u each, and 2^-25 below float16's normal range); sums over up to L keys in
    float32 add L u32 at most."""
    B, H, L, D = q.shape
    Hk = k.shape[1]
    G = H // Hk
    lens = [L] * B if lens is None else [min(max(int(n), 0), L) for n in lens]
    r = {n: torch.zeros_like(q) for n in ("o", "eo", "dq", "edq")}
    r.update({n: torch.zeros_like(k) for n in ("dk", "edk", "dv", "edv")})
    tiny = 2.0 ** -25 if u == half_step(torch.float16) else 0.0
    ur = 0.0 if u == half_step(torch.float32) else u
    for b, n in enumerate(lens):
        if n == 0:
            continue
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        see = (j <= i) & ((i - j < window) | (j < sinks))
        for h in range(H):
            Q, K, V = q[b, h, :n], k[b, h // G, :n], v[b, h // G, :n]
            s = (Q @ K.t()) * scale
            mag = (Q.abs() @ K.t().abs()) * abs(scale)
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            ep = (2 * D * U32 * mag + 8 * U32 * (1 + mag)).masked_fill(~see, 0)
            ep = ep + (p * ep).sum(-1, keepdim=True) + (n + 20) * U32        # the score's own error, the sum's, its rounding
            o = p @ V
            pe = p * (ep + ur) + tiny * see
            r["o"][b, h, :n] = o
            r["eo"][b, h, :n] = pe @ V.abs() + (n + 10) * U32 * (p @ V.abs())
            if do is None:
                continue
            g = do[b, h, :n]
            dp, Dp = g @ V.t(), g.abs() @ V.abs().t()
            # delta comes from the output as it was stored
            eo = r["eo"][b, h, :n] + ur * o.abs()
            delta, ede = (g * o).sum(-1, keepdim=True), (g.abs() * (eo + (D + 4) * U32 * o.abs())).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            eds = p * ((ep + 2 * U32) * (dp - delta).abs() + 2 * D * U32 * Dp + ede) + ur * ds.abs() + tiny * see
            more = (n * G + 20) * U32
            r["dq"][b, h, :n] = ds @ K * scale
            r["edq"][b, h, :n] = (eds + more * ds.abs()) @ K.abs() * abs(scale)
            r["dk"][b, h // G, :n] += ds.t() @ Q * scale
            r["edk"][b, h // G, :n] += (eds + more * ds.abs()).t() @ Q.abs() * abs(scale)
            r["dv"][b, h // G, :n] += p.t() @ g
            r["edv"][b, h // G, :n] += (pe + more * p).t() @ g.abs()
    return r
