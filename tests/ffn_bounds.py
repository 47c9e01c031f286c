"""The dense / gated products in 64 bits with a bound on what fp32 sums and the stated roundings may be off.

u = 2^-24 is fp32's half step, r the half step of the tensors' type (2^-24 or 2^-8: torch.finfo(t).eps / 2).
A sum of n products in any order, in fp32, is off by at most (n + 16) u times the sum of the magnitudes
(16: the three-part products' remainder, at most 2 u a term, and the additions behind the sum).
|a'| <= 1.13 and |a''| <= 1 for every activation; relu and leakyrelu jump by at most 1 where the sign of
a value within its own bound of zero is open. Elementwise functions: 8 u (fp32), 2^-18 (bf16: hardware exp2
and reciprocal, 2^-21 each, over at most 4 steps)."""
import torch

U = 2.0 ** -24


def act64(kind, v):
    F = torch.nn.functional
    return {None: lambda t: t, "relu": F.relu, "leakyrelu": F.leaky_relu, "elu": F.elu, "gelu": F.gelu,
            "silu": F.silu}[kind](v)


def dact64(kind, v):
    if kind is None:
        return torch.ones_like(v)
    v = v.clone().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act64(kind, v).sum(), v)[0]


def restored64(x):
    """The values the 8-bit form of x stands for, by its definition."""
    M, K = x.shape
    g = torch.nn.functional.pad(x.double(), (0, -K % 32)).view(M, -1, 32)
    top = g.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -126)
    for k in range(-126, 123):
        e = torch.where(127 * 2.0 ** (k - 1) < top, torch.full_like(e, k), e) if k > -126 else e
    e = e.clamp(min=-126)
    q = (g * torch.exp2(-e)).round()
    q = torch.where(e == 122, q.clamp(-63, 63), q)
    v = torch.where(torch.isfinite(top), q * torch.exp2(e), torch.full_like(top, float("nan")))
    return v.reshape(M, -1)[:, :K]


def product64(x, ws, bs, act, res, dy, dtype, kept=None):
    """({name: value}, {name: bound}) of the forward and, with dy, of every gradient. x, ws, bs, res, dy: any float
    tensors on the CPU; kept: what the backward takes for x."""
    u, r = U, torch.finfo(dtype).eps / 2
    el = 8 * u if dtype == torch.float32 else 2.0 ** -18
    x, ws = x.double(), [w.double() for w in ws]
    bs = [b.double() if b is not None else None for b in bs]
    K, N, M = x.shape[1], ws[0].shape[0], x.shape[0]
    two = len(ws) == 2

    def pre(v):
        out, err = [], []
        for w, b in zip(ws, bs):
            p, s = v @ w.t(), v.abs() @ w.abs().t()
            if b is not None:
                p, s = p + b, s + b.abs()
            out.append(p)
            err.append((K + 16) * u * s)
        return out, err

    val, tol = {}, {}
    p, e = pre(x)
    a = act64(act, p[0])
    ea = (1.13 if act else 1.0) * e[0] + (el * a.abs() if act else 0)
    if two:
        y, ey = a * p[1], ea * (p[1].abs() + e[1]) + a.abs() * e[1]
    else:
        y, ey = (a, ea) if res is None else (a + res.double(), ea + u * (a.abs() + res.double().abs()))
    ey = ey + 2 * u * y.abs()
    val["y"], tol["y"] = y, ey + r * (y.abs() + ey)
    if dy is None:
        return val, tol
    d = dy.double()
    kept = x if kept is None else kept.double()
    p, e = pre(kept)
    da = dact64(act, p[0])
    eda = e[0] + el * da.abs() + (1.0 * (p[0].abs() <= e[0]) if act in ("relu", "leakyrelu") else 0) if act else \
        torch.zeros_like(da)
    a = act64(act, p[0])
    ea = 1.13 * e[0] + el * a.abs()
    if two:
        dp = [d * p[1] * da, d * a]
        ed = [d.abs() * (e[1] * (da.abs() + eda) + p[1].abs() * eda) + 4 * u * dp[0].abs(), d.abs() * ea + 4 * u * dp[1].abs()]
    else:
        dp, ed = [d * da], [d.abs() * eda + 4 * u * (d * da).abs()]
    # db sums the unrounded values; dx and dW those rounded to the matrix instructions' type
    rr = r if dtype != torch.float32 else 0.0
    for i, n in enumerate("01"[:len(ws)]):
        s = dp[i].sum(0)
        es = ed[i].sum(0) + (M + 16) * u * dp[i].abs().sum(0)
        val["db" + n], tol["db" + n] = s, es + r * (s.abs() + es)
    ed = [x_ + rr * (v.abs() + x_) for x_, v in zip(ed, dp)]
    dx = sum(v @ w for v, w in zip(dp, ws))
    edx = sum(x_ @ w.abs() + (2 * N + 16) * u * ((v.abs() + x_) @ w.abs()) for x_, v, w in zip(ed, dp, ws))
    val["dx"], tol["dx"] = dx, edx + r * (dx.abs() + edx)
    for i, n in enumerate("01"[:len(ws)]):
        g = dp[i].t() @ kept
        eg = ed[i].t() @ kept.abs() + (M + 16) * u * ((dp[i].abs() + ed[i]).t() @ kept.abs())
        val["dw" + n], tol["dw" + n] = g, eg + r * (g.abs() + eg)
    if res is not None:
        val["dres"], tol["dres"] = d, torch.zeros_like(d)
    return val, tol


def outside(got, val, tol):
    """[(name, worst ratio of error to bound)] of what is out of bounds or not finite where it should be."""
    bad = []
    for k, v in got.items():
        t = tol[k].clamp(min=1e-30)
        ratio = ((v.double().cpu() - val[k]).abs() / t).nan_to_num(nan=float("inf"))
        if v.numel() and not ratio.max() <= 1:
            bad.append((k, float(ratio.max())))
    return bad
