"""embedding on the MI355X against its definition in 64 bits, and the modules around the feed-forward operators.

Forward: one fp32 multiplication, rounded once. Gradient of a token that n rows fall on: n - 1 additions and a
multiplication in fp32 and one rounding to the type, so at most n * 2^-24 of the sum of magnitudes, times
|scale|, and half a step of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _ops():
    from aimx import ops
    return ops


def _check(index, V, D, dtype, scale=1.0, pad=None, view=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(V, D, generator=g).to(dtype)
    dy = torch.randn(*index.shape, D + (3 if view else 0), generator=g).to(dtype)
    t = table.to(DEV).requires_grad_()
    out = _ops().embedding(index.to(DEV), t, scale, pad)
    ok = (index >= 0) & (index < V)
    want = table[index.clamp(0, V - 1).long()].double() * torch.tensor(scale, dtype=F32).double()
    want = torch.where(ok[..., None], want, torch.zeros_like(want))
    r = torch.finfo(dtype).eps / 2
    assert out.dtype == dtype and out.shape == (*index.shape, D)
    assert ((out.detach().double().cpu() - want).abs() <= (r + 2.0 ** -24) * want.abs()).all()
    dyd = dy.to(DEV)[..., 2:2 + D] if view else dy.to(DEV)
    got, = torch.autograd.grad(out, t, dyd, retain_graph=True)
    again, = torch.autograd.grad(out, t, dyd)
    assert torch.equal(got, again)
    d = (dy[..., 2:2 + D] if view else dy).double().reshape(-1, D)
    i = index.reshape(-1).long()
    keep = ok.reshape(-1)
    if pad is not None:
        keep = keep & (i != pad % V)
    ref = torch.zeros(V, D, dtype=torch.float64).index_add_(0, i[keep], d[keep]) * scale
    mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, i[keep], d[keep].abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64).index_add_(0, i[keep], torch.ones(int(keep.sum()), dtype=torch.float64))
    tol = (n[:, None] + 2) * 2.0 ** -24 * mag + r * ref.abs() * (1 + 2.0 ** -7)
    err = (got.double().cpu() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-30)).max())
    assert (got[n.to(DEV) == 0] == 0).all()


def _index(n, V, skew, seed=0):
    g = torch.Generator().manual_seed(seed + n * 7 + V)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    return ((V + 1.0) ** u - 1).long().clamp(0, V - 1) if skew else torch.randint(0, V, (n,), generator=g)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(0, 5, 8), (1, 1, 1), (1, 300, 64), (23, 119, 256), (31, 7, 5), (64, 64, 33),
                                   (257, 255, 16), (257, 256, 24), (1000, 3, 153), (5000, 70000, 9),
                                   (9186, 119, 64), (3000, 65535, 8), (3000, 65536, 8), (20000, 1000, 520)])
def test_embedding(n, V, D, dtype):
    for skew in (False, True):
        _check(_index(n, V, skew), V, D, dtype, scale=1.0 if skew else 27.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_token_for_all_and_long_runs(dtype):
    """A run over every segment, and runs that begin and end at each place of a segment of 32."""
    _check(torch.full((4100,), 2), 5, 40, dtype)
    for lead in (0, 1, 31, 32, 33):
        index = torch.cat([torch.zeros(lead), torch.ones(64), torch.full((33,), 2), torch.full((31,), 4)]).long()
        _check(index, 6, 12, dtype)
    many = torch.randint(0, 2, (140000,), generator=torch.Generator().manual_seed(1))  # segments of 40 rows
    _check(many, 3, 8, dtype)


def test_padding_and_out_of_range():
    index = torch.tensor([[3, 0, -1, 7], [5, 3, 2 ** 40, -2 ** 40]])
    for pad in (None, 3, -4, 0, 6):
        _check(index, 7, 16, F32, scale=-2.0, pad=pad)
        _check(index, 7, 15, BF16, pad=pad)
    _check(torch.tensor([9, -3, 8]), 8, 4, F32)  # nothing in range
    _check(index[:, 1].int(), 7, 16, F32)


def test_views_and_unaligned():
    _check(_index(500, 50, True), 50, 64, BF16, view=True)
    _check(_index(500, 50, True).view(4, 125).t(), 50, 7, F32, view=True)
    t = torch.randn(11, 9, device=DEV)[:, :8]  # rows 36 bytes apart
    assert torch.equal(_ops().embedding(torch.arange(11, device=DEV), t), t)
    flat = torch.randn(1 + 6 * 8, device=DEV)[1:].view(6, 8)  # contiguous rows at a 4-byte boundary
    assert torch.equal(_ops().embedding(torch.arange(6, device=DEV), flat, 2.0), flat * 2)


class _Kept(torch.autograd.Function):
    """fn(x, *params) whose gradients are those at `kept` in place of x."""

    @staticmethod
    def forward(ctx, fn, x, kept, *params):
        ctx.fn, ctx.at = fn, (kept, *params)
        return fn(x, *params)

    @staticmethod
    def backward(ctx, dy):
        at = [t.detach().requires_grad_() for t in ctx.at]
        with torch.enable_grad():
            grads = torch.autograd.grad(ctx.fn(*at), at, dy)
        return None, grads[0], None, *grads[1:]


def test_run_of_operators_trains_like_64_bits():
    """Lookup -> two gated blocks with skips -> a gated head, forward and every gradient, with and without
    8-bit checkpoints, against the same chain in 64 bits; with checkpoints the 64-bit backward stands at the
    values that the 8 bits of the GPU's own activations stand for. Each of the six products is off by 2^-24 times
    the square root of its up to 96 terms, forward and backward: under 600 half steps of the norm together."""
    from ffn_bounds import restored64
    from models import GatedBlock, ScaledEmbedding
    ops = _ops()
    torch.manual_seed(0)
    index = torch.randint(0, 50, (40, 7))

    def build(ck):
        torch.manual_seed(1)
        return torch.nn.ModuleList([ScaledEmbedding(50, 48, scale=4.0, padding_idx=3), GatedBlock(48, 96, 48, checkpoint8=ck),
                                    GatedBlock(48, 75, 48, activation_type="gelu", checkpoint8=ck), GatedBlock(48, 64, 5)])

    def plain(m, i, kept):
        x = m[0].weight[i.reshape(-1)] * 4.0
        x = torch.where((i.reshape(-1) == 3)[:, None], x.detach(), x)
        lin = torch.nn.functional.linear
        for k, b in enumerate(list(m)[1:]):
            act = b.activation
            gated = lambda v, wg, bg, wu, bu, act=act: act(lin(v, wg, bg)) * lin(v, wu, bu)  # noqa: E731
            kx, kh = kept[k] if kept[k] else (x, None)
            h = _Kept.apply(gated, x, kx.detach(), b.gate.weight, b.gate.bias, b.up.weight, b.up.bias)
            y = _Kept.apply(lin, h, (h if kh is None else kh).detach(), b.down.weight, b.down.bias)
            x = x + y if b.use_skip else y
        return x.view(*i.shape, -1)

    dy = torch.randn(40, 7, 5)
    for ck in (False, True):
        m = build(ck).to(DEV)
        x = index.to(DEV)
        kept = []
        for layer in m:
            if isinstance(layer, GatedBlock):
                with torch.no_grad():
                    h = ops.gated_linear(x, layer.gate.weight, layer.up.weight, layer.gate.bias, layer.up.bias,
                                         act="gelu" if isinstance(layer.activation, torch.nn.GELU) else "silu")
                rows = lambda t: restored64(t.detach().cpu().reshape(-1, t.shape[-1]))  # noqa: E731
                kept.append((rows(x), rows(h)) if layer.checkpoint8 else None)
            x = layer(x)
        ref = build(ck).double()
        want = plain(ref, index, kept)
        wg = torch.autograd.grad(want, list(ref.parameters()), dy.double())
        assert (x.double().cpu() - want).norm() <= 600 * 2.0 ** -24 * want.norm()
        for (name, _), a, b in zip(m.named_parameters(), torch.autograd.grad(x, list(m.parameters()), dy.to(DEV)), wg):
            assert (a.double().cpu() - b).norm() <= 600 * 2.0 ** -24 * b.norm(), (name, ck)


def test_gradient_against_differences():
    """Directional derivatives of the gated block and the lookup by central differences of the 64-bit forward
    at the same point: a step h leaves h^2 |f'''| / 6, below 1e-6 of the slope here."""
    from models import GatedBlock, ScaledEmbedding
    torch.manual_seed(2)
    emb, blk = ScaledEmbedding(11, 24, scale=2.0), GatedBlock(24, 40, 24)
    index, dy = torch.randint(0, 11, (30,)), torch.randn(30, 24).double()
    params = list(emb.parameters()) + list(blk.parameters())
    dirs = [torch.randn_like(p).double() for p in params]

    def f(t):
        e, wg, bg, wu, bu, wd, bd = [p.detach().double() + t * d for p, d in zip(params, dirs)]
        x = e[index] * 2.0
        L = torch.nn.functional.linear
        return ((L(torch.nn.functional.silu(L(x, wg, bg)) * L(x, wu, bu), wd, bd) + x) * dy).sum()

    slope = (f(1e-4) - f(-1e-4)) / 2e-4
    emb, blk = emb.to(DEV), blk.to(DEV)
    out = blk(emb(index.to(DEV)))
    got = torch.autograd.grad(out, list(emb.parameters()) + list(blk.parameters()), dy.float().to(DEV))
    have = sum((g.double().cpu() * d).sum() for g, d in zip(got, dirs))
    size = sum((g.double().cpu().abs() * d.abs()).sum() for g, d in zip(got, dirs))
    assert abs(have - slope) <= 1e-5 * size


def _graph(fn, warm=3):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(warm):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fn()
    return g, out


def test_captured_training_step_replays():
    """Lookup, gated block and head with gradients captured once; every replay, on new inputs, gives the eager
    result bit for bit, with eager work of the same operators between the replays."""
    ops = _ops()
    torch.manual_seed(4)
    table = torch.randn(90, 64, device=DEV, requires_grad=True)
    w = [torch.randn(s, device=DEV).mul_(0.1).requires_grad_() for s in ((80, 64), (80, 64), (64, 80))]
    index, dy = torch.zeros(300, dtype=torch.int64, device=DEV), torch.zeros(300, 64, device=DEV)

    def step():
        leaves = [t.detach().requires_grad_() for t in (table, *w)]
        x = ops.embedding(index, leaves[0], 3.0)
        h = ops.gated_linear(x, leaves[1], leaves[2], checkpoint8=True)
        y = ops.dense(h, leaves[3], residual=x)
        return (y, *torch.autograd.grad(y, leaves, dy))

    graph, out = _graph(step)
    for k in range(4):
        index.copy_(torch.randint(0, 90, (300,), device=DEV))
        dy.copy_(torch.randn(300, 64, device=DEV))
        want = [t.detach().clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_two_streams_at_once():
    """Calls on two streams share nothing: both give what one alone gives."""
    ops = _ops()
    x = torch.randn(3000, 100, device=DEV)
    w, u = torch.randn(200, 100, device=DEV), torch.randn(200, 100, device=DEV)
    index, table = torch.randint(0, 40, (5000,), device=DEV), torch.randn(40, 64, device=DEV, requires_grad=True)
    dy = torch.randn(5000, 64, device=DEV)
    want = ops.gated_linear(x, w, u), torch.autograd.grad(ops.embedding(index, table), table, dy)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((ops.gated_linear(x, w, u), torch.autograd.grad(ops.embedding(index, table), table, dy)[0]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in got)


def test_table_past_2_31_elements():
    ops = _ops()
    V, D = 2 ** 22 + 3, 520
    table = torch.zeros(V, D, dtype=BF16, device=DEV)
    rows = torch.tensor([0, 5, V - 1, V // 2, V - 1, 0], device=DEV)
    table[rows] = torch.randn(6, D, device=DEV).to(BF16)
    table.requires_grad_()
    y = ops.embedding(rows, table, 2.0)
    assert torch.equal(y, table[rows] * 2)
    dy = torch.randn(6, D, device=DEV).to(BF16)
    g, = torch.autograd.grad(y, table, dy)
    for v in (0, 5, V // 2, V - 1):
        want = (dy[rows == v].float().sum(0) * 2).to(BF16)
        assert torch.equal(g[v], want)
    g[rows] = 0
    assert not g.view(-1, 4).any(dim=0).any()
