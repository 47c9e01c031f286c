"""dense / gated_linear / pack8 on the MI355X against their definitions in 64 bits (tests/ffn_bounds.py has the
bounds and where they come from)."""
import pytest
import torch

from ffn_bounds import outside, product64, restored64

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _ops():
    from aimx import ops
    return ops


def _make(M, K, N, dtype, halves=1, bias=True, res=False, view=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    x = rnd(M, K + 5)[:, 3:3 + K] if view else rnd(M, K)
    ws = [(rnd(N, K).float() * K ** -0.5).to(dtype) for _ in range(halves)]
    bs = [rnd(N) if bias else None for _ in range(halves)]
    return x, ws, bs, rnd(M, N) if res else None, rnd(M, N)


def _run(x, ws, bs, act, res, dy, checkpoint8=False):
    """{name: tensor} of the forward and every gradient on the GPU."""
    ops = _ops()
    wide = torch.empty(x.shape[0], x.stride(0), dtype=x.dtype, device=DEV) if x.stride(0) > x.shape[1] else None
    if wide is not None:
        wide.fill_(float("nan"))
        off = 3
        wide[:, off:off + x.shape[1]] = x.to(DEV)
        xd = wide[:, off:off + x.shape[1]].detach().requires_grad_(dy is not None)
    else:
        xd = x.to(DEV).requires_grad_(dy is not None)
    put = lambda t: None if t is None else t.to(DEV).requires_grad_(dy is not None)  # noqa: E731
    ws, bs, res = [put(w) for w in ws], [put(b) for b in bs], put(res)
    if len(ws) == 2:
        y = ops.gated_linear(xd, *ws, *bs, act=act, checkpoint8=checkpoint8)
    else:
        y = ops.dense(xd, ws[0], bs[0], act=act, residual=res, checkpoint8=checkpoint8)
    out = {"y": y.detach()}
    if dy is not None:
        leaves = [("dx", xd)] + [(f"dw{i}", w) for i, w in enumerate(ws)] + \
            [(f"db{i}", b) for i, b in enumerate(bs) if b is not None] + ([("dres", res)] if res is not None else [])
        out.update(zip([k for k, _ in leaves], torch.autograd.grad(y, [t for _, t in leaves], dy.to(DEV))))
    return out


def _check(M, K, N, dtype, halves=1, act=None, bias=True, res=False, view=False, train=True, ckpt=False):
    x, ws, bs, r, dy = _make(M, K, N, dtype, halves, bias, res, view)
    got = _run(x, ws, bs, act, r, dy if train else None, ckpt)
    val, tol = product64(x, ws, bs, act, r, dy if train else None, dtype, restored64(x) if ckpt else None)
    assert not outside(got, val, tol), outside(got, val, tol)
    assert all(v.dtype == dtype for v in got.values())


SHAPES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (17, 33, 65), (16, 64, 128), (64, 64, 64), (65, 153, 307), (130, 256, 128),
          (257, 307, 613), (300, 1024, 70), (1000, 96, 33), (63, 4097, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_dense(M, K, N, dtype):
    _check(M, K, N, dtype, act="silu", res=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gated(M, K, N, dtype):
    _check(M, K, N, dtype, halves=2, act="silu")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("act", [None, "relu", "leakyrelu", "elu", "gelu"])
@pytest.mark.parametrize("halves", [1, 2])
def test_activations_without_bias(halves, act, dtype):
    if halves == 2 and act is None:
        pytest.skip("a gate has an activation")
    _check(70, 100, 90, dtype, halves=halves, act=act, bias=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N,halves,act", [
    (12800, 64, 1024, 1, None), (6400, 64, 1100, 2, "silu"),  # the largest tiles, their edges
    (2048, 128, 1536, 1, "gelu"), (1999, 64, 770, 2, "gelu"),  # the middle ones
    (40, 8192, 48, 1, "silu"), (200, 4096, 200, 1, None),  # k split over workgroups
    (9001, 40, 24, 2, "silu")])  # weight gradients over many rows
def test_tiles_and_splits(M, K, N, halves, act, dtype):
    _check(M, K, N, dtype, halves=halves, act=act, res=halves == 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("halves", [1, 2])
@pytest.mark.parametrize("M,K,N", [(1, 32, 8), (5, 31, 9), (130, 256, 96), (257, 307, 130)])
def test_checkpoint8(M, K, N, halves, dtype):
    _check(M, K, N, dtype, halves=halves, act="silu", ckpt=True, res=halves == 1)
    if halves == 1:
        _check(M, K, N, dtype, act=None, ckpt=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("halves", [1, 2])
def test_views_and_inference(halves, dtype):
    _check(77, 153, 51, dtype, halves=halves, act="silu", view=True)
    _check(77, 153, 51, dtype, halves=halves, act="silu", view=True, train=False)
    _check(77, 64, 64, dtype, halves=halves, act="silu", train=False, bias=False)


def test_fp32_is_fp32():
    """The three-part products reach fp32's own accuracy: against 64 bits the norm of the error stays below
    sqrt(K) half steps (the growth of K independent roundings), and no bf16 rounding shows."""
    for M, K, N in ((512, 256, 256), (333, 1024, 500)):
        x, ws, bs, _, _ = _make(M, K, N, F32)
        y = _run(x, ws, bs, None, None, None)["y"].double().cpu()
        ref = x.double() @ ws[0].double().t() + bs[0].double()
        assert (y - ref).norm() / ref.norm() < K ** 0.5 * 2.0 ** -24


def test_few_bf16_values_round_once():
    """One row: dW is an outer product and dx one row, so a rounding of the gradient before the activation would show
    whole. Each result is within one rounding to bf16 (2^-8) of the 64-bit value, and fp32 sums' error."""
    for halves, M, K, N in ((2, 1, 32, 32), (1, 3, 50, 40), (2, 40, 96, 70)):
        x, ws, bs, _, dy = _make(M, K, N, BF16, halves)
        got = _run(x, ws, bs, "silu", None, dy)
        val, tol = product64(x, ws, bs, "silu", None, dy, F32)
        for k, v in got.items():
            err = (v.double().cpu() - val[k]).abs()
            # the hardware exp2 and reciprocal of the 16-bit forward are off by 2^-18 at most (y only)
            assert (err <= tol[k] * 2 + 2.0 ** -8 * val[k].abs() * (1 + 2.0 ** -6) + 2.0 ** -18 * val[k].abs()).all(), k


def test_magnitudes_fp32():
    """Exponents from 2^-60 to 2^60 in one product, and values at the end of the range in either operand."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 96, generator=g) * torch.exp2(torch.randint(-60, 60, (40, 96), generator=g).float())
    w = torch.randn(50, 96, generator=g) * torch.exp2(torch.randint(-20, 20, (50, 96), generator=g).float())
    val, tol = product64(x, [w], [None], None, None, None, F32)
    got = _run(x, [w], [None], None, None, None)
    assert not outside(got, val, tol), outside(got, val, tol)
    big = torch.full((1, 1), 3.4028234e38)
    y = _run(big, [torch.ones(1, 1)], [None], None, None, None)["y"]
    assert float(y) == 3.4028234663852886e38


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nonfinite_rows_stay_apart(dtype):
    """A NaN or an infinity reaches its own row of y (and every weight gradient), no other row."""
    x, ws, bs, _, dy = _make(70, 96, 40, dtype)
    x[3, 5], x[69, 95] = float("nan"), float("inf")
    got = _run(x, ws, bs, None, None, dy)
    fin = torch.isfinite(got["y"]).all(1).cpu()
    assert not fin[3] and not fin[69] and fin[[i for i in range(70) if i not in (3, 69)]].all()
    assert torch.isfinite(got["dx"]).all()
    assert not torch.isfinite(got["dw0"][:, 5]).any() and not torch.isfinite(got["dw0"][:, 95]).any()
    assert torch.isfinite(got["dw0"][:, :5]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("halves", [1, 2])
def test_no_rows(halves, dtype):
    got = _run(*_make(0, 48, 40, dtype, halves)[:3], "silu", None, torch.zeros(0, 40, dtype=dtype))
    assert got["y"].shape == (0, 40) and got["dx"].shape == (0, 48)
    assert all((got[k] == 0).all() for k in got if k.startswith(("dw", "db")))


def test_shapes_and_partial_gradients():
    ops = _ops()
    x, (w,), (b,), _, _ = _make(12, 20, 30, F32)
    x, w, b = x.to(DEV), w.to(DEV), b.to(DEV)
    full = ops.dense(x, w, b, act="silu")
    assert torch.equal(ops.dense(x.view(3, 4, 20), w, b, act="silu"), full.view(3, 4, 30))
    assert torch.equal(ops.dense(x[5], w, b, act="silu"), full[5]) or \
        (ops.dense(x[5], w, b, act="silu") - full[5]).abs().max() < 1e-5
    # one leaf at a time gives what all together give; expanded gradients and residuals
    xs, wl, bl = x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    whole = torch.autograd.grad(ops.dense(xs, wl, bl, act="silu").sum(), [xs, wl, bl])
    for leaf, want in zip((0, 1, 2), whole):
        t = [x, w, b]
        t[leaf] = t[leaf].clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(ops.dense(*t, act="silu").sum(), t[leaf])[0], want)
    r = torch.randn(1, 30, device=DEV, requires_grad=True)
    y = ops.dense(x, w, b, residual=r.expand(12, 30))
    assert torch.allclose(y, ops.dense(x, w, b) + r)
    assert torch.equal(torch.autograd.grad(y.sum(), r)[0], torch.full((1, 30), 12.0, device=DEV))
    # transposed weights and rows out of order in memory
    wt = w.t().contiguous().t()
    assert torch.equal(ops.dense(x, wt, b, act="silu"), full)
    assert torch.equal(ops.dense(x.t().contiguous().t(), w, b, act="silu"), full)


def test_autocast_takes_bf16_operands():
    """fp32 tensors under autocast: operands rounded to bf16, fp32 sums and results (as aimx.linear)."""
    ops = _ops()
    for halves in (1, 2):
        x, ws, bs, _, dy = _make(130, 96, 70, F32, halves)
        with torch.autocast("cuda", dtype=BF16):
            got = _run(x, ws, bs, "silu", None, dy)
        rounded = [x.to(BF16)] + [w.to(BF16) for w in ws]
        val, tol = product64(rounded[0], rounded[1:], bs, "silu", None, dy, BF16)
        assert not outside(got, val, tol), outside(got, val, tol)
        ref, _ = product64(x, ws, bs, "silu", None, None, F32)
        assert got["y"].dtype == F32
        err = (got["y"].double().cpu() - val["y"]).norm() / val["y"].norm()
        away = (got["y"].double().cpu() - ref["y"]).norm() / ref["y"].norm()
        assert err < 2e-5 and away > 1e-4


# ---------------------------------------------------------------------------------------------
# 8 bits
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 31), (5, 32), (7, 33), (64, 256), (33, 153), (2, 4097)])
def test_pack8_values(M, K, dtype):
    ops = _ops()
    g = torch.Generator().manual_seed(M * 31 + K)
    x = (torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-30, 30, (M, K), generator=g).float())).to(dtype)
    for view in (False, True):
        xd = torch.nn.functional.pad(x, (3, 2), value=float("nan")).to(DEV)[:, 3:3 + K] if view else x.to(DEV)
        p = ops.pack8(xd)
        want = restored64(x)
        for t in (F32, BF16):
            y = ops.unpack8(p, t)
            assert y.dtype == t and torch.equal(y.double().cpu(), want)
        assert p.nbytes == M * (-(-K // 32) * 33)


def test_pack8_edges():
    """Each power of two and its neighbours as a group's largest, both ends of the range, subnormals, NaN and
    infinities; 127/128 is where the exponent steps."""
    ops = _ops()
    tops = []
    for e in list(range(-149, -120)) + list(range(-8, 9)) + list(range(118, 128)):
        for m in (1.0, 1.0 + 2 ** -23, 1.984375, 1.984375 + 2 ** -23, 2 - 2 ** -23):
            v = m * 2.0 ** e
            if v <= 3.4028234663852886e38:
                tops.append(v)
    x = torch.zeros(len(tops), 32)
    g = torch.Generator().manual_seed(1)
    x[:] = (torch.rand(len(tops), 32, generator=g, dtype=torch.float64) * 2 - 1).mul_(
        torch.tensor(tops, dtype=torch.float64)[:, None]).float()
    x[:, 7] = torch.tensor(tops, dtype=torch.float64).float()
    y = ops.unpack8(ops.pack8(x.to(DEV)))
    assert torch.equal(y.double().cpu(), restored64(x))
    assert torch.isfinite(y).all()
    z = torch.ones(4, 70)
    z[0, 40], z[1, 3], z[2, 69] = float("inf"), float("nan"), -float("inf")
    y = ops.unpack8(ops.pack8(z.to(DEV))).cpu()
    assert torch.isnan(y[0, 32:64]).all() and torch.isnan(y[1, :32]).all() and torch.isnan(y[2, 64:]).all()
    assert int(torch.isnan(y).sum()) == 32 + 32 + 6 and (y[3] == 1).all()


def test_pack8_shapes():
    ops = _ops()
    x = torch.randn(2, 3, 50, device=DEV)
    p = ops.pack8(x)
    assert ops.unpack8(p).shape == x.shape
    assert ops.unpack8(ops.pack8(x[0, 0])).shape == (50,)
    assert ops.unpack8(ops.pack8(x[:0])).shape == (0, 3, 50)
    assert torch.equal(ops.unpack8(ops.pack8(x.transpose(0, 1))), ops.unpack8(p).transpose(0, 1))


def test_checkpoint_with_a_diverged_group_gives_nan():
    ops = _ops()
    x = torch.randn(8, 64, device=DEV)
    x[2, 10] = float("inf")
    w = torch.randn(16, 64, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(ops.dense(x, w, checkpoint8=True).sum(), w)
    assert torch.isnan(g[:, :32]).all() and torch.isfinite(g[:, 32:]).all()


# ---------------------------------------------------------------------------------------------
# Long tensors, captured graphs, streams
# ---------------------------------------------------------------------------------------------
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


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("halves,act,ckpt,M,K,N", [(2, "silu", False, 700, 128, 96), (1, "gelu", True, 333, 77, 45),
                                                   (1, None, False, 40, 4096, 48)])
def test_captured_passes_replay(halves, act, ckpt, M, K, N, dtype):
    """Forward and gradients captured once; each replay on new inputs equals the eager pass bit for bit, with eager
    passes of the same operator between the replays. Two graphs share nothing."""
    ops = _ops()
    x, ws, bs, _, dy = [t.to(DEV) if torch.is_tensor(t) else [v.to(DEV) for v in t] if t else t
                        for t in _make(M, K, N, dtype, halves)]

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, *ws, *bs)]
        if halves == 2:
            y = ops.gated_linear(*leaves, act=act, checkpoint8=ckpt)
        else:
            y = ops.dense(*leaves, act=act, checkpoint8=ckpt)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    graphs = [_graph(step) for _ in range(2)]
    for k in range(3):
        x.copy_(torch.randn(M, K, device=DEV))
        dy.copy_(torch.randn(M, N, device=DEV))
        want = [t.clone() for t in step()]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_same_bits_every_time():
    """Split sums and column sums are joined in a fixed order."""
    for dtype in (F32, BF16):
        args = _make(5000, 200, 72, dtype, 2)
        first = _run(*args[:3], "silu", None, args[4])
        for _ in range(3):
            again = _run(*args[:3], "silu", None, args[4])
            assert all(torch.equal(first[k], again[k]) for k in first)


@pytest.mark.parametrize("K", [512, 520])
def test_rows_past_2_31_elements(K):
    """4.2 million rows, read in place (512 columns) and staged (520): the last rows equal the same rows alone."""
    ops = _ops()
    M = 4_200_003
    x = torch.empty(M, K, dtype=BF16, device=DEV)
    x[-70:] = torch.randn(70, K, device=DEV)
    x[:70] = torch.randn(70, K, device=DEV)
    x[70:-70] = 0.25
    w, b = torch.randn(24, K, device=DEV, dtype=BF16), torch.randn(24, device=DEV, dtype=BF16)
    y = ops.gated_linear(x, w, w * 0.5, b, b)
    for rows in (slice(0, 70), slice(M - 70, M)):
        assert torch.equal(y[rows], ops.gated_linear(x[rows].clone(), w, w * 0.5, b, b))
    assert torch.equal(y[M // 2], y[M // 2 + 1])
    p = ops.unpack8(ops.pack8(x))
    for rows in (slice(0, 70), slice(M - 70, M)):
        assert torch.equal(p[rows], ops.unpack8(ops.pack8(x[rows].clone())))
    with pytest.raises(Exception, match="2\\^22 rows"):
        ops.dense(x, w.requires_grad_())


def test_gradients_of_two_million_rows():
    """Weight and bias gradients over 2^21 + 5 rows: ones in some rows, zeros elsewhere, so the sums are exact."""
    ops = _ops()
    M, K, N = 2 ** 21 + 5, 40, 24
    x, dy = torch.zeros(M, K, dtype=BF16, device=DEV), torch.zeros(M, N, dtype=BF16, device=DEV)
    hot = torch.arange(0, M, 16411, device=DEV)
    x[hot], dy[hot] = 1, 2
    x[-1], dy[-1] = 1, 2
    w, b = torch.zeros(N, K, dtype=BF16, device=DEV, requires_grad=True), torch.zeros(N, dtype=BF16, device=DEV,
                                                                                      requires_grad=True)
    n = int((dy[:, 0] != 0).sum())
    dw, db = torch.autograd.grad(ops.dense(x, w, b), [w, b], dy)
    want = torch.full((), 2.0 * n).to(BF16)
    assert (dw.cpu() == want).all() and (db.cpu() == want).all()


def test_one_weight_twice_and_no_second_derivative():
    ops = _ops()
    x = torch.randn(30, 40, device=DEV, requires_grad=True)
    w = torch.randn(50, 40, device=DEV, requires_grad=True)
    dy = torch.randn(30, 50, device=DEV)
    a, b = w.detach().requires_grad_(), w.detach().requires_grad_()
    ga, gb = torch.autograd.grad(ops.gated_linear(x, a, b), [a, b], dy)
    assert torch.equal(torch.autograd.grad(ops.gated_linear(x, w, w), w, dy)[0], ga + gb)
    # refused where the first gradient is asked for: detached, it would drop the second-order terms unseen
    for call in (lambda: ops.dense(x, w, act="silu"), lambda: ops.dense(x, w, checkpoint8=True),
                 lambda: ops.gated_linear(x, w, w)):
        for up in (dy, dy.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="no second derivatives"):
                torch.autograd.grad(call(), x, up, create_graph=True)


def test_calls_on_other_streams():
    ops = _ops()
    x, ws, bs, _, dy = _make(900, 130, 70, F32, 2)
    want = _run(x, ws, bs, "silu", None, dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_run(x, ws, bs, "silu", None, dy))
    torch.cuda.synchronize()
    assert all(torch.equal(g[k], want[k]) for g in got for k in want)
