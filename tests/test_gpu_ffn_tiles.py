"""Every tile of the dense and gated products with every epilogue and operand order, over one stage of k and many, in one
range of k and several, at sizes that end inside a tile (the estimate would take the large tiles at large
sizes only). Bounds as in tests/ffn_bounds.py."""
import functools

import pytest
import torch

from ffn_bounds import outside, product64, restored64

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16

# M, K, N; what each product of it takes for k: forward K, dx N (gated: twice), dW M. One of them or more is summed in
# several ranges at each shape but the first; each has more than 65536 values before the activation.
SHAPES = [(300, 136, 270), (1030, 64, 520), (513, 1000, 152), (97, 520, 1000), (2500, 200, 136)]
MODES = ["bf16", "fp32", "autocast"]
OPERATORS = [(1, None), (1, "gelu"), (2, "silu")]


@functools.lru_cache(maxsize=2)
def _case(M, K, N, mode, halves, act, ckpt):
    """Inputs and, in 64 bits, every result with its bound."""
    g = torch.Generator().manual_seed(M + K + N)
    dtype = BF16 if mode == "bf16" else F32
    rnd = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    x, dy = rnd(M, K), rnd(M, N)
    ws = [(rnd(N, K).float() * K ** -0.5).to(dtype) for _ in range(halves)]
    bs, res = [rnd(N) for _ in range(halves)], rnd(M, N) if halves == 1 else None
    # inside autocast: operands rounded to bf16, everything else fp32
    as_read = (lambda t: t.to(BF16)) if mode == "autocast" else (lambda t: t)
    ref = product64(as_read(x), [as_read(w) for w in ws], bs, act, res, dy, F32 if mode == "fp32" else BF16,
                    restored64(x) if ckpt else None)
    return (x, ws, bs, res, dy), ref


def _step(ops, inputs, act, ckpt):
    """Forward and every gradient."""
    x, ws, bs, res, dy = inputs
    leaf = lambda t: t.to(DEV).requires_grad_()  # noqa: E731
    x, ws, bs = leaf(x), [leaf(w) for w in ws], [leaf(b) for b in bs]
    if len(ws) == 2:
        y = ops.gated_linear(x, *ws, *bs, act=act, checkpoint8=ckpt)
    else:
        y = ops.dense(x, ws[0], bs[0], act=act, residual=res.to(DEV), checkpoint8=ckpt)
    names = ["dx"] + [f"dw{i}" for i in range(len(ws))] + [f"db{i}" for i in range(len(ws))]
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, [x, *ws, *bs], dy.to(DEV))))}


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("halves,act", OPERATORS)
@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("tile", [0, 1, 2])
def test_tiles(shape, mode, halves, act, ckpt, tile):
    from aimx import _lib, ops
    inputs, (val, tol) = _case(*shape, mode, halves, act, ckpt)
    with _lib.options(AIMX_DENSE_TILE=tile, AIMX_DENSE_SPLIT_TILE=tile), torch.autocast("cuda", BF16, mode == "autocast"):
        got = _step(ops, inputs, act, ckpt)
        again = _step(ops, inputs, act, ckpt)
    assert not outside(got, val, tol), outside(got, val, tol)
    assert all(v.dtype == inputs[0].dtype for v in got.values())
    assert all(torch.equal(got[k], again[k]) for k in got)  # fixed order of every sum


@pytest.mark.parametrize("tile", [0, 1, 2])
def test_bare_forward_of_every_tile(tile):
    """No gradient asked for, no bias: the same tiles without the values before the activation."""
    from aimx import _lib, ops
    for M, K, N in SHAPES:
        for dtype in (BF16, F32):
            (x, ws, _, _, _), _ = _case(M, K, N, "bf16" if dtype == BF16 else "fp32", 2, "silu", False)
            val, tol = product64(x, ws, [None, None], "silu", None, None, dtype)
            with _lib.options(AIMX_DENSE_TILE=tile, AIMX_DENSE_SPLIT_TILE=tile):
                got = {"y": ops.gated_linear(x.to(DEV), *[w.to(DEV) for w in ws])}
            assert not outside(got, val, tol), (M, K, N, dtype, outside(got, val, tol))


def test_tile_options_out_of_range_are_ignored():
    from aimx import _lib, ops
    x, w = torch.randn(40, 64, device=DEV, dtype=BF16), torch.randn(24, 64, device=DEV, dtype=BF16)
    want = ops.dense(x, w), ops.dense(x.float(), w.float())
    for bad in (-2, 3, 1 << 40):
        with _lib.options(AIMX_DENSE_TILE=bad, AIMX_DENSE_SPLIT_TILE=bad):
            assert torch.equal(ops.dense(x, w), want[0]) and torch.equal(ops.dense(x.float(), w.float()), want[1])


@pytest.mark.parametrize("halves", [1, 2])
@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("tile", [-1, 0, 1, 2])
def test_fp32_products_hold_all_24_bits(tile, ckpt, halves):
    """One value in each row of x and of dy, no two of dy in a column: every sum has one term (dx of the gated product
    two), zeros add exactly, and the length of k drops out. A product of three-part operands is then off by 2 u for what
    is left out and u for each of the up to six additions; a missing part product leaves 127 u or more somewhere.
    gated: relu of a positive gate, h = g u', dG = dy u', dU = dy g, so two products and three more roundings stand
    behind one another in the gradients; all factors are positive, so the magnitudes are the values."""
    from aimx import _lib, ops
    for M, K, N in SHAPES:
        g = torch.Generator().manual_seed(M)
        rnd = lambda *s: torch.rand(*s, generator=g) + 0.5  # noqa: E731
        x, dy = torch.zeros(M, K), torch.zeros(M, N)
        x[torch.arange(M), torch.randint(0, K, (M,), generator=g)] = rnd(M)
        rows = torch.randperm(M, generator=g)[:min(M, N)]
        dy[rows, torch.randperm(N, generator=g)[:len(rows)]] = rnd(len(rows))
        ws = [rnd(N, K) for _ in range(halves)]
        leaves = [t.to(DEV).requires_grad_() for t in (x, *ws)]
        with _lib.options(AIMX_DENSE_SPLIT_TILE=tile):
            y = ops.gated_linear(*leaves, act="relu", checkpoint8=ckpt) if halves == 2 else \
                ops.dense(*leaves, checkpoint8=ckpt)
            got = [y.detach(), *torch.autograd.grad(y, leaves, dy.to(DEV))]
        xd, kept, d, wd = x.double(), restored64(x) if ckpt else x.double(), dy.double(), [w.double() for w in ws]
        if halves == 2:
            p, q = [kept @ w.t() for w in wd]
            dp = [d * q, d * p]
            want = [(xd @ wd[0].t()) * (xd @ wd[1].t()), dp[0] @ wd[0] + dp[1] @ wd[1], dp[0].t() @ kept, dp[1].t() @ kept]
        else:
            want = [xd @ wd[0].t(), d @ wd[0], d.t() @ kept]
        for name, a, b in zip(("y", "dx", "dw0", "dw1"), got, want):
            worst = float(((a.double().cpu() - b).abs() / b.clamp(min=1e-30)).max()) * 2.0 ** 24
            assert worst <= (8 if halves == 1 else 20), (M, K, N, name, worst)
