"""The feed-forward operators where values, layouts and modes are unusual: NaN and infinities in front of an
activation, forward-mode derivatives, tracing, long row strides. Bounds as in tests/ffn_bounds.py."""
import pytest
import torch

from ffn_bounds import act64, dact64

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
ACTS = ["relu", "leakyrelu", "elu", "gelu", "silu"]


def _ops():
    from aimx import ops
    return ops


def _finite_or(a, b):
    """NaN where b is NaN, the same infinities, finite elsewhere."""
    a, b = a.detach().double().cpu(), b.double()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isposinf(), b.isposinf()) and \
        torch.equal(a.isneginf(), b.isneginf())


# (70, 96, 40): at most 65536 values before the activation; (1100, 64, 200): more, N no multiple of 64
SHAPES = [(70, 96, 40), (1100, 64, 200)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("act", ACTS)
def test_nan_passes_every_activation(act, M, K, N, dtype):
    """A row of x with a NaN gives a row of NaN, whatever the activation, in both products; no other row does."""
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    x = torch.randn(M, K, generator=g).to(dtype)
    w, u = [(torch.randn(N, K, generator=g) * K ** -0.5).to(dtype).to(DEV) for _ in range(2)]
    x[3, 5] = x[M - 1, K - 1] = float("nan")
    hit = torch.zeros(M, dtype=torch.bool)
    hit[[3, M - 1]] = True
    xd = x.to(DEV)
    for y in (ops.dense(xd, w, act=act), ops.dense(xd, w, act=act, residual=torch.ones(M, N, dtype=dtype, device=DEV)),
              ops.gated_linear(xd, w, u, act=act)):
        nan = y.isnan().cpu()
        assert nan[hit].all() and not nan[~hit].any()
    # a gate that is infinite, u of either sign: what the definition gives where the product itself is exact
    if dtype == BF16:
        x[3, 5], x[M - 1, K - 1] = float("inf"), -float("inf")
        want = act64(act, x.double() @ w.cpu().double().t())
        got = ops.dense(x.to(DEV), w, act=act)
        # silu and gelu of -inf are 0 * inf, NaN by the formula: not asked for
        fin = ~torch.isnan(want)
        assert _finite_or(torch.where(fin, got.cpu(), 0), torch.where(fin, want, 0))


def test_overflow_is_not_swallowed():
    """An infinite fp32 activation may make NaN in the three-part product, and relu keeps the row from looking finite."""
    ops = _ops()
    x = torch.randn(40, 64, device=DEV)
    x[7, 9] = float("inf")
    w = torch.rand(30, 64, device=DEV) + 0.5  # every value of row 7 is infinite
    for y in (ops.dense(x, w, act="relu"), ops.gated_linear(x, w, w, act="relu")):
        assert not torch.isfinite(y[7]).any()
        assert torch.isfinite(y[:7]).all() and torch.isfinite(y[8:]).all()


def test_relu_of_nan_in_the_layer_products():
    """The framework's own fp32 products use the same activation: nn.ReLU keeps a NaN too."""
    ops = _ops()
    x = torch.randn(70, 64, device=DEV)
    x[3, 5] = float("nan")
    w, b = torch.randn(48, 64, device=DEV), torch.randn(48, device=DEV)
    y = ops.linear(x, w, b, act="relu")
    want = torch.relu(x.cpu() @ w.cpu().t() + b.cpu())
    assert torch.equal(y.isnan().cpu(), want.isnan()) and int(y.isnan().sum()) == 48


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("act", ["relu", "leakyrelu", "elu"])
def test_infinite_rows_keep_finite_gradients(act, ckpt, dtype):
    """A row of x with an infinity: relu', leakyrelu' and elu' of plus and minus infinity are finite, and so is dx,
    whatever N (columns that pad dP to 64 stay out of it). fp32's three-part product and the 8-bit form make NaN of
    the row itself; every other row stays finite in each."""
    ops = _ops()
    for M, K, N in ((1100, 64, 200), (1100, 64, 192), (700, 72, 101), (70, 96, 40)):
        g = torch.Generator().manual_seed(N)
        x = torch.randn(M, K, generator=g).to(dtype)
        w = (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype)
        w[w == 0] = 0.01
        dy = torch.randn(M, N, generator=g).to(dtype)
        x[3, 5] = float("inf")
        xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        dx, dw = torch.autograd.grad(ops.dense(xd, wd, act=act, checkpoint8=ckpt), [xd, wd], dy.to(DEV))
        rows = [i for i in range(M) if i != 3]
        assert torch.isfinite(dx[rows]).all()
        if dtype == BF16 and not ckpt:
            assert torch.isfinite(dx).all(), (M, K, N)
            p = x.double() @ w.double().t()
            want = (dy.double() * dact64(act, p)) @ w.double()
            # two roundings to bf16, of dP and of dx, and fp32 sums
            mag = (dy.double() * dact64(act, p)).abs() @ w.double().abs()
            assert ((dx.double().cpu() - want).abs() <= 2.0 ** -8 * (mag + want.abs()) * 1.01)[3].all()


def test_lookup_out_of_range_is_zero_at_any_scale():
    ops = _ops()
    index = torch.tensor([0, 9, -1, 2], device=DEV)
    for dtype in (F32, BF16):
        table = torch.randn(4, 24, device=DEV).to(dtype)
        for scale in (float("inf"), float("nan"), -2.0):
            y = ops.embedding(index, table, scale)
            assert (y[1] == 0).all() and (y[2] == 0).all()


def test_forward_mode_is_refused():
    """No tangent leaves these operators: a dual input raises, in whichever argument it stands, and plain inputs inside a
    dual level work."""
    import torch.autograd.forward_ad as fw
    ops = _ops()
    x, w, b = torch.randn(20, 32, device=DEV), torch.randn(24, 32, device=DEV), torch.randn(24, device=DEV)
    index, table = torch.randint(0, 9, (12,), device=DEV), torch.randn(9, 16, device=DEV)
    want = ops.dense(x, w, b, act="silu"), ops.gated_linear(x, w, w), ops.embedding(index, table)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.dense(dual(x), w, b), lambda: ops.dense(x, dual(w), b), lambda: ops.dense(x, w, dual(b)),
                     lambda: ops.dense(x, w, b, residual=dual(want[0])), lambda: ops.gated_linear(x, w, dual(w)),
                     lambda: ops.embedding(index, dual(table))):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()
        got = ops.dense(x, w, b, act="silu"), ops.gated_linear(x, w, w), ops.embedding(index, table)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traced_calls_run_again():
    ops = _ops()
    w, u, b = torch.randn(24, 32, device=DEV), torch.randn(24, 32, device=DEV), torch.randn(24, device=DEV)
    table = torch.randn(9, 16, device=DEV)
    for fn, make in ((lambda x: ops.dense(x, w, b, act="gelu"), lambda: torch.randn(20, 32, device=DEV)),
                     (lambda x: ops.gated_linear(x, w, u), lambda: torch.randn(20, 32, device=DEV)),
                     (lambda i: ops.embedding(i, table, 2.0), lambda: torch.randint(0, 9, (20,), device=DEV))):
        traced = torch.jit.trace(fn, (make(),), check_trace=False)
        for _ in range(3):
            v = make()
            assert torch.equal(traced(v), fn(v))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_far_apart(dtype):
    """Row strides over 2^21 elements are copied, in the inputs and in the gradient that autograd hands in."""
    ops = _ops()
    wide = torch.randn(3, 2 ** 21 + 72, device=DEV).to(dtype)
    w, u = torch.randn(24, 40, device=DEV).to(dtype), torch.randn(24, 40, device=DEV).to(dtype)
    r, dy, x = wide[:, 64:88], wide[:, 128:152], wide[:, 3:43]
    assert x.stride(0) > 2 ** 21 and dy.stride(0) > 2 ** 21

    def run(x, r, dy):
        xs, ws, us, rs = [t.detach().requires_grad_() for t in (x, w, u, r)]
        y = ops.dense(xs, ws, act="silu", residual=rs)
        h = ops.gated_linear(xs, ws, us)
        return [y, h, *torch.autograd.grad(y, [xs, ws, rs], dy), *torch.autograd.grad(h, [xs, ws, us], dy)]

    for rows in (slice(0, 3), slice(1, 2)):
        a, c, d = x[rows], r[rows], dy[rows]
        assert all(torch.equal(p, q) for p, q in zip(run(a, c, d), run(a.clone(), c.clone(), d.clone())))
    emb = torch.randn(5, 24, device=DEV).to(dtype).requires_grad_()
    index = torch.tensor([1, 4, 1], device=DEV)
    y = ops.embedding(index, emb)
    assert torch.equal(torch.autograd.grad(y, emb, dy, retain_graph=True)[0], torch.autograd.grad(y, emb, dy.clone())[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pack8_error_bound(dtype):
    """Values come back within max(top / 127, 2^-127) of themselves, top the group's largest; within 2^122 where top is
    above 127 * 2^121. Both ends pass top / 127 alone: 2^-128 comes back as 0, the largest floats 2^122 off."""
    ops = _ops()
    g = torch.Generator().manual_seed(2)
    tops = torch.exp2(torch.cat([torch.linspace(-149, -100, 99), torch.linspace(-99, 127.99, 500),
                                 torch.linspace(127.9, 127.999, 30)]).double()).float().to(dtype)
    x = (torch.rand(len(tops), 32, generator=g, dtype=torch.float64) * 2 - 1).mul_(tops.double()[:, None]).to(dtype)
    x[:, 3] = tops
    x = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    v, top = x.double(), x.double().abs().amax(1, keepdim=True)
    err = (ops.unpack8(ops.pack8(x.to(DEV))).double().cpu() - v).abs()
    bound = torch.where(top > 127 * 2.0 ** 121, torch.full_like(top, 2.0 ** 122), (top / 127).clamp(min=2.0 ** -127))
    assert (err <= bound).all()
    past = (err > top / 127).any(1)
    assert past[top[:, 0] < 2.0 ** -127].any() and past[top[:, 0] > 127 * 2.0 ** 121].any()
    assert not past[(top[:, 0] > 2.0 ** -120) & (top[:, 0] <= 127 * 2.0 ** 121)].any()


@pytest.mark.parametrize("low,high", [(-110, -60), (-140, -110)])
def test_small_magnitudes_fp32(low, high):
    """Three bf16 parts are an fp32 value down to 2^-110, where the last bit of the third is bf16's least subnormal
    2^-133; below, their sum is off by at most half of that. Either operand of the forward product and of both
    gradient products small, the other around 2^30."""
    g = torch.Generator().manual_seed(-low)

    def small(*s):
        v = (torch.rand(*s, generator=g) + 1) * torch.exp2(torch.randint(low, high, s, generator=g).float())
        return torch.where(torch.rand(*s, generator=g) < 0.5, v, -v)

    lost = 2.0 ** -134 if low < -110 else 0.0
    ops = _ops()
    for M, K, N in ((40, 96, 50), (130, 200, 70)):
        large = lambda *s: torch.randn(*s, generator=g) * 2.0 ** 30  # noqa: E731

        def check(got, a, b):  # got = a b^T, a small
            a, b = a.double(), b.double()
            bound = ((a.shape[1] + 16) * 2.0 ** -24 * a.abs() + lost) @ b.t().abs() + 2.0 ** -24 * (a @ b.t()).abs()
            assert ((got.double().cpu() - a @ b.t()).abs() <= bound).all(), (M, K, N)

        x, w = small(M, K), large(N, K)
        check(ops.dense(x.to(DEV), w.to(DEV)), x, w)
        check(ops.dense(w.to(DEV), x.to(DEV)).t(), x, w)  # the small operand as the weight
        dy, x = small(M, N), large(M, K)
        xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
        dx, dw = torch.autograd.grad(ops.dense(xs, ws), [xs, ws], dy.to(DEV))
        check(dx, dy, w.t())
        check(dw, dy.t(), x.t())
        dx, dw = torch.autograd.grad(ops.dense(xs, ws, checkpoint8=True), [xs, ws], dy.to(DEV))
        check(dx, dy, w.t())
