"""What the feed-forward operators decide on the host, on CPU tensors with the launches recorded in place of run:
which tensors reach a kernel, what is kept for a backward, and what is refused before a kernel could read memory that
is not there."""
import ctypes

import pytest
import torch

from aimx import _lib, ops

E = _lib.AimxError


@pytest.fixture
def launches(monkeypatch):
    """[(what, C arguments)] of every call that would have been enqueued."""
    seen = []
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    monkeypatch.setattr(ops, "_launch", lambda device, what, fn, *args: seen.append((what, args)))
    return seen


def _packed(m=3, k=50, shape=None, q=None, exps=None):
    kq = -(-k // 32) * 32
    q = torch.zeros(m, kq, dtype=torch.int8) if q is None else q
    exps = torch.zeros(m, kq // 32, dtype=torch.int8) if exps is None else exps
    return ops.Packed8(q, exps, (m, k) if shape is None else shape, torch.float32)


I8 = torch.int8


@pytest.mark.parametrize("bad", [
    dict(shape=(3, 70)), dict(shape=(4, 50)), dict(shape=(2, 50)), dict(shape=(3, 2, 50)), dict(shape=(150,)), dict(shape=()),
    dict(shape=(3, 0)), dict(q=torch.zeros(3, 32, dtype=I8)), dict(q=torch.zeros(192, dtype=I8)), dict(q=torch.zeros(3, 64)),
    dict(q=torch.zeros(64, 3, dtype=I8).t()), dict(q=torch.zeros(3, 128, dtype=I8)[:, :64]),
    dict(exps=torch.zeros(3, 1, dtype=I8)), dict(exps=torch.zeros(2, 2, dtype=I8)), dict(exps=torch.zeros(3, 2)),
    dict(exps=torch.zeros(3, 4, dtype=I8)[:, ::2]), dict(exps=torch.zeros(3, 2, dtype=I8, device="meta"))])
def test_unpack8_refuses_parts_that_do_not_fit(bad, launches):
    """The kernel reads as many bytes as the shape asks for: q and exps have to hold them."""
    with pytest.raises(E, match="unpack8"):
        ops.unpack8(_packed(**bad))
    assert not launches


def test_unpack8_takes_what_pack8_makes(launches):
    assert ops.unpack8(_packed()).shape == (3, 50)
    assert ops.unpack8(_packed(6, 50, (2, 3, 50))).shape == (2, 3, 50)
    assert ops.unpack8(_packed(1, 50, (50,))).shape == (50,)
    assert ops.unpack8(_packed(0, 50, (0, 4, 50))).shape == (0, 4, 50)
    for shape in ((4, 33), (2, 0, 5), (7,)):
        assert ops.unpack8(ops.pack8(torch.zeros(shape))).shape == shape


def test_unpack8_refuses_host_memory():
    """A form moved to the host (to offload it) is brought back by the caller: a kernel cannot read it there."""
    with pytest.raises(E, match="HIP device"):
        ops.unpack8(_packed())


def _calls():
    """One call of each differentiable operator, as a function of each of its tensors."""
    x, w, b, r, t = torch.randn(4, 64), torch.randn(8, 64), torch.randn(8), torch.randn(4, 8), torch.randn(9, 16)
    index = torch.tensor([1, 4])
    return [(x, lambda v: ops.dense(v, w, b)), (w, lambda v: ops.dense(x, v)), (b, lambda v: ops.dense(x, w, v)),
            (r, lambda v: ops.dense(x, w, residual=v, act="silu")), (x, lambda v: ops.gated_linear(v, w, w)),
            (w, lambda v: ops.gated_linear(x, w, v, checkpoint8=True)), (t, lambda v: ops.embedding(index, v, 2.0))]


def test_forward_mode_raises_instead_of_dropping_the_tangent(launches):
    import torch.autograd.forward_ad as fw
    for v, call in _calls():
        with fw.dual_level():
            with pytest.raises(NotImplementedError, match="jvp"):
                call(fw.make_dual(v, torch.ones_like(v)))
            assert call(v) is not None  # no tangent: nothing to refuse
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (v,), (v,))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_traces_record_the_call(launches):
    """torch.jit.trace holds the operator itself, not the allocation of its result."""
    for v, call in _calls():
        graph = str(torch.jit.trace(call, (v,), check_trace=False).graph)
        assert ("^_DenseFn" in graph) != ("^_Embedding" in graph) and "aten::empty" not in graph
    index = torch.tensor([1, 4])
    assert "^_Embedding" in str(torch.jit.trace(lambda i: ops.embedding(i, torch.zeros(9, 16)), (index,),
                                                check_trace=False).graph)
    packed = ops.pack8(torch.zeros(4, 64))
    for fn in (lambda v: ops.unpack8(ops.pack8(v)), lambda v: v + ops.unpack8(packed)):
        with pytest.raises(E, match="torch.jit.trace"):
            torch.jit.trace(fn, (torch.zeros(4, 64),), check_trace=False)


def test_long_row_strides_are_copied(launches):
    """No layout of x, the residual or the incoming gradient is refused; what reaches the C entry keeps its limit."""
    far = 2 ** 21 + 8

    def rows(m, k):
        return torch.empty_strided((m, k), (far, 1))

    w, w2 = torch.randn(8, 16, requires_grad=True), torch.randn(8, 16)
    for m in (1, 2, 3):
        for x, r in ((rows(m, 16), None), (torch.randn(m, 16), rows(m, 8)), (rows(m, 16)[None], rows(m, 8)[None])):
            launches.clear()
            ys = [ops.dense(x, w, residual=r), ops.dense(x, w2, residual=r)] + ([ops.gated_linear(x, w, w)] if r is None else [])
            for y in ys:
                if y.requires_grad:
                    torch.autograd.grad(y, w, rows(m, 8).view(y.shape))
            kinds = [what for what, _ in launches]
            assert kinds.count("dense_forward") == len(ys) and kinds.count("dense_backward") == len(ys) - 1
            for what, args in launches:
                d = args[0]._obj
                assert d.M == m and 16 <= d.ldx <= 2 ** 21 and (not d.res or 8 <= d.ldr <= 2 ** 21)
                if what == "dense_backward":
                    assert 8 <= args[1]._obj.ldd <= 2 ** 21


def test_a_residual_alone_keeps_nothing(launches):
    """The residual's gradient is the incoming one: no input is kept for it, packed or held to the rows of a backward."""
    x, w, r = torch.randn(4, 64), torch.randn(8, 64), torch.randn(4, 8, requires_grad=True)
    dy = torch.randn(4, 8)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        for kw in (dict(act="silu"), dict(checkpoint8=True)):
            assert torch.equal(torch.autograd.grad(ops.dense(x, w, residual=r, **kw), r, dy)[0], dy)
    assert not kept and [what for what, _ in launches] == ["dense_forward"] * 2
    many = torch.empty(1, dtype=torch.bfloat16).expand(2 ** 22 + 1, 1)
    ops.dense(many, many[:1], residual=torch.empty(1, dtype=torch.bfloat16, requires_grad=True).expand(2 ** 22 + 1, 1))
    with pytest.raises(E, match="2\\^22 rows"):
        ops.dense(many, torch.empty(1, 1, dtype=torch.bfloat16, requires_grad=True))
    # beside other gradients it is still dy
    ws = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.dense(x, ws, residual=r), [ws, r], dy)[1], dy)
    assert launches[-1][0] == "dense_backward"


def test_c_products_refuse_more_work_items_than_a_dispatch_counts():
    """2^32 work items in a dimension: refused here, before the launch, not left to the runtime."""
    lib = _lib.load()
    d = _lib.Dense()
    d.M, d.N, d.K, d.halves, d.act, d.dtype = 2 ** 36, 64, 64, 1, -1, 1
    d.x, d.ldx, d.w[0], d.ldw, d.y, d.ldy = 4096, 64, 8192, 64, 16384, 64
    assert lib.aimx_dense_workspace_bytes(ctypes.byref(d)) == 0  # read in place: the product is the first launch
    assert lib.aimx_dense_forward(ctypes.byref(d), None) == -1
    d.M, d.N, d.K, d.dtype = 2 ** 22, 2 ** 21, 2 ** 21, 0  # db alone: the column sums of dy
    d.ldx = d.ldw = d.ldy = 2 ** 21
    g = _lib.DenseGrad()
    g.dy, g.ldd, g.db[0], g.workspace, g.workspace_bytes = 4096, 2 ** 21, 8192, 1 << 20, 1 << 62
    assert lib.aimx_dense_backward(ctypes.byref(d), ctypes.byref(g), None) == -1
