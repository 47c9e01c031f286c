"""What the feed-forward operators refuse, before anything reaches a device: the Python checks on CPU tensors and
the C entry points' own argument checks."""
import ctypes

import pytest
import torch

from aimx import _lib, ops

E = _lib.AimxError
T = torch.zeros


@pytest.mark.parametrize("args,kw,said", [
    ((T(4, 8).half(), T(6, 8).half()), {}, "fp32 or bf16"),
    ((T(4, 8), T(6, 7)), {}, "weights"),
    ((T(4, 8), T(6)), {}, "weights"),
    ((T(4, 0), T(6, 0)), {}, "weights"),
    ((T(4, 8), T(6, 8), T(5)), {}, "biases"),
    ((T(4, 8), T(6, 8), T(6).bfloat16()), {}, "dtype"),
    ((T(4, 8), T(6, 8).bfloat16()), {}, "dtype"),
    ((T(4, 8), T(6, 8)), dict(residual=T(4, 8)), "residual"),
    ((T(4, 8), T(6, 8)), dict(residual=T(1, 6)), "residual"),
    ((T(4, 8), T(6, 8)), dict(act="tanh"), "act is one of"),
    ((T(4, 8), T(6, 8)), {}, "HIP device"),
])
def test_dense_refuses(args, kw, said):
    with pytest.raises(E, match=said):
        ops.dense(*args, **kw)


@pytest.mark.parametrize("args,kw,said", [
    ((T(4, 8), T(6, 8), T(5, 8)), {}, "weights"),
    ((T(4, 8), T(6, 8), T(6, 8), T(6)), {}, "both biases"),
    ((T(4, 8), T(6, 8), T(6, 8)), dict(act=None), "act names"),
    ((T(4, 8), T(6, 8), T(6, 8)), {}, "HIP device"),
])
def test_gated_refuses(args, kw, said):
    with pytest.raises(E, match=said):
        ops.gated_linear(*args, **kw)


def test_pack8_refuses():
    for x in (T(4, 8).double(), T(4, 8).long()):
        with pytest.raises(E, match="fp32 or bf16"):
            ops.pack8(x)
    for x in (T(4, 0), torch.tensor(1.0)):
        with pytest.raises(E, match="last dimension"):
            ops.pack8(x)
    with pytest.raises(E, match="HIP device"):
        ops.pack8(T(4, 8))
    with pytest.raises(E, match="fp32 or bf16"):
        ops.unpack8(ops.Packed8(T(1, 32).char(), T(1, 1).char(), (1, 20), torch.float32), torch.float16)


@pytest.mark.parametrize("args,said", [
    ((T(3).long(), T(4)), "table"),
    ((T(3).long(), T(4, 2).half()), "table"),
    ((T(3).long(), T(0, 2)), "table"),
    ((T(3), T(4, 2)), "integer"),
    ((T(3).bool(), T(4, 2)), "integer"),
    ((T(3).long(), T(4, 2), 1.0, 4), "padding_idx"),
    ((T(3).long(), T(4, 2), 1.0, -5), "padding_idx"),
    ((T(3).long(), T(4, 2)), "HIP device"),
])
def test_embedding_refuses(args, said):
    with pytest.raises(E, match=said):
        ops.embedding(*args)


def _dense(**kw):
    d = _lib.Dense()
    d.M, d.N, d.K, d.halves, d.act, d.dtype = 4, 8, 16, 1, -1, 0
    d.x, d.ldx, d.w[0], d.ldw, d.y, d.ldy = 4096, 16, 8192, 16, 16384, 8
    d.workspace, d.workspace_bytes = 1 << 20, 1 << 30
    for k, v in kw.items():
        if k in ("w0", "w1"):
            d.w[int(k[1])] = v
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(N=0), dict(K=0), dict(halves=0), dict(halves=3), dict(act=5), dict(act=-2), dict(dtype=2),
    dict(precision=2), dict(x=None), dict(y=None), dict(w0=None), dict(halves=2, act=4), dict(halves=2, w1=8192),
    dict(ldx=15), dict(ldw=15), dict(ldy=7), dict(res=4096, ldr=7), dict(halves=2, w1=8192, act=4, res=4096, ldr=8),
    dict(workspace_bytes=0), dict(workspace=None), dict(workspace=(1 << 20) + 4), dict(ldx=(1 << 21) + 1),
    dict(K=(1 << 21) + 1, ldx=1 << 22, ldw=1 << 22), dict(N=(1 << 21) + 1, ldy=1 << 22)])
def test_c_dense_refuses(kw):
    assert _lib.load().aimx_dense_forward(ctypes.byref(_dense(**kw)), None) == -1


@pytest.mark.parametrize("kw,gk", [
    (dict(), dict(dy=None)), (dict(), dict(ldd=7)), (dict(), dict(lddx=15)), (dict(x=None), {}),
    (dict(x=None, q=4096), {}), (dict(M=(1 << 22) + 1), {}), (dict(halves=2, w1=8192, act=4), {}),
    (dict(), dict(workspace_bytes=0)), (dict(), dict(workspace=None)), (dict(ldx=3), {})])
def test_c_dense_backward_refuses(kw, gk):
    g = _lib.DenseGrad()
    g.dy, g.ldd, g.dx, g.lddx, g.workspace, g.workspace_bytes = 4096, 8, 8192, 16, 1 << 20, 1 << 34
    g.dw[0] = 16384
    for k, v in gk.items():
        setattr(g, k, v)
    assert _lib.load().aimx_dense_backward(ctypes.byref(_dense(**kw)), ctypes.byref(g), None) == -1


def test_c_pack8_refuses():
    lib = _lib.load()
    good = [0, 4096, 32, 4, 32, 8192, 16384, None]
    for i, v in ((0, 2), (1, None), (2, 31), (3, -1), (4, 0), (5, None), (5, 8196), (6, None)):
        assert lib.aimx_pack8(*[v if j == i else a for j, a in enumerate(good)]) == -1, (i, v)
    good = [0, 4096, 8192, 4, 32, 16384, 32, None]
    for i, v in ((0, 2), (1, None), (1, 4100), (2, None), (3, -1), (4, 0), (5, None), (6, 31)):
        assert lib.aimx_unpack8(*[v if j == i else a for j, a in enumerate(good)]) == -1, (i, v)
    assert lib.aimx_pack8(0, None, 32, 0, 32, None, None, None) == 0


def test_c_embedding_refuses():
    lib = _lib.load()
    good = [0, 4096, 4, 8192, 10, 8, 1.0, 16384, None]
    for i, v in ((0, 2), (1, None), (2, -1), (2, 2 ** 31), (3, None), (4, 0), (4, 2 ** 31), (5, 0), (7, None)):
        assert lib.aimx_token_embedding_forward(*[v if j == i else a for j, a in enumerate(good)]) == -1, (i, v)
    good = [0, 4096, 4, 8192, 8, 10, 8, 1.0, -1, 16384, 1 << 20, 1 << 30, None]
    for i, v in ((0, 2), (1, None), (2, -1), (3, None), (4, 7), (5, 0), (6, 0), (9, None), (9, 16388), (10, None),
                 (10, (1 << 20) + 4), (11, 0)):
        assert lib.aimx_token_embedding_backward(*[v if j == i else a for j, a in enumerate(good)]) == -1, (i, v)
    assert lib.aimx_token_embedding_backward_workspace_bytes(0, 1000, 50, 64) > 0


def test_modules():
    from models import GatedBlock, ScaledEmbedding
    b = GatedBlock(8, 20, 8, bias=False)
    assert sorted(b.state_dict()) == ["down.weight", "gate.weight", "up.weight"] and b.use_skip
    assert not GatedBlock(8, 20, 9).use_skip
    with pytest.raises(ValueError):
        GatedBlock(8, 20, 8, activation_type="tanh")
    with pytest.raises(ValueError):
        ScaledEmbedding(4, 2, sparse=True)
    assert ScaledEmbedding(4, 2, padding_idx=1).padding_idx == 1


def test_struct_layouts_match_header():
    import os
    import re

    from conftest import ROOT
    src = open(os.path.join(ROOT, "include", "aimx.h")).read()
    for cname, py in (("AimxDense", _lib.Dense), ("AimxDenseGrad", _lib.DenseGrad)):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{([^{}]*)\} %s;" % (cname, cname), src, re.S).group(1),
                      flags=re.S)
        assert re.findall(r"\**\s*(\w+)\s*(?:\[[^\]]*\])?\s*[;,]", body) == [f[0] for f in py._fields_]
