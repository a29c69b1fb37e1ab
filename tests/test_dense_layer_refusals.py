"""What the layers of any width and the gradient set refuse, without a GPU: every refusal comes before a launch."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from neus2_b200 import _lib as L
    from neus2_b200 import build
    build.build()
    return L, L.lib()


FAKE = 4096  # addresses that are never dereferenced
X, W, Y, DY, DX = (FAKE * k for k in (3, 5, 7, 11, 13))
INVALID, UNSUPPORTED, TOO_LARGE = -1, -2, -5


def test_linear_forward(lib):
    L, f = lib
    ok = dict(n=4, in_width=32, out_width=16, dtype=L.F16, activation=0, x=X, xs=32, w=W, b=None, r=None, rs=0, y=Y, ys=16, z=None, zs=0, ws=None, wsb=0)

    def call(**kw):
        a = dict(ok, **kw)
        d = L.LinearDesc(a["n"], a["in_width"], a["out_width"], a["dtype"], a["activation"])
        return f.neus2b_linear_forward(C.byref(d), a["x"], a["xs"], a["w"], a["b"], a["r"], a["rs"], a["y"], a["ys"], a["z"], a["zs"], a["ws"], a["wsb"], None)
    assert f.neus2b_linear_forward(None, FAKE, 32, FAKE, None, None, 0, FAKE, 16, None, 0, None, 0, None) == INVALID
    assert call(dtype=L.F32) == UNSUPPORTED and call(dtype=7) == UNSUPPORTED
    for bad in (dict(activation=4), dict(in_width=0), dict(out_width=0), dict(x=None), dict(w=None), dict(y=None), dict(xs=31), dict(ys=15), dict(r=FAKE, rs=15),
                dict(z=FAKE, zs=3), dict(x=X + 1), dict(w=W + 1), dict(b=FAKE + 1), dict(y=Y + 1), dict(r=FAKE + 1, rs=16)):
        assert call(**bad) == INVALID, bad
    B = FAKE * 2
    for bad in (dict(y=X, ys=32), dict(y=W), dict(z=Y, zs=16), dict(z=X, zs=32), dict(z=W, zs=16), dict(r=B, rs=16, z=B, zs=16),
                dict(r=Y, rs=24)):  # outputs on inputs
        assert call(**bad) == INVALID, bad
    assert call(n=(1 << 30) + 1) == TOO_LARGE and call(in_width=(1 << 30) + 1, xs=1 << 31) == TOO_LARGE
    assert call(n=0, x=None, y=None) == 0
    need = C.c_uint64(7)
    d = L.LinearDesc(500, 33, 16, L.F16, 0)
    assert f.neus2b_linear_forward_workspace(C.byref(d), 0, C.byref(need)) == 0 and need.value == 0
    assert f.neus2b_linear_forward_workspace(C.byref(d), 1, C.byref(need)) == 0 and need.value >= (500 + 16) * 40 * 2
    assert f.neus2b_linear_forward_workspace(C.byref(d), 1, None) == INVALID
    for bad in (dict(), dict(ws=FAKE), dict(ws=FAKE, wsb=need.value - 1), dict(ws=FAKE + 8, wsb=need.value)):  # copies of x and W need room
        assert call(n=500, in_width=33, xs=33, **bad) == INVALID, bad


def test_linear_backward(lib):
    L, f = lib
    ok = dict(n=4, dtype=L.BF16, activation=0, x=X, xs=32, w=W, z=None, zs=0, dy=DY, dys=16, below=0, bz=None, bzs=0, skip=None, ss=0, dx=DX,
              dxs=32, dw=FAKE, db=FAKE, mode=1, ws=None, wsb=0)

    def call(**kw):
        a = dict(ok, **kw)
        d = L.LinearDesc(a["n"], 32, 16, a["dtype"], a["activation"])
        if a["ws"] is None and "wsb" not in kw:
            need = C.c_uint64(0)
            if f.neus2b_linear_backward_workspace(C.byref(d), 0, C.byref(need)) == 0:
                a["ws"], a["wsb"] = FAKE, need.value
        return f.neus2b_linear_backward(C.byref(d), a["x"], a["xs"], a["w"], a["z"], a["zs"], a["dy"], a["dys"], a["below"], a["bz"], a["bzs"], a["skip"],
                                        a["ss"], a["dx"], a["dxs"], a["dw"], a["db"], a["mode"], a["ws"], a["wsb"], None)
    assert call(dtype=L.F32) == UNSUPPORTED
    for bad in (dict(dy=None), dict(dys=15), dict(x=None), dict(w=None), dict(dx=DX + 1), dict(dxs=31), dict(dw=FAKE + 2), dict(db=FAKE + 1), dict(mode=3),
                dict(mode=-1), dict(below=4), dict(below=2), dict(below=2, bz=FAKE, bzs=31), dict(skip=FAKE, ss=31), dict(activation=2),
                dict(activation=2, z=FAKE, zs=15), dict(activation=2, z=FAKE, zs=16, ws=FAKE, wsb=4), dict(activation=2, z=FAKE, zs=16, ws=FAKE + 8, wsb=1 << 30)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(dx=X), dict(dx=DY), dict(dx=W), dict(below=1, bz=DX, bzs=32), dict(activation=1, z=DX, zs=16), dict(skip=DX, ss=40)):  # outputs on inputs
        assert call(**bad) == INVALID, bad
    assert call(n=(1 << 30) + 1) == TOO_LARGE
    d = L.LinearDesc(4, 32, 16, L.BF16, 0)
    assert f.neus2b_linear_backward_workspace(C.byref(d), 0, None) == INVALID
    assert call(dy=DY + 2) == INVALID and call(x=X + 2) == INVALID  # the workspace has no room for their copies


def test_layer_norm(lib):
    L, f = lib

    def fwd(n=4, width=32, dtype=L.F16, pdtype=L.F16, eps=1e-5, x=FAKE, xs=32, g=FAKE, b=None, y=FAKE, ys=32, mean=None, rstd=None):
        d = L.LayerNormDesc(n, width, dtype, pdtype, eps)
        return f.neus2b_layer_norm_forward(C.byref(d), x, xs, g, b, y, ys, mean, rstd, None)
    assert fwd(dtype=3) == UNSUPPORTED and fwd(pdtype=L.BF16) == UNSUPPORTED and fwd(dtype=L.F32, pdtype=L.F16) == UNSUPPORTED
    for bad in (dict(width=0), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None), dict(g=None), dict(y=None),
                dict(xs=31), dict(ys=31), dict(x=FAKE + 1), dict(g=FAKE + 1), dict(pdtype=L.F32, g=FAKE + 2), dict(mean=FAKE), dict(rstd=FAKE),
                dict(mean=FAKE, rstd=FAKE + 1)):
        assert fwd(**bad) == INVALID, bad
    assert fwd(xs=40) == INVALID  # in place, rows elsewhere
    assert fwd(n=(1 << 31) + 1, y=FAKE * 2) == TOO_LARGE
    assert fwd(n=0, x=None, y=None) == 0

    def bwd(n=4, x=X, xs=32, g=FAKE, mean=FAKE, rstd=FAKE, dy=DY, dys=32, skip=None, ss=0, dx=DX, dxs=32, dg=FAKE, db=FAKE, mode=1, short=0):
        d = L.LayerNormDesc(n, 32, L.F16, L.F16, 1e-5)
        need = C.c_uint64(0)
        assert f.neus2b_layer_norm_backward_workspace(C.byref(d), C.byref(need)) == 0
        return f.neus2b_layer_norm_backward(C.byref(d), x, xs, g, mean, rstd, dy, dys, skip, ss, dx, dxs, dg, db, mode, FAKE, need.value - short, None)
    for bad in (dict(x=None), dict(g=None), dict(mean=None), dict(rstd=None), dict(dy=None), dict(xs=31), dict(dys=31), dict(skip=FAKE, ss=31), dict(dxs=31),
                dict(dx=X), dict(dx=DY, dxs=40), dict(skip=DX, ss=40), dict(dg=FAKE + 1), dict(mode=5), dict(mean=FAKE + 1), dict(dx=FAKE + 1)):
        assert bwd(**bad) == INVALID, bad


def test_gradient_set(lib):
    L, f = lib

    def table(*tensors, write=True):
        rows = (L.GradTensor * max(1, len(tensors)))(*[L.GradTensor(*t) for t in tensors])
        size, pieces = C.c_uint64(0), C.c_uint32(0)
        rc = f.neus2b_grad_table(rows, len(tensors), None, C.byref(size), C.byref(pieces))
        if rc == 0 and write:
            host = (C.c_char * (size.value + 1))()
            rc = f.neus2b_grad_table(rows, len(tensors), host, C.byref(size), C.byref(pieces))
        return rc, pieces.value
    A, B = 1 << 20, 1 << 24
    assert table() == (0, 0)
    assert table((None, None, 0, 0)) == (0, 0)
    rc, pieces = table((A, A, 100000, 1), (B, None, 5, 0))
    assert rc == 0 and pieces >= 2
    assert table((A, A, 4, 3))[0] == UNSUPPORTED
    for bad in ([(None, A, 4, 0)], [(A + 2, None, 4, 0)], [(A, A + 1, 4, 1)], [(A, A, 4, 0), (A, A, 4, 0)], [(A, B, 100, 0), (A, B + 396, 100, 0)],
                [(A, A + 4, 100, 0)], [(A, B, 8, 0), (B + 4, None, 8, 0)]):
        assert table(*bad)[0] == INVALID, bad
    assert table((A, B, 100, 0), (A + 4, B + 400, 100, 0))[0] == 0  # inputs may overlap
    assert table((A, None, 1 << 61, 0), write=False)[0] == -5

    def call(table=FAKE, pieces=3, scale=1.0, bound=1.0, flags=0, result=FAKE, bad=None, ws=FAKE, short=0, clip=True):
        g = f.neus2b_grad_clip if clip else f.neus2b_grad_norm
        return g(table, pieces, scale, bound, flags, result, bad, ws, f.neus2b_grad_norm_workspace(pieces) - short, None)
    for kw in (dict(table=None), dict(table=FAKE + 8), dict(scale=float("nan")), dict(scale=float("inf")), dict(bound=0.0), dict(bound=-1.0),
               dict(bound=float("nan")), dict(flags=2), dict(result=None), dict(result=FAKE + 2), dict(bad=FAKE + 1), dict(ws=None), dict(ws=FAKE + 8),
               dict(short=17)):
        assert call(**kw) == INVALID and call(clip=False, **kw) == INVALID, kw


def test_wrappers_refuse_cpu_tensors():
    from neus2_b200 import _lib as L
    from neus2_b200 import ops
    h = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    for call in (lambda: ops.linear_forward(h(4, 8), h(8, 8)), lambda: ops.linear_backward(h(4, 8), h(8, 8), h(4, 8)),
                 lambda: ops.layer_norm_forward(h(4, 8), h(8)), lambda: ops.layer_norm_backward(h(4, 8), h(8), h(4), h(4), h(4, 8)),
                 lambda: ops.GradientSet([h(4)]), lambda: ops.GradientSet([])):
        with pytest.raises(L.Neus2bError):
            call()
