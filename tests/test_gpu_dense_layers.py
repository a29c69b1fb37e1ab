"""Linear layers, layer norm and gradient clipping (any width) against 64-bit restatements."""
import ctypes as C
import math

import pytest
import torch

import dense_reference as R

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from neus2_b200 import ops as o
    return o


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(g, n, width, t, scale=1.0, pad=0, offset=0):
    """[n][width] values cut out of rows of width + pad entries, `offset` entries behind the buffer's start."""
    full = torch.empty(offset + n * (width + pad), device="cuda").normal_(0.0, scale, generator=g).to(t)
    return full[offset:].view(n, width + pad)[:, :width]


def framed(n, width, t, pad):
    """An output inside a larger buffer full of a marker, and a check that nothing around it was written."""
    full = torch.full((n + 2, width + pad), 77.0, dtype=t, device="cuda")
    out = full[1:n + 1, :width]

    def untouched():
        keep = full.clone()
        keep[1:n + 1, :width] = 77.0
        return bool((keep == 77.0).all())
    return out, untouched


#        n, in, out
SHAPES = [(1, 1, 1), (1, 16, 16), (2, 7, 5), (1, 4096, 264), (7, 1024, 129), (16, 2048, 64), (17, 48, 64), (33, 333, 77), (64, 520, 1000),
          (65, 128, 256), (128, 64, 128), (129, 1000, 333), (200, 8, 2048), (257, 72, 520), (700, 31, 3), (1000, 4100, 24), (3000, 48, 64),
          (5000, 64, 16), (512, 2048, 1536), (2600, 136, 2100), (9472, 23, 512), (100, 40, 37888), (1500, 128, 40),
          (1111, 56, 120), (300, 8, 100), (100000, 64, 64), (3, 24, 40000), (50, 7, 38000), (100, 520, 512), (300, 2056, 120), (5000, 513, 947), (70, 40, 7000),
          (20, 6000, 130), (6000, 8192, 300), (8192, 2100, 600), (8192, 2100, 1030)]


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear_forward(ops, shape, t):
    n, i, o = shape
    g = gen(n * 7 + i)
    w = (torch.empty((o, i), device="cuda").uniform_(-1, 1, generator=g) * math.sqrt(6.0 / (i + o))).to(t)
    b = rows(g, 1, o, t, 0.3)[0]
    for k, (kind, pad, offset, bias, residual) in enumerate([(R.NONE, 0, 0, False, False), (R.RELU, 0, 0, True, False), (R.GELU, 8, 0, True, True),
                                                              (R.SILU, 3, 1, True, True), (R.GELU, 8, 8, False, True)]):
        x = rows(g, n, i, t, 1.0, pad, offset)
        r = rows(g, n, o, t, 1.0, pad, offset) if residual else None
        y, untouched = framed(n, o, t, pad + (8 if k % 2 else 0))
        bb = b if bias else None
        got = ops.linear_forward(x, w, bb, r, kind, out=y, want_preact=k >= 2)
        want, z, ey, ez = R.linear(x, w, bb, r, kind, t)
        R.within(f"y {k}", y, want, ey)
        assert untouched(), k
        if k >= 2:
            R.within(f"z {k}", got[1], z, ez)


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear_backward(ops, shape, t):
    from neus2_b200 import _lib as L
    n, i, o = shape
    g = gen(n * 11 + i)
    w = (torch.empty((o, i), device="cuda").uniform_(-1, 1, generator=g) * math.sqrt(6.0 / (i + o))).to(t)
    for k, (kind, pad, offset, skip) in enumerate([(R.NONE, 0, 0, False), (R.RELU, 0, 0, True), (R.GELU, 8, 0, False), (R.SILU, 5, 1, True)]):
        x, dy = rows(g, n, i, t, 1.0, pad, offset), rows(g, n, o, t, 0.1, pad, offset)
        zb = rows(g, n, i, t, 1.0, pad, offset) if kind != R.NONE else None
        sk = rows(g, n, i, t, 0.1, pad, offset) if skip else None
        base_w = torch.randn((o, i), device="cuda", generator=g) if k == 1 else None
        base_b = torch.randn(o, device="cuda", generator=g) if k == 1 else None
        dx, dw, db = ops.linear_backward(x, w, dy, below_activation=kind, below_preact=zb, skip=sk, mode=L.GRAD_ACCUMULATE if k == 1 else L.GRAD_OVERWRITE,
                                         wgrad=base_w.clone() if k == 1 else None, bgrad=base_b.clone() if k == 1 else None)
        wx, ww, wb, ex, ew, eb = R.linear_backward(x, w, dy, kind, zb, sk, t)
        if k == 1:
            ww, wb = ww + base_w.double(), wb + base_b.double()
            ew, eb = ew + 2.0 ** -23 * (ww.abs() + base_w.double().abs()), eb + 2.0 ** -23 * (wb.abs() + base_b.double().abs())
        R.within(f"dx {k}", dx, wx, ex)
        R.within(f"dw {k}", dw, ww, ew)
        R.within(f"db {k}", db, wb, eb)


@pytest.mark.parametrize("shape", [(1000, 37, 64), (700, 64, 37), (300, 61, 33), (5000, 13, 9), (40, 37, 29), (500, 1001, 333), (2000, 100, 201)],
                         ids=lambda s: "x".join(map(str, s)))
def test_rows_on_16_byte_boundaries_with_odd_widths(ops, shape):
    """Widths that fill no 16-byte unit in rows that start on 16-byte boundaries: what lies behind a row (NaN in the inputs, a marker
    around the outputs) is neither used nor written."""
    n, i, o = shape
    t = torch.float16
    g = gen(n + i)

    def padded(rows_, width, scale=1.0):
        full = torch.full((rows_, (width + 15) // 8 * 8), float("nan"), dtype=t, device="cuda")
        full[:, :width] = rows(g, rows_, width, t, scale)
        return full[:, :width]
    x, r, dy, zb = padded(n, i), padded(n, o), padded(n, o, 0.1), padded(n, i)
    w, b = rows(g, o, i, t, 0.3), rows(g, 1, o, t)[0]
    y, untouched = framed(n, o, t, (o + 15) // 8 * 8 - o)
    _, z = ops.linear_forward(x, w, b, r, R.GELU, want_preact=True, out=y)
    wy, wz, ey, ez = R.linear(x, w, b, r, R.GELU, t)
    R.within("y", y, wy, ey)
    R.within("z", z, wz, ez)
    assert untouched()
    dx, dw, db = ops.linear_backward(x, w, dy, below_activation=R.SILU, below_preact=zb)
    wx, ww, wb, ex, ew, eb = R.linear_backward(x, w, dy, R.SILU, zb, None, t)
    R.within("dx", dx, wx, ex)
    R.within("dw", dw, ww, ew)
    R.within("db", db, wb, eb)


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
def test_linear_backward_of_an_activated_layer(ops, t):
    """The layer's own activation: dz is rounded to the layer's type on the way, which the bound counts."""
    n, i, o = 150, 72, 40
    g = gen(5)
    x, w, dy = rows(g, n, i, t), rows(g, o, i, t, 0.2), rows(g, n, o, t, 0.1)
    for kind in (R.RELU, R.GELU, R.SILU):
        y, z = ops.linear_forward(x, w, activation=kind, want_preact=True)
        dx, dw, db = ops.linear_backward(x, w, dy, activation=kind, preact=z)
        dz = dy.double() * R.slope(kind, z.double())
        e = dy.double().abs() * (R.ACT_REL + 8 * R.ACT_ABS) + R.half_step(t, dz) * 1.01
        wx, ww, wb, ex, ew, eb = R.linear_backward(x, w, dz, R.NONE, None, None, t)
        R.within("dx", dx, wx, ex + 1.01 * (e @ w.double().abs()))
        R.within("dw", dw, ww, ew + e.T @ x.double().abs())
        R.within("db", db, wb, eb + e.sum(0))


@pytest.mark.parametrize("n", [1, 100, 5000, 40000])
def test_bias_gradient_alone_and_frozen_inputs(ops, n):
    """Each of the three gradients alone, and none: the same values as together."""
    from neus2_b200 import _lib as L
    g = gen(n)
    t = torch.bfloat16
    for i, o in ((16, 72), (520, 9), (40, 300)):
        x, w, dy = rows(g, n, i, t), rows(g, o, i, t, 0.2), rows(g, n, o, t, 0.1)
        dx, dw, db = ops.linear_backward(x, w, dy)
        assert torch.equal(ops.linear_backward(x, w, dy, mode=L.GRAD_IGNORE)[0], dx)
        only = ops.linear_backward(x, w, dy, want_din=False, want_bias=False)
        assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
        d, need = L.LinearDesc(n, i, o, L.BF16, 0), C.c_uint64(0)
        L.check(L.lib().neus2b_linear_backward_workspace(C.byref(d), 1, C.byref(need)))
        ws, out = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda"), torch.full((o,), 7.0, device="cuda")
        L.check(L.lib().neus2b_linear_backward(C.byref(d), None, 0, None, None, 0, dy.data_ptr(), o, 0, None, 0, None, 0, None, 0, None, out.data_ptr(),
                                               L.GRAD_ACCUMULATE, ws.data_ptr(), need.value, L.cur_stream()))
        want = dy.double().sum(0)
        R.within("db", out, want + 7.0, (n + 8) * 2.0 ** -23 * (dy.double().abs().sum(0) + 7.0))
        R.within("db", db, want, (n + 4) * 2.0 ** -23 * dy.double().abs().sum(0))


def test_linear_gradients_against_differences(ops):
    """The backward pass against central differences of the 64-bit forward pass, through activation, residual and bias."""
    t, n, i, o = torch.float16, 9, 24, 16
    g = gen(3)
    x, w, b = rows(g, n, i, t), rows(g, o, i, t, 0.3), rows(g, 1, o, t, 0.3)[0]
    dy = rows(g, n, o, t, 1.0)
    z = ops.linear_forward(x, w, b, want_preact=True)[1]
    dx, dw, db = ops.linear_backward(x, w, dy, activation=R.GELU, preact=z, skip=None)
    h = 1e-5

    def loss(xx, ww, bb):
        return float((R.act(R.GELU, xx @ ww.T + bb) * dy.double()).sum())
    args = [x.double(), w.double(), b.double()]
    for k, grad in enumerate((dx, dw, db)):
        flat = args[k].clone()
        for e in (0, 5, flat.numel() - 1):
            v = []
            for sgn in (1, -1):
                a = [q.clone() for q in args]
                a[k].view(-1)[e] += sgn * h
                v.append(loss(*a))
            want = (v[0] - v[1]) / (2 * h)
            # dz is rounded once (2^-11), z was (its slope moves by at most 2^-11 |z|), and sums of up to 24 terms of size < 4 follow
            assert abs(float(grad.reshape(-1)[e]) - want) <= 24 * 4 * 2 ** -10 + abs(want) * 2 ** -10, (k, e)


def test_linear_special_values(ops):
    """Infinities and NaN stay in their rows; a large negative argument of an activation gives 0, not NaN."""
    t = torch.bfloat16
    x = torch.zeros((70, 64), dtype=t, device="cuda")
    x[:, 0] = 1.0
    x[3, 5], x[4, 6], x[69, 1] = float("nan"), float("inf"), -3e38
    w = torch.ones((48, 64), dtype=t, device="cuda")
    for kind in (R.NONE, R.RELU, R.GELU, R.SILU):
        y = ops.linear_forward(x, w, activation=kind)
        assert bool(torch.isnan(y[3]).all())
        assert bool(torch.isinf(y[4]).all()) and bool((y[4] > 0).all())
        assert bool(torch.isfinite(y[[0, 1, 2, 5, 68, 69]]).all())
        if kind != R.NONE:
            assert bool((y[69] == 0).all()), kind
    z = torch.full((70, 64), -3e38, dtype=t, device="cuda")
    z[1] = 3e38
    dx, _, _ = ops.linear_backward(x[:, :64], w, torch.ones((70, 48), dtype=t, device="cuda"), below_activation=R.GELU, below_preact=z)
    assert bool((dx[0] == 0).all()) and bool((dx[1] == 48).all())


def test_linear_same_bits_and_in_place(ops):
    g = gen(8)
    t = torch.float16
    for n, i, o in ((5, 1000, 200), (4000, 256, 96)):
        x, w, r = rows(g, n, i, t), rows(g, o, i, t, 0.05), rows(g, n, o, t)
        dy = rows(g, n, o, t)
        a = ops.linear_forward(x, w, None, r, R.SILU)
        assert torch.equal(a, ops.linear_forward(x, w, None, r, R.SILU))
        y = r.clone()
        assert torch.equal(a, ops.linear_forward(x, w, None, y, R.SILU, out=y))
        p, q = ops.linear_backward(x, w, dy), ops.linear_backward(x, w, dy)
        assert all(torch.equal(u, v) for u, v in zip(p, q))


def test_empty_batches(ops):
    from neus2_b200 import _lib as L
    e = lambda *s: torch.empty(s, dtype=torch.float16, device="cuda")  # noqa: E731
    w = torch.ones((8, 16), dtype=torch.float16, device="cuda")
    assert ops.linear_forward(e(0, 16), w).shape == (0, 8)
    dx, dw, db = ops.linear_backward(e(0, 16), w, e(0, 8))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    keep = torch.full((8, 16), 3.0, device="cuda")
    assert bool((ops.linear_backward(e(0, 16), w, e(0, 8), wgrad=keep, mode=L.GRAD_ACCUMULATE)[1] == 3.0).all())
    gamma = torch.ones(16, dtype=torch.float16, device="cuda")
    assert ops.layer_norm_forward(e(0, 16), gamma).shape == (0, 16)
    s = torch.empty(0, device="cuda")
    dx, dg, db = ops.layer_norm_backward(e(0, 16), gamma, s, s, e(0, 16))
    assert dx.shape == (0, 16) and not dg.any() and not db.any()


# ------------------------------------------------------------------------------------------------ layer norm
NORM_SHAPES = [(1, 1), (3, 2), (5, 8), (2, 16), (100, 48), (1001, 64), (37, 129), (64, 255), (129, 256), (33, 1000), (300, 1024), (7, 1111), (50, 2048),
               (20, 4096), (9, 5001), (3, 8192), (4, 12288), (2, 16384), (2, 20001), (1, 70000), (4000, 72)]


@pytest.mark.parametrize("t", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", NORM_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm(ops, shape, t):
    """Forward and backward.  Bounds: a mean of W values in 32 bits loses at most W 2^-23 of the mean magnitude m; the centred
    values x - mean then W 2^-23 m, and the scale 1/std (W + 8) 2^-23 of itself and what the centring moved the variance by, at most
    2 W 2^-23 m |x - mean| / var in the mean, below 2 W 2^-23 m rstd.  Widths here are at most 70000 and their sums are
    taken in a few hundred partial sums, so that the effective number of steps is below 1024."""
    n, width = shape
    g = gen(width + n)
    steps = min(width, 1024) * 2.0 ** -23
    for k, (pad, offset, pt) in enumerate([(0, 0, t), (8, 0, torch.float32), (3, 1, t)]):
        x = rows(g, n, width, t, 1.5, pad, offset)
        gamma, beta = (1 + 0.2 * torch.randn(width, device="cuda", generator=g)).to(pt), (0.2 * torch.randn(width, device="cuda", generator=g)).to(pt)
        bb = beta if k != 2 else None
        y, untouched = framed(n, width, t, pad)
        _, mean, rstd = ops.layer_norm_forward(x, gamma, bb, want_stats=True, out=y)
        wy, wm, wr = R.layer_norm(x, gamma, bb, 1e-5)
        m = x.double().abs().mean(1)
        e_mean = steps * m + 1e-30
        e_rstd = wr * ((8 * 2.0 ** -23 + steps) + 2 * e_mean * wr)
        R.within(f"mean {k}", mean, wm, e_mean)
        R.within(f"rstd {k}", rstd, wr, e_rstd)
        xc = (x.double() - wm[:, None]).abs()
        e = gamma.double().abs() * (wr[:, None] * (e_mean[:, None] + 2.0 ** -22 * (xc + wm.abs()[:, None])) + xc * e_rstd[:, None]) + 2.0 ** -22 * wy.abs()
        e = e + 2.0 ** -23 * (0 if bb is None else bb.double().abs())
        R.within(f"y {k}", y, wy, e + R.half_step(t, wy.abs() + e))
        assert untouched(), k

        dy = rows(g, n, width, t, 0.1, pad, offset)
        skip = rows(g, n, width, t, 0.1, pad, offset) if k != 1 else None
        base = torch.randn(width, device="cuda", generator=g) if k == 1 else None
        from neus2_b200 import _lib as L
        dx, dg, db = ops.layer_norm_backward(x, gamma, mean, rstd, dy, skip=skip, dgamma=None if base is None else base.clone(),
                                             dbeta=None if base is None else base.clone(), mode=L.GRAD_OVERWRITE if base is None else L.GRAD_ACCUMULATE)
        wx, wg, wb = R.layer_norm_backward(x, gamma, mean, rstd, dy, skip)
        xh = (x.double() - mean.double()[:, None]).abs() * rstd.double()[:, None]
        # (x - mean) rstd in 32 bits: the difference is rounded once, the product once
        e_xh = 2.0 ** -22 * xh
        a = (dy.double() * gamma.double()).abs()
        s1, s2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
        e = rstd.double()[:, None] * (8 * 2.0 ** -23 * a + (steps + 8 * 2.0 ** -23) * (s1 + xh * s2) + e_xh * s2 + xh * (a * e_xh).mean(1, keepdim=True))
        e = e + 2.0 ** -22 * (wx.abs() + (0 if skip is None else skip.double().abs()))
        R.within(f"dx {k}", dx, wx, e + R.half_step(t, wx.abs() + e))
        col = (n + 8) * 2.0 ** -23
        eg, eb = (dy.double().abs() * (xh * col + e_xh)).sum(0) + 1e-30, col * dy.double().abs().sum(0) + 1e-30
        if base is not None:
            wg, wb = wg + base.double(), wb + base.double()
            eg, eb = eg + 2.0 ** -22 * (wg.abs() + base.double().abs()), eb + 2.0 ** -22 * (wb.abs() + base.double().abs())
        R.within(f"dgamma {k}", dg, wg, eg)
        R.within(f"dbeta {k}", db, wb, eb)


@pytest.mark.parametrize("shape", [(1, 100), (9, 1024), (32, 1111), (32, 4096), (33, 1111), (200, 64)], ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_backward_parts(ops, shape):
    """Parameter gradients without dL/dx, dL/dx without them, one of the two alone: the bits of the whole call."""
    from neus2_b200 import _lib as L
    n, width = shape
    t = torch.bfloat16
    g = gen(width)
    x, dy = rows(g, n, width, t), rows(g, n, width, t)
    gamma = torch.randn(width, device="cuda", generator=g)
    _, mean, rstd = ops.layer_norm_forward(x, gamma, want_stats=True)
    dx, dg, db = ops.layer_norm_backward(x, gamma, mean, rstd, dy)
    none, dg1, db1 = ops.layer_norm_backward(x, gamma, mean, rstd, dy, want_din=False)
    assert none is None and torch.equal(dg, dg1) and torch.equal(db, db1)
    dx2, none, _ = ops.layer_norm_backward(x, gamma, mean, rstd, dy, mode=L.GRAD_IGNORE)
    assert none is None and torch.equal(dx, dx2)
    lib, d, need = L.lib(), L.LayerNormDesc(n, width, 2, 0, 1e-5), C.c_uint64(0)
    L.check(lib.neus2b_layer_norm_backward_workspace(C.byref(d), C.byref(need)))
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    for which in (0, 1):
        out = torch.full((width + 2,), 7.0, device="cuda")
        at = out[1:].data_ptr()
        L.check(lib.neus2b_layer_norm_backward(C.byref(d), x.data_ptr(), width, gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), width, None, 0,
                                               None, 0, None if which else at, at if which else None, L.GRAD_OVERWRITE, ws.data_ptr(), need.value,
                                               torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out[1:-1], db if which else dg) and float(out[0]) == float(out[-1]) == 7.0


@pytest.mark.parametrize("shape", [(9, 1024), (33, 1111), (300, 4096), (4000, 64), (5, 20001)], ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_backward_in_place(ops, shape):
    """dL/dx in the place of dL/dy, or of the skip connection's gradient."""
    from neus2_b200 import _lib as L
    n, width = shape
    g = gen(width + 1)
    x, dy, skip = rows(g, n, width, torch.float16), rows(g, n, width, torch.float16), rows(g, n, width, torch.float16)
    gamma = torch.randn(width, device="cuda", generator=g)
    _, mean, rstd = ops.layer_norm_forward(x, gamma, want_stats=True)
    want = ops.layer_norm_backward(x, gamma, mean, rstd, dy, skip=skip)
    lib, d, need = L.lib(), L.LayerNormDesc(n, width, 1, 0, 1e-5), C.c_uint64(0)
    L.check(lib.neus2b_layer_norm_backward_workspace(C.byref(d), C.byref(need)))
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    for k in (0, 1):
        y, s = dy.clone(), skip.clone()
        dg, db = torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
        out = s if k else y
        L.check(lib.neus2b_layer_norm_backward(C.byref(d), x.data_ptr(), width, gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), y.data_ptr(), width,
                                               s.data_ptr(), width, out.data_ptr(), width, dg.data_ptr(), db.data_ptr(), L.GRAD_OVERWRITE, ws.data_ptr(),
                                               need.value, torch.cuda.current_stream().cuda_stream))
        assert all(torch.equal(u, v) for u, v in zip((out, dg, db), want)), k


@pytest.mark.parametrize("shape", [(20, 300, 100), (1000, 64, 64), (1000, 512, 256), (500, 333, 77), (300, 2056, 120), (5000, 1024, 1024)],
                         ids=lambda s: "x".join(map(str, s)))
def test_linear_backward_in_place(ops, shape):
    """dL/dx in the place of the skip connection's gradient."""
    from neus2_b200 import _lib as L
    n, i, o = shape
    g = gen(i + o)
    t = torch.bfloat16
    x, dy, zb, skip, w = rows(g, n, i, t), rows(g, n, o, t, 0.1), rows(g, n, i, t), rows(g, n, i, t, 0.1), rows(g, o, i, t, 0.1)
    want = ops.linear_backward(x, w, dy, below_activation=R.GELU, below_preact=zb, skip=skip)
    lib, d, need = L.lib(), L.LinearDesc(n, i, o, 2, 0), C.c_uint64(0)
    L.check(lib.neus2b_linear_backward_workspace(C.byref(d), 1, C.byref(need)))
    ws = torch.empty(need.value + 16, dtype=torch.uint8, device="cuda")
    out, dw, db = skip.clone(), torch.empty((o, i), device="cuda"), torch.empty(o, device="cuda")
    L.check(lib.neus2b_linear_backward(C.byref(d), x.data_ptr(), i, w.data_ptr(), None, 0, dy.data_ptr(), o, L.ACT_GELU, zb.data_ptr(), i, out.data_ptr(), i,
                                       out.data_ptr(), i, dw.data_ptr(), db.data_ptr(), L.GRAD_OVERWRITE, ws.data_ptr(), need.value,
                                       torch.cuda.current_stream().cuda_stream))
    assert all(torch.equal(u, v) for u, v in zip((out, dw, db), want))


def test_layer_norm_rows_far_from_zero_and_constant(ops):
    """A mean a thousand times the spread costs no accuracy beyond the inputs' own; constant rows give beta."""
    g = gen(4)
    x = 1000.0 + torch.randn((40, 600), device="cuda", generator=g)
    gamma, beta = torch.ones(600, device="cuda"), torch.full((600,), 0.25, device="cuda")
    y = ops.layer_norm_forward(x, gamma, beta)
    want, _, _ = R.layer_norm(x, gamma, beta, 1e-5)
    # the mean is off by at most 600 * 2^-24 * 1000 = 0.036 in the worst order; pairwise partial sums of 4 to 32 terms keep it below
    # 40 * 2^-24 * 1000 = 0.0024, which moves the centred values by as much and the variance by its square
    R.within("y", y, want, torch.full_like(want, 0.0026))
    for t in (torch.float32, torch.float16):
        c = torch.full((5, 200), 3.0, dtype=t, device="cuda")
        assert bool((ops.layer_norm_forward(c, gamma[:200].to(t), beta[:200].to(t)) == 0.25).all())


def test_layer_norm_in_place_same_bits_and_special_values(ops):
    g = gen(6)
    for width in (64, 1111, 4096):
        x = rows(g, 50, width, torch.bfloat16)
        x[7, 3] = float("nan")
        x[8, 1] = float("inf")
        gamma = rows(g, 1, width, torch.bfloat16)[0]
        y, mean, rstd = ops.layer_norm_forward(x, gamma, want_stats=True)
        assert bool(torch.isnan(y[[7, 8]]).all()) and bool(torch.isfinite(y[:7]).all()) and bool(torch.isfinite(y[9:]).all())
        z = x.clone()
        ops.layer_norm_forward(z, gamma, out=z)
        assert torch.equal(z[:7], y[:7]) and torch.equal(z[9:], y[9:])
        dy = rows(g, 50, width, torch.bfloat16)
        p, q = (ops.layer_norm_backward(x, gamma, mean, rstd, dy) for _ in range(2))
        assert torch.equal(p[0][:7], q[0][:7]) and torch.equal(p[2], q[2])


# ------------------------------------------------------------------------------------------------ clipping
def clip_reference(grads, max_norm, scale=1.0, skip=False):
    total = 0.0
    for g in grads:
        v = g.double().flatten()
        if skip:
            v = v[torch.isfinite(v)]
        total += float((v * v).sum())
    norm = abs(scale) * math.sqrt(total)
    return norm, max_norm / norm if norm > max_norm and math.isfinite(norm) else 1.0


@pytest.mark.parametrize("sizes", [[1], [5, 0, 3], [8192, 8193, 16384], [4, 12288, 1000003], [100 + 37 * i for i in range(700)]], ids=lambda s: f"{len(s)}_tensors_of_{s[-1]}")
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16", "mixed"])
def test_clip(ops, sizes, kind):
    if len(sizes) > 10 and kind != "mixed":
        sizes = sizes[:40]
    g = gen(len(sizes))
    types = {"f32": [torch.float32], "f16": [torch.float16], "bf16": [torch.bfloat16], "mixed": [torch.float32, torch.float16, torch.bfloat16]}[kind]
    for offset in (0, 1):
        base = [torch.randn(s + offset + 3, device="cuda", generator=g).mul(10.0 ** -(i % 4)).to(types[i % len(types)]) for i, s in enumerate(sizes)]
        grads = [b[offset:offset + s] for b, s in zip(base, sizes)]
        norm = clip_reference(grads, 1.0)[0]
        for max_norm in (0.37 * norm, 2 * norm):
            want_norm, c = clip_reference(grads, max_norm)
            outs = [torch.full((s + 5,), 55.0, dtype=b.dtype, device="cuda") for b, s in zip(base, sizes)]
            got = ops.GradientSet(grads, out=[o[2:2 + s] for o, s in zip(outs, sizes)]).clip(max_norm)
            # the sum is in 64 bits: norm and factor are rounded once, the product once more in 32 bits, and the result to its type
            assert abs(float(got[0]) - want_norm) <= 2.0 ** -23 * want_norm
            assert abs(float(got[1]) - c) <= 2.0 ** -22 * c
            for gr, o, s in zip(grads, outs, sizes):
                want = gr.double() * c
                R.within("clipped", o[2:2 + s], want, 2.0 ** -21 * want.abs() + R.half_step(gr.dtype, want * (1 + 1e-6)))
                assert bool((o[:2] == 55).all()) and bool((o[2 + s:] == 55).all())
            copies = [b.clone() for b in base]
            ops.GradientSet([b[offset:offset + s] for b, s in zip(copies, sizes)]).clip(max_norm)
            for b, old, o, s in zip(copies, base, outs, sizes):
                assert torch.equal(b[offset:offset + s], o[2:2 + s])
                assert torch.equal(b[:offset], old[:offset]) and torch.equal(b[offset + s:], old[offset + s:])


def test_clip_extreme_and_nonfinite(ops):
    big = torch.full((3000,), 3e38, device="cuda")
    assert float(ops.GradientSet([big[:1]]).norm()[0]) == pytest.approx(3e38, rel=1e-6)
    tiny = torch.full((10000,), 1e-30, dtype=torch.bfloat16, device="cuda")
    assert float(ops.GradientSet([tiny]).norm()[0]) == pytest.approx(1e-28, rel=0.01)
    r = ops.GradientSet([big, tiny], out=[torch.empty_like(big), torch.empty_like(tiny)]).clip(1.0)
    assert math.isinf(float(r[0])) and float(r[1]) == pytest.approx(1 / (3e38 * math.sqrt(3000)), rel=1e-3, abs=2e-45)
    for bad in (float("nan"), float("inf"), -float("inf")):
        g = [torch.ones(500, device="cuda"), torch.ones(300, dtype=torch.float16, device="cuda")]
        g[1][299] = bad
        g[0][0] = bad
        count = torch.zeros(1, dtype=torch.int32, device="cuda")
        s = ops.GradientSet(g)
        r = s.clip(1.0, nonfinite=count)
        assert not math.isfinite(float(r[0])) and float(r[1]) == 1.0 and int(count) == 2 and bool((g[0][1:] == 1).all())
        r = s.clip(1.0, skip_nonfinite=True, nonfinite=count)
        assert float(r[0]) == pytest.approx(math.sqrt(798.0), rel=1e-6) and int(count) == 4
        assert float(g[0][1]) == pytest.approx(1 / math.sqrt(798.0), rel=1e-6) and not math.isfinite(float(g[0][0]))
    z = torch.zeros(10, device="cuda")
    assert ops.GradientSet([z]).clip(1.0).tolist() == [0.0, 1.0]
    v = torch.full((4,), 3.0, device="cuda")
    assert ops.GradientSet([v]).norm(max_norm=1.5, scale=-0.5).tolist() == [3.0, 0.5]


def test_tensors_of_another_device_are_refused(ops, monkeypatch):
    from neus2_b200 import _lib as L
    x = torch.ones((8, 16), dtype=torch.float16, device="cuda")
    w, s, g = torch.ones((16, 16), dtype=torch.float16, device="cuda"), torch.ones(8, device="cuda"), torch.ones(16, device="cuda")
    gset = ops.GradientSet([g])
    monkeypatch.setattr(ops, "_current_device", lambda: x.get_device() + 1)
    for call in (lambda: ops.linear_forward(x, w), lambda: ops.linear_backward(x, w, x), lambda: ops.layer_norm_forward(x, g),
                 lambda: ops.layer_norm_backward(x, g, s, s, x), lambda: ops.GradientSet([g]), lambda: gset.clip(1.0)):
        with pytest.raises(L.Neus2bError, match="current device"):
            call()


FIRST_CALLS_IN_A_CAPTURE = """
import sys
sys.path.insert(0, {root!r})
import torch
from neus2_b200 import ops
t = torch.float16
x, w, wide, gamma = (torch.ones(s, dtype=t, device="cuda") for s in ((300, 64), (64, 64), (320, 64), (64,)))
few, odd = torch.ones((3, 64), dtype=t, device="cuda"), torch.ones((300, 63), dtype=t, device="cuda")
wodd, grad = torch.ones((40, 63), dtype=t, device="cuda"), torch.ones(1000, device="cuda")
gset = ops.GradientSet([grad])
torch.cuda.synchronize()
g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(g, stream=s):
    y = ops.linear_forward(x, w, activation=2)
    out = [y, ops.linear_forward(x, wide), ops.linear_forward(few, w), ops.linear_forward(odd, wodd), *ops.linear_backward(x, w, y), *ops.linear_backward(few, w, few)]
    h, mean, rstd = ops.layer_norm_forward(x, gamma, want_stats=True)
    out += [h, *ops.layer_norm_backward(x, gamma, mean, rstd, y), gset.clip(1.0)]
g.replay()
torch.cuda.synchronize()
assert float(y[0, 0]) == 64 and float(out[1][299, 319]) == 64 and float(out[2][2, 0]) == 64 and float(out[3][299, 39]) == 63
assert float(grad[0]) < 0.04 and all(bool(torch.isfinite(o.float()).all()) for o in out)
print("captured")
"""


def test_first_calls_of_a_process_inside_a_capture():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS_IN_A_CAPTURE.format(root=root)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_streams_and_graph(ops):
    """A call on another stream, and a captured block of all three operators replayed on new inputs."""
    g = gen(21)
    t = torch.float16
    n, width = 96, 64
    x, dy = rows(g, n, width, t), rows(g, n, width, t, 0.1)
    w, b, gamma = rows(g, width, width, t, 0.1), rows(g, 1, width, t, 0.1)[0], torch.ones(width, device="cuda")
    wg, bg = torch.empty((width, width), device="cuda"), torch.empty(width, device="cuda")
    gset = ops.GradientSet([wg, bg])

    def block():
        h, mean, rstd = ops.layer_norm_forward(x, gamma, want_stats=True)
        y, z = ops.linear_forward(h, w, b, x, R.GELU, want_preact=True)
        dh, _, _ = ops.linear_backward(h, w, dy, activation=R.GELU, preact=z, wgrad=wg, bgrad=bg)
        dx, dg, db = ops.layer_norm_backward(x, gamma, mean, rstd, dh, skip=dy)
        return [y, dx, dg, db, gset.clip(0.01), wg, bg]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [v.clone() for v in block()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = block()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(held, first))
        x.copy_(rows(g, n, width, t))
        dy.copy_(rows(g, n, width, t, 0.1))
        first = [v.clone() for v in block()]


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
def test_residual_block_and_clipping(ops, t):
    """h + W2 gelu(W1 LN(h) + b1) + b2 forward and backward as a user chains the calls, then clipping, against autograd in 64 bits.  Norms of
    differences: a result is behind at most six roundings to the type (u, z, a, dz, du, dh), each at most eps / 2 of its value; the factors
    between them (slopes, projections of the norm) do not enlarge a norm, the slopes of a rounded z add one more."""
    from neus2_b200 import _lib as L
    g = gen(5)
    n, width, hidden = 300, 256, 520
    h, dh1 = rows(g, n, width, t), rows(g, n, width, t)
    gamma, beta = 1 + 0.1 * torch.randn(width, device="cuda", generator=g), 0.1 * torch.randn(width, device="cuda", generator=g)
    w1, w2 = rows(g, hidden, width, t, 0.06), rows(g, width, hidden, t, 0.04)
    b1, b2 = rows(g, 1, hidden, t, 0.3)[0], rows(g, 1, width, t, 0.3)[0]
    u, mean, rstd = ops.layer_norm_forward(h, gamma, beta, want_stats=True)
    a, z = ops.linear_forward(u, w1, b1, activation=L.ACT_GELU, want_preact=True)
    h1 = ops.linear_forward(a, w2, b2, residual=h)
    dz, gw2, gb2 = ops.linear_backward(a, w2, dh1, below_activation=L.ACT_GELU, below_preact=z)
    du, gw1, gb1 = ops.linear_backward(u, w1, dz)
    dh, ggamma, gbeta = ops.layer_norm_backward(h, gamma, mean, rstd, du, skip=dh1)
    leaves = [v.double().requires_grad_() for v in (h, gamma, beta, w1, b1, w2, b2)]
    H, G, B, W1, B1, W2, B2 = leaves
    centred = H - H.mean(1, keepdim=True)
    U = centred / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5) * G + B
    Z = U @ W1.T + B1
    Y = 0.5 * Z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (Z + 0.044715 * Z ** 3))) @ W2.T + B2 + H
    Y.backward(dh1.double())
    bound = 7 * torch.finfo(t).eps / 2
    for name, got, want in [("h1", h1, Y.detach()), ("dh", dh, H.grad), ("ggamma", ggamma, G.grad), ("gbeta", gbeta, B.grad), ("gw1", gw1, W1.grad),
                            ("gb1", gb1, B1.grad), ("gw2", gw2, W2.grad), ("gb2", gb2, B2.grad)]:
        assert float((got.double() - want).norm() / want.norm()) <= bound, name
    grads = [gw2, gb2, gw1, gb1, ggamma, gbeta]
    before = [v.clone() for v in grads]
    norm = math.sqrt(sum(float((v.double() ** 2).sum()) for v in before))
    got_norm, factor = ops.GradientSet(grads).clip(max_norm=norm / 3).tolist()
    assert abs(got_norm / norm - 1) <= 2.0 ** -22 and abs(factor * 3 - 1) <= 2.0 ** -21
    assert all(torch.equal(v, u * factor) for v, u in zip(grads, before))


def test_two_streams_at_once(ops):
    """Calls of every kind issued to two streams in turn, without waiting in between, give the bits that they give one after another."""
    g = gen(77)
    t = torch.bfloat16
    jobs = []
    for n, i, o in [(5, 512, 300), (64, 1000, 1000), (300, 2056, 120), (2000, 131, 257), (5000, 64, 64), (1500, 512, 512), (3000, 1024, 2048)]:
        x, dy, zb = rows(g, n, i, t), rows(g, n, o, t, 0.1), rows(g, n, i, t)
        w, b = rows(g, o, i, t, 0.05), rows(g, 1, o, t)[0]
        gamma = torch.ones(i, device="cuda")

        def job(x=x, dy=dy, zb=zb, w=w, b=b, gamma=gamma):
            y, z = ops.linear_forward(x, w, b, None, R.GELU, want_preact=True)
            dx, dw, db = ops.linear_backward(x, w, dy, activation=R.GELU, preact=z, below_activation=R.SILU, below_preact=zb)
            h, mean, rstd = ops.layer_norm_forward(x, gamma, want_stats=True)
            dh, dg, dbeta = ops.layer_norm_backward(x, gamma, mean, rstd, dx, skip=h)
            return [y, z, dx, dw, db, h, dh, dg, dbeta]
        jobs.append(job)
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for turn in range(4):
        for k, job in enumerate(jobs):
            with torch.cuda.stream(streams[(k + turn) % 2]):
                got.append((k, job()))
    torch.cuda.synchronize()
    for k, out in got:
        assert all(torch.equal(u, v) for u, v in zip(out, want[k])), k


def test_no_wait_ran_out(ops):
    from neus2_b200 import _lib as L
    torch.cuda.synchronize()
    assert L.device_error_flags() == 0
