"""Backward passes through activations of infinite preactivations: fp16 holds a preactivation beyond its range as infinity, and the forward
pass, which evaluates the activation ahead of that rounding, gives 0 or z there.  The slopes are the limits, 0 and 1."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")
RELU, GELU, SILU = 1, 2, 3

#         n, in, out, pad: few samples, few unaligned, narrow, general, general unaligned, even widths, pairs
SHAPES = [(1, 64, 64, 0), (20, 300, 100, 0), (20, 301, 77, 3), (1000, 64, 64, 0), (300, 256, 264, 0), (500, 333, 77, 1), (700, 130, 66, 0),
          (8192, 2048, 1024, 0)]


@pytest.fixture(scope="module")
def ops():
    from neus2_b200 import ops as o
    return o


def rows(g, n, width, t, scale=1.0, pad=0):
    return torch.empty((n, width + pad), device="cuda").normal_(0.0, scale, generator=g).to(t)[:, :width]


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_slopes_of_the_layer_below(ops, shape, t):
    """A slope of 1 changes no bit of dL/dx and a slope of 0 leaves 0, whatever the neighbours; NaN stays NaN."""
    n, i, o, pad = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(n + i)
    x, dy, w = rows(g, n, i, t, 1.0, pad), rows(g, n, o, t, 0.1, pad), rows(g, o, i, t, 0.1)
    plain, pw, pb = ops.linear_backward(x, w, dy)
    for kind in (RELU, GELU, SILU):
        z = rows(g, n, i, t, 1.0, pad)
        z[:, 0], z[:, 1], z[:, -1], z[n // 2] = INF, -INF, -INF, INF
        z[0, 3] = NAN
        dx, dw, db = ops.linear_backward(x, w, dy, below_activation=kind, below_preact=z)
        assert torch.equal(dx[:, 0], plain[:, 0]), kind
        assert torch.equal(dx[n // 2, 4:], plain[n // 2, 4:]), kind
        away = torch.arange(n, device="cuda") != n // 2
        assert bool((dx[away][:, [1, -1]] == 0).all()), kind
        finite = torch.isfinite(dx)
        finite[0, 3] = True
        assert bool(finite.all()), kind
        if kind != RELU and n > 1:  # (of the single row all z are +infinity, but for the NaN)
            assert bool(torch.isnan(dx[0, 3])), kind
        assert torch.equal(dw, pw) and torch.equal(db, pb), kind


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_slopes_of_the_layer_itself(ops, shape, t):
    """With every preactivation infinite dz is dL/dy or 0, exactly: the gradients are those of that dz, bit by bit."""
    n, i, o, pad = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(n + o)
    x, dy, w = rows(g, n, i, t, 1.0, pad), rows(g, n, o, t, 0.1, pad), rows(g, o, i, t, 0.1)
    up = torch.rand((n, o), device="cuda", generator=g) < 0.5
    z = torch.where(up, INF, -INF).to(t)
    z = torch.cat([z, rows(g, n, max(pad, 1), t)], 1)[:, :o]
    dz = torch.where(up, dy, torch.zeros_like(dy))
    want = ops.linear_backward(x, w, dz)
    for kind in (RELU, GELU, SILU):
        got = ops.linear_backward(x, w, dy, activation=kind, preact=z)
        assert all(torch.equal(u, v) for u, v in zip(got, want)), kind


def test_forward_and_backward_beyond_the_range_of_fp16(ops):
    """z = +-70000: y is 0 or beyond the range, the stored z infinite, and the gradient that of the slopes 0 and 1."""
    t = torch.float16
    for n, i, o in ((2, 64, 64), (400, 64, 64), (400, 256, 128)):
        x = torch.full((n, i), 1.0, dtype=t, device="cuda")
        w = torch.full((o, i), -70000.0 / i, dtype=t, device="cuda")
        w[1::2] *= -1
        dy = torch.full((n, o), 0.5, dtype=t, device="cuda")
        for kind in (RELU, GELU, SILU):
            y, z = ops.linear_forward(x, w, activation=kind, want_preact=True)
            assert bool((y[:, 0::2] == 0).all()) and bool((z[:, 0::2] == -INF).all()) and bool((z[:, 1::2] == INF).all())
            _, dw, db = ops.linear_backward(x, w, dy, activation=kind, preact=z)
            assert bool((dw[0::2] == 0).all()) and bool((db[0::2] == 0).all())
            assert bool((dw[1::2] == 0.5 * n).all()) and bool((db[1::2] == 0.5 * n).all())
