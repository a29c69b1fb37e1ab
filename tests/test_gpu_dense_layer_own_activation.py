"""Backward passes through a layer's own activation: odd widths, strided rows, and more of them than the grid takes in one step."""
import pytest
import torch

import dense_reference as R
from dense_sums import whole

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]
RELU, GELU, SILU = 1, 2, 3


@pytest.fixture(scope="module")
def ops():
    from neus2_b200 import ops as o
    return o


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def rows(g, n, width, t, scale=1.0, pad=0, offset=0):
    full = torch.empty(offset + n * (width + pad), device="cuda").normal_(0.0, scale, generator=g).to(t)
    return full[offset:].view(n, width + pad)[:, :width]


#          n, out, pad, offset: whole units and not, strides, many rows
OWN = [(1, 1, 0, 0), (3, 7, 0, 0), (2, 8, 5, 0), (150, 40, 0, 0), (150, 40, 8, 8), (777, 77, 0, 0), (777, 77, 3, 1), (500, 300, 0, 0), (500, 301, 11, 0),
       (200000, 24, 0, 0), (200000, 24, 5, 1), (150001, 17, 0, 0), (3000, 1001, 0, 0), (3000, 1001, 7, 3), (9000, 520, 8, 0)]


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", OWN, ids=lambda s: "x".join(map(str, s)))
def test_slopes_of_the_layer_itself(ops, shape, t):
    """The weights are the unit matrix, so that dL/dx is dz, entry by entry: dL/dy times the slope, rounded once."""
    n, o, pad, offset = shape
    g = gen(n + o)
    w = torch.eye(o, device="cuda").to(t)
    x = rows(g, n, o, t)
    for kind in (RELU, GELU, SILU):
        for z_pad, z_offset in ((pad, offset), (0, 0)):
            z, dy = rows(g, n, o, t, 2.0, z_pad, z_offset), rows(g, n, o, t, 1.0, pad, offset)
            dx, _, _ = ops.linear_backward(x, w, dy, activation=kind, preact=z)
            want = dy.double() * R.slope(kind, z.double())
            e = dy.double().abs() * (R.ACT_REL + 8 * R.ACT_ABS if kind != RELU else 0.0)
            R.within("dz", dx, want, e + R.half_step(t, want.abs() + e))


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", OWN, ids=lambda s: "x".join(map(str, s)))
def test_slopes_of_the_layer_itself_exact(ops, shape, t):
    """Preactivations of 0 and of +-1000, where the slopes are exactly 1/2 (of GELU and SiLU; 0 of ReLU), 0 and 1, and even whole numbers as
    dL/dy: all three gradients, bit by bit, beside a layer below with its own activation and a skip connection."""
    n, o, pad, offset = shape
    i = 40 if o % 2 == 0 else 37
    g = gen(n + o + 1)
    x, w = whole(g, n, i, t, pad=pad, offset=offset), whole(g, o, i, t)
    skip, zb = whole(g, n, i, t), whole(g, n, i, t)
    for kind in (RELU, GELU, SILU):
        z, dy = whole(g, n, o, t, 1, 1000, pad, offset), whole(g, n, o, t, 2, 2, pad, offset)
        half = 0.0 if kind == RELU else 0.5
        dz = dy.double() * torch.where(z > 0, 1.0, torch.where(z < 0, 0.0, half))
        dx, dw, db = ops.linear_backward(x, w, dy, activation=kind, preact=z, below_activation=RELU, below_preact=zb, skip=skip)
        assert torch.equal(dx, (dz @ w.double() * (zb > 0) + skip.double()).to(t))
        assert torch.equal(dw.double(), dz.T @ x.double()) and torch.equal(db.double(), dz.sum(0))
