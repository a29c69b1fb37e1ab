"""Linear layers at sizes where a block takes many tiles and rounds: exact comparisons on whole numbers, and bounds of the parameter gradients
that follow how their sums are taken (dense_sums.py) on random ones."""
import pytest
import torch

import dense_reference as R
from dense_sums import sum_bound, whole

pytestmark = pytest.mark.gpu
HALF = [torch.float16, torch.bfloat16]
RELU = 1


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


#         n, in, out.  Narrow: a second tile, a second round of four tiles, a third, all of them ragged; both widths of dz
SHAPES = [(100000, 64, 64), (150001, 64, 128), (75777, 56, 40), (262144, 48, 64), (90000, 16, 72), (80000, 64, 61), (120000, 8, 128),
          # general: samples split over all SMs, over a cluster, not at all; pairs; a matrix of tiles wider than the grid
          (20000, 130, 100), (50001, 200, 136), (1328, 160, 192), (33333, 129, 65), (70000, 72, 136), (8192, 2048, 1024), (30001, 512, 768), (5000, 1024, 1025),
          (2049, 4096, 2056), (600, 3000, 2500), (130, 5000, 40), (64, 1000, 3000), (31, 700, 520)]


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear_exact(ops, shape, t):
    """Whole numbers of up to 2: every sum is exact (the largest, 4 n, is below 2^24), every result is one rounding of it."""
    from neus2_b200 import _lib as L
    n, i, o = shape
    assert 4 * max(shape) + 8 < 1 << 24
    g = gen(n + 3 * i)
    w, b = whole(g, o, i, t), whole(g, 1, o, t)[0]
    for pad, offset in ((0, 0), (3, 1)):
        x, dy, r = whole(g, n, i, t, pad=pad, offset=offset), whole(g, n, o, t, pad=pad, offset=offset), whole(g, n, o, t, pad=pad, offset=offset)
        zb, skip = whole(g, n, i, t, pad=pad, offset=offset), whole(g, n, i, t, pad=pad, offset=offset)
        z = x.double() @ w.double().T + b.double()
        y, kept = ops.linear_forward(x, w, b, r, RELU, want_preact=True)
        assert torch.equal(kept, z.to(t)) and torch.equal(y, (z.clamp(min=0) + r.double()).to(t))
        wx = dy.double() @ w.double()
        ww, wb = dy.double().T @ x.double(), dy.double().sum(0)
        dx, dw, db = ops.linear_backward(x, w, dy, below_activation=RELU, below_preact=zb, skip=skip)
        assert torch.equal(dx, (wx * (zb > 0) + skip.double()).to(t))
        assert torch.equal(dw.double(), ww) and torch.equal(db.double(), wb)
        base_w, base_b = whole(g, o, i, torch.float32, 100), whole(g, 1, o, torch.float32, 100)[0]
        dx, dw, db = ops.linear_backward(x, w, dy, wgrad=base_w.clone(), bgrad=base_b.clone(), mode=L.GRAD_ACCUMULATE)
        assert torch.equal(dx, wx.to(t))
        assert torch.equal(dw.double(), ww + base_w.double()) and torch.equal(db.double(), wb + base_b.double())
        none, dw, db = ops.linear_backward(x, w, dy, want_din=False)
        assert none is None and torch.equal(dw.double(), ww) and torch.equal(db.double(), wb)
        dw = ops.linear_backward(x, w, dy, want_din=False, want_bias=False)[1]
        assert torch.equal(dw.double(), ww)


@pytest.mark.parametrize("t", HALF, ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", [(100000, 64, 64), (150001, 64, 128), (262144, 48, 64), (50001, 200, 136), (33333, 129, 65), (8192, 2048, 1024), (30001, 512, 768)],
                         ids=lambda s: "x".join(map(str, s)))
def test_linear_parameter_gradients(ops, shape, t):
    n, i, o = shape
    g = gen(n)
    x, dy, w = rows(g, n, i, t), rows(g, n, o, t, 0.1), rows(g, o, i, t, 0.1)
    _, dw, db = ops.linear_backward(x, w, dy)
    R.within("dw", dw, dy.double().T @ x.double(), sum_bound(n, dy.double().abs().T @ x.double().abs()))
    R.within("db", db, dy.double().sum(0), sum_bound(n, dy.double().abs().sum(0)))
