"""Layer norm of so many rows that every group takes several: forward row by row, backward exactly on whole numbers."""
import pytest
import torch

import dense_reference as R
from dense_sums import whole

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
    full = torch.empty(offset + n * (width + pad), device="cuda").normal_(0.0, scale, generator=g).to(t)
    return full[offset:].view(n, width + pad)[:, :width]


#        rows: rings (of depth 4, 2 and 1), rows fetched ahead, rows read plainly, rows of the wide kernels; several for every group and
#        the last of them ragged
NORMS = [(24001, 1024), (40003, 256), (6001, 4096), (3001, 8192), (1501, 16384), (150001, 64), (70001, 120), (40001, 129), (9001, 1000), (6003, 2049), (1301, 9837),
         (2001, 5003), (4001, 12288), (1501, 3001)]


@pytest.mark.parametrize("t", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", NORMS, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_forward_of_many_rows(ops, shape, t):
    """Row by row.  With m the mean magnitude of a row and partial sums of at most `steps` values: the mean is off by steps 2^-23 m, the
    centred values by as much, 1 / std by (8 + steps) 2^-23 of itself and by what the centring moved the variance."""
    n, width = shape
    g = gen(width + n)
    steps = min(width, 1024) * 2.0 ** -23
    for pad, offset, pt, in_place in ((0, 0, t, False), (8, 0, torch.float32, True), (3, 1, t, False)):
        x = rows(g, n, width, t, 1.5, pad, offset)
        x += 0.5
        gamma, beta = (1 + 0.2 * torch.randn(width, device="cuda", generator=g)).to(pt), (0.2 * torch.randn(width, device="cuda", generator=g)).to(pt)
        wy, wm, wr = R.layer_norm(x, gamma, beta, 1e-5)
        m = x.double().abs().mean(1)
        e_mean = steps * m + 1e-30
        e_rstd = wr * ((8 * 2.0 ** -23 + steps) + 2 * e_mean * wr)
        xc = (x.double() - wm[:, None]).abs()
        e = gamma.double().abs() * (wr[:, None] * (e_mean[:, None] + 2.0 ** -22 * (xc + wm.abs()[:, None])) + xc * e_rstd[:, None]) + 2.0 ** -22 * (wy.abs() + beta.double().abs())
        y, mean, rstd = ops.layer_norm_forward(x, gamma, beta, want_stats=True, out=x if in_place else None)
        R.within("mean", mean, wm, e_mean)
        R.within("rstd", rstd, wr, e_rstd)
        R.within("y", y, wy, e + R.half_step(t, wy.abs() + e))


@pytest.mark.parametrize("t", [torch.float32] + HALF, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", NORMS + [(32, 1111), (31, 8192), (17, 64), (33, 16384)], ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_backward_of_many_rows_exact(ops, shape, t):
    """The statistics are inputs of the backward pass.  Whole numbers in x and the means, scales of 1 and 2, whole numbers in gamma and dL/dy:
    the parameter gradients are whole numbers below 2^24 and compared bit by bit.  dL/dx has to be the exact value within the
    roundings of its two means (quotients by the width) and of the three operations behind them, and its own."""
    from neus2_b200 import _lib as L
    n, width = shape
    g = gen(width + 2 * n)
    assert n * 2 * 3 * 2 < 1 << 24
    for pad, offset, pt, with_skip, accumulate in ((0, 0, t, True, False), (8, 0, torch.float32, False, True), (3, 1, t, True, False)):
        x, dy = whole(g, n, width, t, 2, 1, pad, offset), whole(g, n, width, t, 2, 1, pad, offset)
        skip = whole(g, n, width, t, 2, 1, pad, offset) if with_skip else None
        gamma = whole(g, 1, width, pt)[0]
        mean = torch.randint(-1, 2, (n,), device="cuda", generator=g).float()
        rstd = torch.randint(1, 3, (n,), device="cuda", generator=g).float()
        base = whole(g, 2, width, torch.float32, 100)
        dx, dg, db = ops.layer_norm_backward(x, gamma, mean, rstd, dy, skip=skip, dgamma=base[0].clone() if accumulate else None,
                                             dbeta=base[1].clone() if accumulate else None, mode=L.GRAD_ACCUMULATE if accumulate else L.GRAD_OVERWRITE)
        wx, wg, wb = R.layer_norm_backward(x, gamma, mean, rstd, dy, skip)
        if accumulate:
            wg, wb = wg + base[0].double(), wb + base[1].double()
        assert torch.equal(dg.double(), wg) and torch.equal(db.double(), wb)
        xh, a = (x.double() - mean.double()[:, None]).abs() * rstd.double()[:, None], (dy.double() * gamma.double()).abs()
        s1 = (dy.double() * gamma.double()).mean(1, keepdim=True).abs()
        s2 = (dy.double() * gamma.double() * (x.double() - mean.double()[:, None]) * rstd.double()[:, None]).mean(1, keepdim=True).abs()
        e = rstd.double()[:, None] * 6 * 2.0 ** -24 * (a + s1 + xh * s2) + 2.0 ** -23 * (0 if skip is None else skip.double().abs())
        R.within("dx", dx, wx, e + R.half_step(t, wx.abs() + e))
