"""The comparisons of the gradients' sums over the samples notice a tile that is left out (planted here, on the CPU, in the sum itself)."""
import pytest
import torch

import dense_reference as R
from dense_sums import sum_bound, whole


@pytest.mark.parametrize("n,i,o", [(100000, 64, 64), (150001, 64, 128), (33333, 129, 65), (8192, 256, 300)])
def test_one_tile_left_out_is_noticed(n, i, o):
    g = torch.Generator()
    g.manual_seed(n)
    x, dz = torch.randn((n, i), generator=g).double(), (0.1 * torch.randn((n, o), generator=g)).double()
    left = torch.ones(n, 1, dtype=torch.float64)
    left[n // 256 * 128:n // 256 * 128 + 128] = 0.0
    for got, want, mag in (((dz * left).T @ x, dz.T @ x, dz.abs().T @ x.abs()), ((dz * left).sum(0), dz.sum(0), dz.abs().sum(0))):
        bound = sum_bound(n, mag)
        R.within("the whole sum in 32 bits", want.float(), want, bound)
        with pytest.raises(AssertionError):
            R.within("a tile short", got, want, bound)
        # not by a few entries: by many of them
        assert float(((got - want).abs() > bound).double().mean()) > 0.1
    xi, zi = whole(g, n, i, torch.float64), whole(g, n, o, torch.float64)
    assert float(((zi * left).T @ xi != zi.T @ xi).double().mean()) > 0.9


def test_whole_numbers_survive_every_order_in_32_bits():
    g = torch.Generator()
    g.manual_seed(1)
    x, dz = whole(g, 150001, 3, torch.float32), whole(g, 150001, 5, torch.float32)
    want = dz.double().T @ x.double()
    products = dz[:, :, None] * x[:, None, :]
    for order in (slice(None), torch.randperm(150001, generator=g)):
        assert torch.equal(products[order].cumsum(0)[-1].double(), want)
