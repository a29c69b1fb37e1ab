"""Sizes beyond those that the layers of any width take are refused, not cut off to the 32 bits of a descriptor's field.  No GPU: a plan is
made before anything is allocated or launched."""
import pytest
import torch

BEYOND = [(1 << 30) + 1, (1 << 32) - 1, 1 << 32, (1 << 32) + 128, 1 << 40]


@pytest.fixture(scope="module")
def ops():
    from neus2_b200 import build
    build.build()
    from neus2_b200 import ops as o
    return o


@pytest.mark.parametrize("size", BEYOND)
@pytest.mark.parametrize("backward", [False, True], ids=["forward", "backward"])
def test_linear_sizes(ops, size, backward):
    from neus2_b200 import _lib as L
    for sizes in ((size, 4, 4), (4, size, 4), (4, 4, size)):
        with pytest.raises(L.Neus2bError, match="at most"):
            ops._linear_plan(*sizes, torch.float16, 0, backward, 0)
    for sizes in ((1 << 30, 4, 4), (4, 1 << 30, 4), (4, 4, 1 << 30)):
        d, _ = ops._linear_plan(*sizes, torch.float16, 0, backward, 0)
        assert (d.n, d.in_width, d.out_width) == sizes


@pytest.mark.parametrize("size", BEYOND)
def test_layer_norm_sizes(ops, size):
    from neus2_b200 import _lib as L
    for sizes in ((size + (1 << 30), 4), (4, size)):
        with pytest.raises(L.Neus2bError, match="at most"):
            ops._norm_plan(*sizes, torch.float16, torch.float32, 1e-5)
    for sizes in ((1 << 31, 4), (4, 1 << 30)):
        d, _ = ops._norm_plan(*sizes, torch.float16, torch.float32, 1e-5)
        assert (d.n, d.width) == sizes
