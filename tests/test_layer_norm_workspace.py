"""The workspace of layer norm's backward pass: no more than its variants use, and enough for each of them."""
import ctypes as C

import pytest
import torch

SMS = 148


def workspace(n, width, dtype):
    from neus2_b200 import _lib as L
    need = C.c_uint64(0)
    L.check(L.lib().neus2b_layer_norm_backward_workspace(C.byref(L.LayerNormDesc(n, width, dtype, 0, 1e-5)), C.byref(need)))
    return need.value


def test_size():
    from neus2_b200 import build
    build.build()
    for dtype in (0, 1, 2):
        for width, blocks in ((64, 8), (256, 8), (257, 4), (2048, 4), (2049, 2), (4096, 2), (4097, 1), (8192, 1)):
            assert workspace(1 << 20, width, dtype) == blocks * SMS * 2 * width * 4
            assert workspace(40, width, dtype) == 40 * 2 * width * 4
            assert workspace(32, width, dtype) == 0
        assert workspace(1 << 20, 8193, dtype) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [1, 8, 17, 32, 63, 64, 127, 128, 129, 200, 255, 256, 257, 504, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4096, 4097, 5003, 8184, 8192])
def test_nothing_behind_it_is_written(width, t):
    """Enough rows that every variant runs all its blocks; what lies behind the workspace keeps its marker, and the sums are exact."""
    from dense_sums import whole
    from neus2_b200 import _lib as L
    n = 30001 if width <= 512 else 5001
    g = torch.Generator(device="cuda")
    g.manual_seed(width)
    for pad, offset in ((0, 0), (8, 0), (3, 1)):
        x, dy, dx = (whole(g, n, width, t, pad=pad, offset=offset) for _ in range(3))
        gamma, mean, rstd = torch.ones(width, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
        dg, db = torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
        need = workspace(n, width, L.F32 if t is torch.float32 else L.F16 if t is torch.float16 else L.BF16)
        room = torch.full((need + (1 << 20),), 77, dtype=torch.uint8, device="cuda")
        d = L.LayerNormDesc(n, width, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[t], 0, 1e-5)
        L.check(L.lib().neus2b_layer_norm_backward(C.byref(d), x.data_ptr(), x.stride(0), gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(),
                                                   dy.stride(0), None, 0, dx.data_ptr(), dx.stride(0), dg.data_ptr(), db.data_ptr(), L.GRAD_OVERWRITE, room.data_ptr(),
                                                   need, L.cur_stream()))
        assert bool((room[need:] == 77).all())
        assert torch.equal(dg.double(), (dy.double() * x.double()).sum(0)) and torch.equal(db.double(), dy.double().sum(0))


@pytest.mark.gpu
def test_wide_rows_off_16_byte_boundaries_need_none():
    """Rows beyond the variants for such rows are summed column by column."""
    from dense_sums import whole
    from neus2_b200 import _lib as L
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    n, width, t = 300, 5003, torch.float16
    x, dy = whole(g, n, width, t), whole(g, n, width, t)
    gamma, mean, rstd = torch.ones(width, device="cuda"), torch.zeros(n, device="cuda"), torch.ones(n, device="cuda")
    dg, db = torch.empty(width, device="cuda"), torch.empty(width, device="cuda")
    d = L.LayerNormDesc(n, width, L.F16, L.F32, 1e-5)
    args = [C.byref(d), x.data_ptr(), width, gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), width, None, 0, None, 0, dg.data_ptr(), db.data_ptr(),
            L.GRAD_OVERWRITE, None, 0, L.cur_stream()]
    L.check(L.lib().neus2b_layer_norm_backward(*args))
    assert torch.equal(dg.double(), (dy.double() * x.double()).sum(0)) and torch.equal(db.double(), dy.double().sum(0))
