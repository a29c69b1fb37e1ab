"""Clipping by the global gradient norm in the training loop (max_grad_norm) and in the optimizer entry points."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from test_gpu_testbed import cuda_view, make_testbed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def scene():
    from neus2_b200 import synthetic as S
    return S.render_sphere_views(12, 128, 128, device="cpu", seed=1)


def gradients(tb, ng):
    ptrs = tb.device_ptrs()
    torch.cuda.synchronize()
    gm = cuda_view(ptrs["grad_mlp"], (12288 + 4) * 4).view(torch.float32).double().cpu().numpy().copy()
    gg = cuda_view(ptrs["grad_grid"], ng * 2).view(torch.float16).double().cpu().numpy().copy()
    return gm, gg


@pytest.mark.parametrize("ratio", [0.25, 4.0])
def test_training_step_is_clipped(scene, ratio):
    """The norm the step reports is that of its gradients without the loss scale, and Adam's first moments after the first step
    are (1 - beta1) times the clipped gradients (plus the weight decay of the matrix weights, which is switched off here)."""
    probe, _, ng = make_testbed(scene, 1 << 12, l2_reg=0.0)
    probe.train_backward()
    gm, gg = gradients(probe, ng)
    expected = math.sqrt((gm ** 2).sum() + (gg ** 2).sum()) / 128.0
    assert expected > 0
    probe.close()
    tb, _, _ = make_testbed(scene, 1 << 12, l2_reg=0.0, max_grad_norm=expected / ratio)
    tb.train_backward()
    gm, gg = gradients(tb, ng)  # (fp32 atomics: not the probe's to the last bit)
    norm = math.sqrt((gm ** 2).sum() + (gg ** 2).sum()) / 128.0
    factor = min(1.0, expected / ratio / norm)
    tb.optimizer_step()
    # the sum is taken in 64 bits and rounded to 32 once; the scale 1/128 is exact
    assert abs(tb.grad_norm - norm) <= 2.0 ** -23 * norm
    n = 12288 + ng + 4
    m = np.zeros(n, np.float32)
    from neus2_b200 import _lib as L
    L.check(L.lib().neus2b_testbed_get_array(tb._h, C.c_int(1), m.ctypes.data_as(C.c_void_p), C.c_uint64(m.nbytes)))
    want = 0.1 * factor * np.concatenate([gm[:12288], gg, gm[12288:]]) / 128.0
    # factor, product, quotient and moment: five roundings to 32 bits (the quotient within two units), and 1 - 0.9 in 32 bits (6e-8 / 0.1)
    assert np.all(np.abs(m - want) <= 2e-6 * np.abs(want) + 1e-30)
    tb.close()


def test_without_the_option_nothing_is_reported_and_bad_bounds_are_refused(scene):
    from neus2_b200 import _lib as L
    from neus2_b200.testbed import Testbed
    tb, _, _ = make_testbed(scene, 1 << 12)
    tb.train_backward()
    tb.optimizer_step()
    assert tb.grad_norm == 0.0
    tb.close()
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(L.Neus2bError):
            Testbed(batch_size=1 << 12, max_grad_norm=bad)


@pytest.mark.parametrize("packed", [False, True])
def test_adam_with_a_gradient_scale_equals_scaled_gradients(packed):
    """d_grad_scale = 2^-k: the same bits as gradients that were scaled beforehand; NULL and 1: the same bits as each other."""
    from neus2_b200 import _lib as L
    from neus2_b200 import ops
    n_matrix, n_grid = 256, 4096
    n = n_matrix + n_grid + 4
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    w = 0.1 * torch.randn(n, device="cuda", generator=g)
    gm, gg, gv = (torch.randn(s, device="cuda", generator=g) for s in (n_matrix, n_grid, 4))
    gg = (gg.sign() * (1 + gg.abs().clamp(max=1))).half()  # a quarter of these is exact in 16 bits
    scale = torch.tensor([9.0, 0.25], device="cuda")
    one = torch.ones(1, device="cuda")

    def step(factor, address):
        a, b, c = gm * factor, (gg.float() * factor).half(), gv * factor
        P = torch.zeros(n, dtype=torch.float16, device="cuda")
        cfg = L.AdamCfg(1e-2, 0.9, 0.99, 1e-15, 1e-3, 0.95, 128.0, 1, n_matrix, 0, None, address)
        if packed:
            S = torch.stack([w, torch.zeros_like(w), torch.zeros_like(w), w], 1).contiguous()
            ops.adam_step_packed(cfg, a, b, c, S, P)
            return S
        W, M, V = w.clone(), torch.zeros_like(w), torch.zeros_like(w)
        ops.adam_step(cfg, a, b, c, W, M, V, P)
        return torch.stack([W, M, V])
    assert torch.equal(step(1.0, scale.data_ptr() + 4), step(0.25, None))
    assert torch.equal(step(1.0, one.data_ptr()), step(1.0, None))
