"""The "ResidualMLP" network of the tiny-cuda-nn-shaped headers (include/tiny-cuda-nn/networks/residual_mlp.h) as a C++ program uses it."""
import subprocess

import pytest

from test_tcnn_headers import built


def test_factory_and_refusals():
    exe = built("test_residual_mlp")
    if exe is None:
        pytest.skip("no nlohmann/json.hpp on this machine and no prebuilt test binary")
    r = subprocess.run([exe, "--check-only"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "host checks ok" in r.stdout


@pytest.mark.gpu
def test_network_and_its_gradients_against_64_bits():
    exe = built("test_residual_mlp", need_build=False) or built("test_residual_mlp")
    if exe is None:
        pytest.skip("no nlohmann/json.hpp on this machine and no prebuilt test binary")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "residual network ok" in r.stdout
