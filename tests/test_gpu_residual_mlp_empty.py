"""The "ResidualMLP" network of the headers on an empty batch, as a C++ program uses it."""
import subprocess

import pytest

from test_tcnn_headers import built


@pytest.mark.gpu
def test_gradients_of_an_empty_batch():
    exe = built("test_residual_mlp_empty", need_build=False) or built("test_residual_mlp_empty")
    if exe is None:
        pytest.skip("no nlohmann/json.hpp on this machine and no prebuilt test binary")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "empty batches ok" in r.stdout
