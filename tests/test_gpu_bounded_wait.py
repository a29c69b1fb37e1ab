"""The bounded wait inside the layers' kernels runs out on a barrier that nothing completes, and says so."""
import subprocess

import pytest

from test_tcnn_headers import built


@pytest.mark.gpu
def test_a_wait_that_nothing_ends_runs_out():
    exe = built("test_bounded_wait", need_build=False) or built("test_bounded_wait")
    if exe is None:
        pytest.skip("no prebuilt test binary")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "bounded wait ok" in r.stdout
