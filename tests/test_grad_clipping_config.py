"""The clipping bound of the training loop in the network configuration (no GPU needed)."""
import copy

import pytest

from test_network_config import DTU


def test_max_grad_norm_key():
    from neus2_b200 import config
    assert config.testbed_config_from_json(DTU).max_grad_norm == 0.0
    cfg = copy.deepcopy(DTU)
    cfg.setdefault("hyperparams", {})["max_grad_norm"] = 0.5
    assert config.testbed_config_from_json(cfg).max_grad_norm == 0.5
    for bad in (-1.0, float("nan"), float("inf")):
        cfg["hyperparams"]["max_grad_norm"] = bad
        with pytest.raises(ValueError, match="max_grad_norm"):
            config.testbed_config_from_json(cfg)
