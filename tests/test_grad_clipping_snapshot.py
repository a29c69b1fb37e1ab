"""The clipping bound in the configuration that a snapshot carries (no GPU needed)."""
import copy

import pytest

from test_network_config import DTU


@pytest.mark.parametrize("bound", [0.5, 0.1, 1e-6, 3e30])
def test_a_snapshots_configuration_keeps_the_clipping_bound(bound):
    """Training that goes on from a snapshot with its own configuration clips as before."""
    from neus2_b200 import config, snapshot
    cfg = copy.deepcopy(DTU)
    cfg.setdefault("hyperparams", {})["max_grad_norm"] = bound
    first = config.testbed_config_from_json(cfg)
    again = config.testbed_config_from_json(snapshot.network_config(first))
    assert again.max_grad_norm == first.max_grad_norm > 0.0


def test_without_clipping_the_configuration_is_the_references():
    from neus2_b200 import config, snapshot
    doc = snapshot.network_config(config.testbed_config_from_json(DTU))
    assert sorted(doc["hyperparams"]) == ["anneal_end", "batch_size", "ek_loss_weight", "mask_loss_weight"]
