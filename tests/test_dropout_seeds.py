"""Where the seeds of unstored dropout masks come from."""
import pytest
import torch

import ulm_ops


def seeds():
    torch.manual_seed(5)
    return [ulm_ops.next_dropout_seed() for _ in range(3)]


@pytest.mark.parametrize('device', ['meta', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_seeds_are_the_cpu_generators_under_any_default_device(device):
    want = seeds()
    with torch.device(device):
        assert seeds() == want
    torch.set_default_device(device)
    try:
        assert seeds() == want
    finally:
        torch.set_default_device(None)
