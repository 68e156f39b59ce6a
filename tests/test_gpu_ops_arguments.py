"""GPU: devices as arguments of the operators."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def test_devices_to_check(ops):
    for device in (0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0), None):
        ops.check_device(device)
