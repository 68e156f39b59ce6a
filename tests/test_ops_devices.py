"""CPU: devices that cannot be checked are refused before the library is asked."""
import pytest
import torch

from loki_b200 import _lib, ops


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu"), "meta"])
def test_only_cuda_devices(device):
    with pytest.raises(_lib.LokiError, match="CUDA device"):
        ops.check_device(device)


@pytest.mark.parametrize("device", ["cuda", torch.device("cuda"), None, 0, "cuda:0", -1, 4096])
def test_without_a_device(device):
    if _lib.device_count() > 0 and device not in (-1, 4096):
        pytest.skip("there is a CUDA device")
    with pytest.raises(_lib.LokiError):
        ops.check_device(device)
