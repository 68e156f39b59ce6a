"""GPU: devices and numbers as arguments of the operators."""
import numpy as np
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


def test_numbers_that_are_no_filter_are_refused(ops, lk):
    x, u = torch.randn(4, 64, device="cuda"), torch.rand(4, device="cuda")
    for kw in (dict(top_k=2.5), dict(top_k=1 << 31), dict(top_k=-(1 << 31) - 1), dict(top_k=float("nan")), dict(top_k=float("inf")), dict(top_k="7"),
               dict(temperature="1"), dict(top_p=[0.5] * 4), dict(min_p=1j), dict(temperature=1e300), dict(top_p=-(2 ** 2000))):
        with pytest.raises(lk.LokiError):
            ops.sample(x, u, **kw)


def test_numbers_of_other_kinds(ops):
    x, u = torch.randn(4, 64, device="cuda"), torch.rand(4, device="cuda")
    want = ops.sample(x, u, temperature=0.5, top_k=7, top_p=0.75, min_p=0.0)
    for kw in (dict(temperature=np.float32(0.5), top_k=np.int64(7), top_p=np.float64(0.75)), dict(temperature=0.5, top_k=7.0, top_p=0.75, min_p=0),
               dict(temperature=0.5, top_k=7, top_p=0.75, min_p=-float("inf"))):
        assert all(torch.equal(a, b) for a, b in zip(want, ops.sample(x, u, **kw)))
