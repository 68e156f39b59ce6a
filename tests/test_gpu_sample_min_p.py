"""GPU: min-p above 1 (ops.sample), which is taken as 1: the entries that weigh as much as the largest."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


@pytest.mark.parametrize("vocab", [40, 5000, 70000, 300000])
@pytest.mark.parametrize("least", [1.0, 1.5, 2.0, float("inf")])
def test_above_one(ops, vocab, least):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(4, vocab, generator=g, device="cuda")
    x[1, [3, 17, 30]] = 50.0
    u = torch.tensor([0.1, 0.5, 0.9, 0.4], device="cuda")
    ids, probs, kept = ops.sample(x, u, min_p=least)
    assert kept.tolist() == [1, 3, 1, 1]
    assert ids.tolist() == [int(x[0].argmax()), 17, int(x[2].argmax()), int(x[3].argmax())]
    assert torch.equal(probs.cpu(), torch.tensor([1.0, 1 / 3, 1.0, 1.0]))
    # at an infinite temperature all weigh the same
    kept = ops.sample(x, u, min_p=least, temperature=float("inf"))[2]
    assert kept.tolist() == [vocab] * 4
    kept = ops.sample(x, u, min_p=least, temperature=float("inf"), top_k=30)[2]
    assert kept.tolist() == [30] * 4
