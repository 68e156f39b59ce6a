"""GPU: draws (ops.sample) from rows of up to LK_SAMPLE_MAX_VOCAB scores, most of whose entries weigh next to nothing.

A sum of weights is off by at most 2^-26 of the row's weight (a quarter of what u itself resolves): B below is that with the 2e-12
of the weights' series and the 1e-9 that float64 sums of 2^24 entries can lose here.  So the running sum reaches u times the row's at the entry
drawn, to B of the row's weight; a cut by top-p falls where the sum reaches its share, to 2 B; and the probability is within
2^-24 (its rounding) and 2 B relative, and within 2^-48 absolute (one weight's rounding, twice over).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
B = 2.0 ** -26 + 2e-12 + 1e-9
MOST = 1 << 24


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def verify(ops, x, u, top_p=None, temperature=None):
    ids, probs, kept = ops.sample(x, u, top_p=top_p, temperature=temperature)
    for r in range(len(u)):
        row = x[r].double()
        t = 1.0 if temperature is None else float(temperature[r])
        top = row.max()
        w = torch.where(row == top, 1.0, torch.where(row > float("-inf"), torch.exp((row - top) / t), 0.0))
        total = float(w.sum())
        n = int(kept[r])
        p = 1.0 if top_p is None else float(top_p[r])
        if p < 1:  # the first n of the order, ties by index
            order = torch.sort(row, descending=True, stable=True)[1]
            run = torch.cumsum(w[order], 0)
            assert float(run[n - 1]) >= (p - 2 * B) * total, (r, n)
            assert n == 1 or float(run[n - 2]) < (p + 2 * B) * total, (r, n)
            mask = torch.zeros_like(w)
            mask[order[:n]] = w[order[:n]]
            w = mask
        else:
            assert n == int((row > float("-inf")).sum())
        run = torch.cumsum(w, 0)
        whole, at, want = float(run[-1]), int(ids[r]), float(u[r]) * float(run[-1])
        before = float(run[at - 1]) if at else 0.0
        assert before - B * whole <= want <= float(run[at]) + B * whole, (r, at, before, want, float(run[at]))
        assert float(w[at]) > 0
        q = float(w[at]) / whole
        assert abs(float(probs[r]) - q) <= q * (2.0 ** -24 + 2 * B) * 1.01 + 2.0 ** -48, (r, q, float(probs[r]))
    return ids, probs, kept


US = [0.0, 0.3, 1 - 2.0 ** -15, 1 - 2.5 * 2.0 ** -17, 1 - 2.0 ** -18, 1 - 2.0 ** -22, 1 - 2.0 ** -24]


@pytest.mark.parametrize("vocab", [MOST, MOST - 77, 3_000_000, 1_000_003, 400_000])
@pytest.mark.parametrize("depth", [15.0, 27.0, 27.1])
def test_one_score_and_a_flat_tail(ops, vocab, depth):
    """At a depth of 27 the tail of the longest row has 3e-5 of the weight, in entries of 2e-12."""
    x = torch.full((2, vocab), -depth, device="cuda")
    x[0, 5] = 0.0
    x[1, vocab - 2] = 0.0
    for u in US:
        verify(ops, x, torch.full((2,), u, device="cuda"))
    tail = (vocab - 1) * np.exp(-depth)
    p = torch.tensor([1 - 0.7 * tail / (1 + tail), 1 - 0.2 * tail / (1 + tail)], device="cuda").float()
    verify(ops, x, torch.tensor([0.9, 1 - 2.0 ** -20], device="cuda"), top_p=p)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_rows(ops, dtype):
    x = torch.full((1, MOST), -27.0, dtype=dtype, device="cuda")
    x[0, MOST // 2] = 0.0
    for u in US:
        verify(ops, x, torch.full((1,), u, device="cuda"))


@pytest.mark.parametrize("temperature", [0.1, 1.0, 30.0, float("inf")])
def test_scattered_peaks(ops, temperature):
    """A peak in every stretch of 500 entries, so that no part of the row is without weight, and a flat rest."""
    x = torch.full((1, MOST), -24.0 * min(temperature, 100.0), device="cuda")
    x[0, ::500] = 0.0
    x[0, 1::7000] = float("-inf")
    x[0, 2::9000] = float("nan")
    t = torch.full((1,), temperature, device="cuda")
    for u in (0.0, 0.123456, 0.5, 0.87654, 1 - 2.0 ** -24):
        verify(ops, x.nan_to_num(nan=float("-inf"), neginf=float("-inf")), torch.full((1,), u, device="cuda"), temperature=t)
        a = ops.sample(x, torch.full((1,), u, device="cuda"), temperature=t)
        b = ops.sample(x.nan_to_num(nan=float("-inf"), neginf=float("-inf")), torch.full((1,), u, device="cuda"), temperature=t)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("vocab", [MOST, 700_001])
def test_spread_scores(ops, vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(3, vocab, generator=g, device="cuda") * torch.tensor([[0.01], [2.5], [6.0]], device="cuda")
    u = torch.rand(3, generator=g, device="cuda")
    verify(ops, x, u)
    verify(ops, x, u, top_p=torch.tensor([0.3, 0.9, 0.999], device="cuda"))
    verify(ops, x + 1000.0, u, top_p=torch.tensor([0.3, 0.9, 0.999], device="cuda"))


def test_rows_where_nothing_else_weighs(ops):
    """Infinities, and temperatures at which the next lower score weighs nothing: the largest share all, to the longest row."""
    inf = float("inf")
    x = torch.zeros(4, MOST, device="cuda")
    x[1] = inf
    x[2, 77::3] = inf
    x[3] = 3e38
    u = torch.tensor([0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    ids, probs, kept = ops.sample(x, u, temperature=torch.tensor([1e-30, 1.0, 1.0, 1e-10], device="cuda"))
    assert ids.tolist() == [MOST // 4, MOST // 2, 77 + 3 * int(0.75 * ((MOST - 77 + 2) // 3)), MOST - 1]
    assert kept.tolist() == [MOST] * 4
    assert probs[[0, 1, 3]].tolist() == [2.0 ** -24] * 3


def test_the_same_on_every_call(ops):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(2, 5_000_000, generator=g, device="cuda") * 4
    u = torch.rand(2, generator=g, device="cuda")
    first = ops.sample(x, u, top_p=0.97)
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.sample(x, u, top_p=0.97)))
