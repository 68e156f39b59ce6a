"""GPU: rows of equal scores (ops.sample), where a share of the weight is a share of a count and can be met exactly.

Every entry weighs the same whole number, so a top-p of p keeps ceil(p n) entries of n, and u draws entry floor(u kept): p and u are
taken as the binary fractions that they are, without a rounding on the way.  A quotient of two such sums is 1 / kept to 2^-24.
"""
from fractions import Fraction
from math import ceil, floor

import pytest
import torch

pytestmark = pytest.mark.gpu
SHARES = [0.5, 0.25, 0.75, 0.125, 0.9, 1 / 3, 2.0 ** -20, 1 - 2.0 ** -24]
US = [0.0, 0.5, 0.25, 0.75, 0.375, 1 - 2.0 ** -24, 0.1]


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def check(ops, x, n, shares, **kw):
    """x: rows whose n first scores are equal and the rest masked."""
    for u in US:
        ids, probs, kept = ops.sample(x, torch.full((len(x),), u, device="cuda"), top_p=None if shares is None else torch.tensor(shares, device="cuda"), **kw)
        for r in range(len(x)):
            p = None if shares is None else Fraction(float(torch.tensor(shares[r])))
            want = n if p is None else max(1, ceil(p * n))
            assert int(kept[r]) == want, (r, u)
            at = floor(Fraction(float(torch.tensor(u))) * want)
            assert int(ids[r]) == at, (r, u, want)
            assert abs(float(probs[r]) * want - 1) <= 2.0 ** -24


@pytest.mark.parametrize("value", [0.0, -2.5, 11.0])
@pytest.mark.parametrize("n", [1, 2, 3, 8, 100, 266, 532, 743, 1024, 2048, 9000, 14730, 52562, 81652, 163304, 262144, 262146, 300000, 1 << 20])
def test_shares_of_equal_scores(ops, n, value):
    x = torch.full((len(SHARES), n), value, device="cuda")
    check(ops, x, n, SHARES)
    check(ops, x, n, None)
    check(ops, x, n, SHARES, temperature=0.7)
    if n > 2:
        k = n - n // 3
        check(ops, x, k, SHARES, top_k=k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [600, 50000, 300002])
def test_among_masked_scores(ops, n, dtype):
    x = torch.full((len(SHARES), n + 1000), 3.0, dtype=dtype, device="cuda")
    x[:, n:] = float("-inf")
    check(ops, x, n, SHARES)
    check(ops, x, n, SHARES, min_p=0.5)


def test_the_longest_row(ops):
    n = 1 << 24
    check(ops, torch.zeros(len(SHARES), n, device="cuda"), n, SHARES)
