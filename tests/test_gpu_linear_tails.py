"""GPU: the activations of ops.linear where they are small, relative to their own size.

The product is of zeros and the value comes from the bias, so an activation's input is exact.  Bounds for float32 results, with
e = 2^-24 (half a step), CUDA's stated 2 ulp (4 e) for expf and __fdividef:
SiLU v / (1 + exp(-v)), below 0 v exp(v) / (1 + exp(v)): the exponential 4 e and, halved, again in the sum; a product and the sum e each, the
quotient 4 e: 12 e.
GELU v Phi(v): below 0 Phi is exp(-v^2 / 2) P(t) with t = 1 / (1 + c |v|) to e, to which P is 2.71 times as sensitive; the fit 0.7 e, P's
additions 3 e, the exponential 4 e, products 4 e: 15 e.  Above 0 it is 1 minus such a tail.
GELU (tanh) v / (1 + exp(-t)), t = 2 sqrt(2 / pi) (v + 0.044715 v^3): t carries 7 e (its constants and products), so 7 |t| + 12.
16-bit results use the fast exponential, 2 ulp and 1.17 |its argument| ulp, and for GELU t to 5 e: 27 e, 2.34 v^2 / 2 e for the exponential
and v^2 / 2 e for the square's rounding; for the others 2 e (4 + 4 |t|).  Storing adds half a step of the type.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def exact(v, act):
    from scipy.special import erfc
    if act == "gelu":
        return 0.5 * v * erfc(-v / math.sqrt(2))
    t = v if act == "silu" else 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
    e = np.exp(-np.abs(t))
    return np.where(t >= 0, v / (1 + e), v * e / (1 + e))


def bound(v, act, full):
    x2 = v * v / 2
    if act == "gelu":
        return E * 15 if full else E * (27 + 4 * x2)
    t = np.abs(v if act == "silu" else 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    if not full:
        return 2 * E * (4 + 4 * t)
    return E * 12 if act == "silu" else E * (7 * t + 12)


# to where the result is still a normal float32
REACH = {"silu": 80.0, "gelu": 12.5, "gelu_tanh": 9.0}


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,aligned", [(1, True), (40, True), (300, True), (3, False)])
def test_relative_to_the_result(ops, act, out, m, aligned):
    n, k = 4096, 64
    reach = REACH[act]
    bias = torch.linspace(-reach, reach, n, device="cuda").to(out)
    a = torch.zeros(m, k if aligned else k - 1, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(n, k if aligned else k - 1, dtype=torch.bfloat16, device="cuda")
    got = ops.linear(a, w, bias=bias, act=act, out_dtype=out).double().cpu().numpy()
    v = bias.double().cpu().numpy()
    want = exact(v, act)
    off = np.abs(want) * bound(v, act, out == torch.float32) * 1.001
    if out == torch.float32:
        off += 2.0 ** -149
    else:
        off = off + (np.abs(want) + off) * (torch.finfo(out).eps / 2) + (2.0 ** -25 if out == torch.float16 else 2.0 ** -134)
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), (v[np.nonzero(bad)[1][:4]], got[bad][:4], want[np.nonzero(bad)[1][:4]], (np.abs(got - want) / np.maximum(off, 1e-300)).max())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_the_ends(ops, act):
    """Far out the results are 0 and the value itself, down to the type's lowest and up to its largest; NaN stays NaN."""
    big = torch.finfo(torch.bfloat16).max  # a float32 as well
    v = torch.tensor([-big, -1e30, -1e4, -200.0, -0.0, 0.0, 200.0, 1e4, 1e30, big, float("inf"), float("nan")], device="cuda")
    a, w = torch.zeros(2, 16, dtype=torch.int8, device="cuda"), torch.zeros(12, 16, dtype=torch.int8, device="cuda")
    for out in (torch.float32, torch.bfloat16):
        b = v.to(out)
        got = ops.linear(a, w, bias=b, act=act, out_dtype=out)
        assert torch.all(got[:, :6] == 0) and torch.equal(got[:, 6:11], b[6:11].expand(2, 5)) and torch.all(torch.isnan(got[:, 11]))
