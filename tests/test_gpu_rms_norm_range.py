"""GPU: the norm with an 8-bit output where h * gain, or the normed value, leaves float32's range.

The definition is y = h / sqrt(mean(h^2) + eps) * gain, scale = max|y| / 127, code = round(y / scale), and only h and the
results are held in float32.  Bounds, with e = 2^-24: scale 4 e relative (p = h * g, the maximum's product and the quotient one rounding
each), codes 1/2 + 127 * 5 e from the exact quotient.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
MAX = torch.finfo(torch.float32).max
TINY = 2.0 ** -149


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def verify(got, h, gain, eps):
    codes, scales = got[:2]
    p = h.double() * gain.double()
    top = p.abs().amax(1)
    q = torch.where(top[:, None] > 0, p * 127.0 / top[:, None], torch.zeros_like(p))
    s = torch.where(top > 0, top / torch.sqrt(h.double().square().mean(1) + eps) / 127.0, torch.zeros_like(top))
    over = s > MAX * (1 + E / 2)
    assert torch.all(torch.isnan(scales[over])) and torch.all(codes[over] == 0)
    fine = ~over
    assert torch.all((codes[fine].double() - q[fine]).abs() <= 0.5 + 127 * 5 * E)
    assert torch.all((scales[fine].double() - s[fine]).abs() <= s[fine] * 4 * E + TINY)
    return over


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("dim", [32, 333, 512, 4096, 8192, 20000])
@pytest.mark.parametrize("size,gains", [(1e-30, 1e-20), (1e-40, 1e-10), (1e-44, 0.4), (1e-20, 1e-27)])
def test_products_that_underflow(ops, rows, dim, size, gains):
    """Every h * gain is 0 in float32, and h is not."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    h = ((torch.rand(rows, dim, generator=g, device="cuda") * 2 - 1).double() * size).float()
    gain = ((0.1 + 0.9 * torch.rand(dim, generator=g, device="cuda")) * gains)
    h[0] = 0
    codes, scales, _ = ops.rms_norm_i8(h, gain, eps=0.0)
    verify((codes, scales), h, gain, 0.0)
    assert scales[0] == 0 and torch.all(codes[0] == 0)
    # a sum in the place of one of its inputs
    r = h.clone()
    x = torch.zeros_like(h)
    again = ops.rms_norm_i8(x, gain, residual=r, eps=0.0, out_sum=r)
    assert torch.equal(again[0], codes) and torch.equal(again[1], scales) and torch.equal(r, h)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_products_that_underflow_in_16_bit_rows(ops, dtype):
    h = torch.full((5, 264), float(torch.finfo(dtype).tiny), dtype=dtype, device="cuda")
    h[:, ::2] *= -0.5
    gain = torch.full((264,), 1e-42, device="cuda")
    verify(ops.rms_norm_i8(h, gain, eps=0.0), h.float(), gain, 0.0)


@pytest.mark.parametrize("rows", [2, 700])
@pytest.mark.parametrize("dim", [40, 512, 1000])
def test_gains_of_zero(ops, rows, dim):
    """h is not 0 and every y is: scale 0, codes 0."""
    x = torch.randn(rows, dim, device="cuda")
    codes, scales, _ = ops.rms_norm_i8(x, torch.zeros(dim, device="cuda"), eps=1e-6)
    assert torch.all(codes == 0) and torch.all(scales == 0)
    gain = torch.zeros(dim, device="cuda")
    gain[dim // 2] = 1e-30
    x *= 1e-20
    verify(ops.rms_norm_i8(x, gain, eps=0.0), x, gain, 0.0)


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("dim", [20, 500, 4096, 8192, 16129, 16384, 20001, 32768])
@pytest.mark.parametrize("gains", [1e30, 3e37, 3e38])
def test_values_past_the_range_whose_scale_is_not(ops, rows, dim, gains):
    """One element carries its row, so that the largest y is sqrt(dim) * gain: past float32, where the scale, a 127th of it, is a
    float32 up to dim = 16,129, and beyond with smaller gains.  Where it is not, the row is not finite."""
    if rows > 1 and dim > 8192:
        rows = 5
    h = torch.zeros(rows, dim, device="cuda")
    at = torch.arange(rows, device="cuda") * 7 % dim
    h[torch.arange(rows, device="cuda"), at] = 1.0
    h[:, 3] += 0.125
    gain = torch.full((dim,), gains, device="cuda")
    over = verify(ops.rms_norm_i8(h, gain, eps=0.0), h, gain, 0.0)
    assert bool(over.all()) == (gains == 3e38 and dim > 20001)
    x = torch.zeros_like(h)
    got = ops.rms_norm_i8(x, gain, residual=h, eps=0.0, out_sum=x)
    verify(got, h, gain, 0.0)
    assert torch.equal(x, h)
