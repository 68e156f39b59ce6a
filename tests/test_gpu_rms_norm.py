"""GPU: the norm with an 8-bit output (ops.rms_norm_i8) against float64.

Bounds.  Let e = 2^-24 (half a step of float32).  h = x + r is one float32 rounding and is taken as
given (the definition's h is float32).  p = h * g: one rounding.  scale = fl(fl(top * inv) / 127): top
carries p's rounding, the product and the quotient one each, inv is float64: 3 e relative, with the
second-order terms under 4 e.  code = rint(fl(p * fl(127 / top))): p, top, the quotient and the product
each e relative of a number up to 127, so a code is at most 1/2 + 127 * 5 e from the exact quotient.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def reference(x, gain, residual, eps):
    h = x.float() if residual is None else x.float() + residual.float()
    p = h.double() * (1.0 if gain is None else gain.double())
    inv = 1.0 / torch.sqrt(h.double().square().mean(1) + eps)
    top = p.abs().amax(1)
    q = torch.where(top[:, None] > 0, p * 127.0 / top[:, None], torch.zeros_like(p))
    return h, q, top * inv / 127.0


def verify(got, x, gain, residual, eps):
    codes, scales, total = got
    h, q, s = reference(x, gain, residual, eps)
    assert codes.dtype == torch.int8 and codes.shape == x.shape
    off = (codes.double() - q).abs().max().item() if q.numel() else 0.0
    assert off <= 0.5 + 127 * 5 * E, off
    live = s > 0
    assert torch.all((scales.double()[live] / s[live] - 1).abs() <= 4 * E)
    assert torch.all(scales[~live] == 0) and torch.all(codes[~live] == 0)
    if residual is None:
        assert total is None
    else:
        assert torch.equal(total, h.to(x.dtype))


def make(rows, dim, dtype, seed, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, dim, generator=g, device="cuda") * 2).to(dtype)
    r = torch.randn(rows, dim, generator=g, device="cuda").to(dtype) if residual else None
    gain = (0.5 + torch.rand(dim, generator=g, device="cuda")).to(dtype)
    return x, r, gain


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (5, 8), (2, 9), (130, 64), (4, 255), (4, 256), (4, 257), (33, 768), (7, 771),
                                      (2, 1024), (2, 1025), (9, 4096), (2, 4104), (3, 8192), (2, 8200), (1, 16384), (2, 20001), (1, 32768)])
def test_against_float64(ops, dtype, rows, dim):
    for residual in (False, True):
        x, r, gain = make(rows, dim, dtype, dim + rows, residual)
        verify(ops.rms_norm_i8(x, gain, residual=r, eps=1e-6), x, gain, r, 1e-6)
    verify(ops.rms_norm_i8(x, eps=1e-5), x, None, None, 1e-5)


@pytest.mark.parametrize("gain_type", [torch.float32, torch.float16, torch.bfloat16])
def test_gain_of_another_type(ops, gain_type):
    x, r, gain = make(5, 200, torch.bfloat16, 3)
    gain = gain.to(gain_type)
    verify(ops.rms_norm_i8(x, gain, residual=r, eps=0.0), x, gain, r, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 100, 777, 4096])
def test_strides_and_untouched_neighbours(ops, dtype, dim):
    """Row strides beyond dim, starts off every boundary; what lies between and behind the rows stays."""
    rows = 6
    for start in (0, 1, 8):
        wide = dim + 40
        def view(kind, fill):
            base = torch.full((rows + 2, wide), fill, dtype=kind, device="cuda")
            return base, base[:rows, start:start + dim]
        x, r, gain = make(rows, dim, dtype, 9)
        bx, vx = view(dtype, 7.0)
        br, vr = view(dtype, 7.0)
        bs, vs = view(dtype, 7.0)
        bc, vc = view(torch.int8, 99)
        vx.copy_(x), vr.copy_(r)
        scales = torch.full((rows + 3,), 5.0, device="cuda")
        codes, s, total = ops.rms_norm_i8(vx, gain, residual=vr, out_codes=vc, out_scales=scales[:rows], out_sum=vs)
        assert codes is vc and total is vs
        verify((codes, s, total), x, gain, r, 1e-6)
        for base, fill in ((bs, 7.0), (bc, 99)):
            left = base.clone()
            left[:rows, start:start + dim] = fill
            assert torch.all(left == fill)
        assert torch.all(scales[rows:] == 5.0)
        assert torch.equal(vx, x) and torch.equal(vr, r)


@pytest.mark.parametrize("into", ["x", "residual"])
def test_sum_in_place(ops, into):
    for dim in (96, 101, 5000):
        x, r, gain = make(4, dim, torch.float16, 21)
        want = ops.rms_norm_i8(x, gain, residual=r)
        x2, r2 = x.clone(), r.clone()
        got = ops.rms_norm_i8(x2, gain, residual=r2, out_sum=x2 if into == "x" else r2)
        for a, b in zip(want, got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dim", [40, 1000, 9000])
def test_zero_rows_and_rows_that_are_not_finite(ops, dim):
    x, r, gain = make(8, dim, torch.float32, 5)
    r = r * 0
    x[1] = 0
    x[2, dim - 1] = float("nan")
    x[3, 0] = float("inf")
    x[4, dim // 2] = float("-inf")
    codes, scales, total = ops.rms_norm_i8(x, gain, residual=r, eps=1e-6)
    assert scales[1] == 0 and torch.all(codes[1] == 0)
    assert torch.all(torch.isnan(scales[2:5])) and torch.all(codes[2:5] == 0)
    good = [0, 5, 6, 7]
    verify((codes[good], scales[good], total[good]), x[good], gain, r[good], 1e-6)
    gain[3] = float("nan")  # every row then has a NaN
    assert torch.all(torch.isnan(ops.rms_norm_i8(x, gain)[1]))


@pytest.mark.parametrize("dim", [32, 500, 8192, 20000])
@pytest.mark.parametrize("scale", [1e-40, 1e-33, 1e-20, 1e18, 3e38])
def test_the_ends_of_the_float_range(ops, dim, scale):
    """Squares, and products with the gain, beyond float32's range: the row's codes are what they would be at scale 1.
    (1e-40 is a float32 with 2^-149 / 1e-40 of rounding: the inputs are taken as they are stored.)"""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = ((torch.rand(3, dim, generator=g, device="cuda") * 2 - 1).double() * scale).float()
    gain = 1 + torch.rand(dim, generator=g, device="cuda") * 7
    codes, scales, _ = ops.rms_norm_i8(x, gain, eps=0.0)
    _, q, s = reference(x, gain, None, 0.0)
    assert (codes.double() - q).abs().max() <= 0.5 + 127 * 5 * E
    assert torch.all((scales.double() / s - 1).abs() <= 4 * E)


def test_lowest_values_of_the_type(ops):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.full((2, 300), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        codes, scales, _ = ops.rms_norm_i8(x, torch.full((300,), 2.0, dtype=dtype, device="cuda"), eps=0.0)
        assert torch.all(codes == -127)
        assert torch.all((scales.double() * 127 / 2 - 1).abs() <= 4 * E)


def test_unit_gain_makes_the_rows_of_an_int8_index(ops, lk):
    """With unit gain and eps 0 the codes are those an LK_I8 index stores for the same rows, its scales times sqrt(dim).
    The index rounds the normalised element before it divides, so a quotient next to a half may fall to the other side: the codes
    are held to one step, and to be equal where the exact quotient is not within 127 * 8 e of a half."""
    x, _, _ = make(50, 768, torch.float32, 77, residual=False)
    codes, scales, _ = ops.rms_norm_i8(x, eps=0.0)
    idx = lk.DeviceIndex(768, lk.LK_I8)
    idx.append(x.cpu().numpy())
    want, want_scales = idx.read_rows()
    idx.close()
    _, q, _ = reference(x, None, None, 0.0)
    clear = ((q - q.floor() - 0.5).abs() > 127 * 8 * E).cpu()
    assert torch.equal(codes.cpu()[clear], torch.from_numpy(want)[clear])
    assert (codes.cpu().int() - torch.from_numpy(want).int()).abs().max() <= 1
    ratio = scales.cpu().double() / (torch.from_numpy(want_scales).double() * 768 ** 0.5)
    assert (ratio - 1).abs().max() <= 8 * E


def test_no_rows(ops):
    codes, scales, total = ops.rms_norm_i8(torch.empty(0, 64, device="cuda"), residual=torch.empty(0, 64, device="cuda"))
    assert codes.shape == (0, 64) and scales.shape == (0,) and total.shape == (0, 64)


def test_many_rows(ops):
    x, r, gain = make(70000, 16, torch.bfloat16, 1)
    verify(ops.rms_norm_i8(x, gain, residual=r), x, gain, r, 1e-6)


def test_refusals(ops, lk):
    x, r, gain = make(4, 32, torch.float16, 0)
    bad = [dict(x=x[0]), dict(x=x.cpu()), dict(x=x.to(torch.float64)), dict(x=x.t()), dict(gain=gain[:-1]), dict(gain=gain.cpu()),
           dict(residual=r.float()), dict(residual=r[:2]), dict(out_codes=torch.empty(4, 32, device="cuda")), dict(eps=-1.0),
           dict(out_scales=torch.empty(4, dtype=torch.float16, device="cuda")), dict(x=x[:1].expand(4, 32)), dict(x=x.clone().requires_grad_())]
    for kw in bad:
        a = dict(x=x, gain=gain, residual=None)
        a.update(kw)
        with pytest.raises(lk.LokiError):
            ops.rms_norm_i8(a.pop("x"), a.pop("gain"), **a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", [(592, 264), (700, 1024), (3001, 1032), (1500, 2048), (900, 2056), (2000, 4096), (600, 4104), (640, 8192), (600, 8200)])
def test_many_wide_rows(ops, dtype, rows, dim):
    """Enough rows to stream: every width of thread and stage."""
    for residual in (False, True):
        x, r, gain = make(rows, dim, dtype, dim + rows, residual)
        verify(ops.rms_norm_i8(x, gain, residual=r, eps=1e-6), x, gain, r, 1e-6)
    verify(ops.rms_norm_i8(x, gain.float(), eps=1e-6), x, gain.float(), None, 1e-6)
    verify(ops.rms_norm_i8(x, eps=1e-6), x, None, None, 1e-6)


@pytest.mark.parametrize("dim", [512, 4096])
@pytest.mark.parametrize("into", ["new", "x", "residual"])
def test_odd_rows_among_many(ops, dim, into):
    """Zeros, NaN, infinities, and rows at the ends of the float range between ordinary ones; the sum in place or not."""
    rows = 1900
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(rows, dim, generator=g, device="cuda")
    r = torch.randn(rows, dim, generator=g, device="cuda")
    gain = 1 + torch.rand(dim, generator=g, device="cuda") * 7
    kinds = torch.arange(rows, device="cuda") % 97
    x[kinds == 3] = 0
    r[kinds == 3] = 0
    x[kinds == 10, dim // 3] = float("nan")
    r[kinds == 20, 0] = float("inf")
    x[kinds == 30, dim - 1] = float("-inf")
    for kind, size in ((40, 1e38), (50, 1e-38), (60, 3e-41)):
        x[kinds == kind] *= size
        r[kinds == kind] *= size
    x[kinds == 70] = torch.finfo(torch.float32).max
    r[kinds == 70] = 0
    a, b = x.clone(), r.clone()
    out = None if into == "new" else (a if into == "x" else b)
    codes, scales, total = ops.rms_norm_i8(a, gain, residual=b, eps=0.0, out_sum=out)
    broken = (kinds == 10) | (kinds == 20) | (kinds == 30)
    h = x + r
    broken |= ~torch.isfinite(h).all(1)  # 1e38 times a normal number can pass the end of the range
    assert torch.all(torch.isnan(scales[broken])) and torch.all(codes[broken] == 0)
    verify((codes[~broken], scales[~broken], total[~broken]), x[~broken], gain, r[~broken], 0.0)
    assert torch.equal(torch.nan_to_num(total[broken]), torch.nan_to_num(h[broken]))


def test_no_wait_has_run_out(ops):
    """All calls of this file: none gave up waiting for a copy."""
    ops.check_device()
