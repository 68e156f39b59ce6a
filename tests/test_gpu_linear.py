"""GPU: the matrix product with its epilogue (ops.linear) against float64.

Bounds, with e = 2^-24 (half a step of float32).  The sum: exact for int8 up to its conversion to
float32 (e); for 16-bit operands products are exact and each of the k additions may lose up to a whole
step (2 e, the tensor cores truncate) of a partial sum that is at most sum |a w|.  The scales add two
roundings, the bias one.  Every activation has a slope of at most 1.13 (the GELUs; SiLU 1.1).  Its own
value v * q, with q in (0, 1): the erf form has q to 4 e absolute; the others compute q = 1 / (1 + exp(-t)),
t = v or 2 z, where t carries up to 6 e relative and the exponential's argument as much again (2 ulp and
|t| * 1.2 ulp where the fast exponential is used): 2 e * (4 + 4 |t|) relative, of which never more than all of it.  The residual adds one rounding
of the result; storing it one half step of the result's type (plus half the smallest float16).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]
FLOATS = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def padded(t, extra=0):
    step = 16 // t.element_size()
    wide = torch.zeros((t.shape[0], (t.shape[1] + step - 1) // step * step + extra), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def operands(m, n, k, dtype, seed, scales=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if dtype == torch.int8:
        a = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
        w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
        unit = 1.0 / (73.0 ** 2 * math.sqrt(max(1, k)))  # codes have a deviation of 73: results of order 1
    else:
        a = torch.randn(m, k, generator=g, device="cuda").to(dtype)
        w = (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(max(1, k))).to(dtype)
        unit = 1.0
    sa = (0.5 + torch.rand(m, generator=g, device="cuda")) * unit if scales else None
    sw = (0.5 + torch.rand(n, generator=g, device="cuda")) if scales else None
    return g, padded(a), padded(w), sa, sw


def reference(a, w, sa, sw, bias, act, residual):
    """(value, bound on the float32 error before the result's rounding)."""
    k = a.shape[1]
    x, y = a.double(), w.double()
    v = x @ y.t()
    size = v.abs() * E if a.dtype == torch.int8 else (x.abs() @ y.abs().t()) * (2 * E * max(1, k))
    s = torch.ones((), dtype=torch.float64, device=a.device)
    if sa is not None:
        s = s * sa.double()[:, None]
    if sw is not None:
        s = s * sw.double()
    v, off = v * s, size * s + 2 * E * (v * s).abs()
    if bias is not None:
        v = v + bias.double()
        off = off + E * v.abs()
    if act == "relu":
        v = v.clamp_min(0)
    elif act == "gelu":
        off = 1.13 * off + 5 * E * v.abs()
        v = v * 0.5 * (1 + torch.erf(v / math.sqrt(2)))
    elif act in ("silu", "gelu_tanh"):
        t = v if act == "silu" else 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        r = v * torch.sigmoid(t)
        off = 1.13 * off + r.abs() * (2 * E * (4 + 4 * t.abs())).clamp_max(1)
        v = r
    if residual is not None:
        v = v + residual.double()
        off = off + E * v.abs()
    return v, off * 1.001 + 1e-36


def verify(ops, a, w, out_dtype, sa=None, sw=None, bias=None, act="none", residual=None, out=None):
    got = ops.linear(a, w, a_scales=sa, w_scales=sw, bias=bias, act=act, residual=residual, out_dtype=out_dtype, out=out)
    want, off = reference(a, w, sa, sw, bias, act, residual)
    assert got.dtype == out_dtype and got.shape == want.shape
    off = off + (want.abs() + off) * (torch.finfo(out_dtype).eps / 2) + (2.0 ** -25 if out_dtype == torch.float16 else 0)
    bad = ((got.double() - want).abs() > off) | torch.isnan(got)
    assert not bad.any(), (bad.sum().item(), bad.nonzero()[:5].tolist(), (got.double() - want).abs().max().item())
    return got


SIZES = [(1, 1, 1), (1, 8, 16), (1, 1000, 768), (2, 17, 33), (3, 4096, 128), (7, 100, 771), (8, 128, 64), (15, 129, 127), (16, 4096, 256), (17, 257, 100),
         (32, 1024, 1024), (33, 300, 513), (64, 64, 2048), (65, 130, 48), (128, 256, 128), (129, 255, 129), (200, 1000, 771), (256, 256, 1024), (257, 513, 257),
         (300, 48, 4096), (513, 1030, 200), (1000, 7, 64), (1111, 2050, 320), (2048, 512, 512)]


@pytest.mark.parametrize("dtype", [torch.int8, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_against_float64(ops, dtype, m, n, k):
    g, a, w, sa, sw = operands(m, n, k, dtype, m * 7 + n)
    for i, out_dtype in enumerate(FLOATS):
        bias = torch.randn(n, generator=g, device="cuda").to(out_dtype)
        residual = torch.randn(m, n, generator=g, device="cuda").to(out_dtype)
        verify(ops, a, w, out_dtype, sa, sw)
        verify(ops, a, w, out_dtype, sa, sw, bias, ACTS[(m + n + i) % 5], residual)


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 520, 256), (20, 136, 192), (140, 264, 64)])
def test_activations(ops, dtype, act, m, n, k):
    g, a, w, sa, sw = operands(m, n, k, dtype, 5)
    for out_dtype in FLOATS:
        bias = (torch.randn(n, generator=g, device="cuda") * 3).to(out_dtype)
        residual = torch.randn(m, n, generator=g, device="cuda").to(out_dtype)
        for b in (None, bias):
            for r in (None, residual):
                verify(ops, a, w, out_dtype, sa, sw, b, act, r)


@pytest.mark.parametrize("act", ACTS)
def test_activations_far_out(ops, act):
    """Values from -200 to 200 through the bias alone: no NaN from an overflowing exponential."""
    a, w = torch.zeros(3, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(401, 64, dtype=torch.bfloat16, device="cuda")
    verify(ops, a, w, torch.float32, bias=torch.arange(-200, 201, device="cuda").float(), act=act)


def test_int8_sums_are_exact(ops):
    """Unit scales and float32 results: whole numbers to 2^24 come out as they are, at the ends of the codes too."""
    for m, n, k in [(1, 300, 1040), (40, 200, 1040), (300, 300, 1040)]:
        g, a, w, _, _ = operands(m, n, k, torch.int8, 11, scales=False)
        a[0] = -128
        w[0] = -128
        got = ops.linear(a, w)
        want = a.double() @ w.double().t()
        assert torch.equal(got.double()[want.abs() <= 2 ** 24], want[want.abs() <= 2 ** 24])
        assert torch.equal(got, want.float())
    a = torch.full((130, 65536), -128, dtype=torch.int8, device="cuda")  # 2^30: the largest sum there is
    assert torch.all(ops.linear(a, a[:50]) == 2.0 ** 30)
    assert torch.all(ops.linear(a[:3], a[:50]) == 2.0 ** 30)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 40, 50), (5, 70, 64), (70, 130, 160), (260, 300, 96)])
def test_rows_off_every_boundary(ops, dtype, m, n, k):
    """Operands that no 16-byte copy can read: odd starts, odd strides."""
    g, a, w, sa, sw = operands(m, n, k, dtype, 2)
    for start, wide in ((1, k + 1), (0, k + 3), (3, k + 24)):
        ba, bw = (torch.zeros(t.shape[0], wide + start, dtype=dtype, device="cuda")[:, start:start + k] for t in (a, w))
        ba.copy_(a), bw.copy_(w)
        verify(ops, ba, bw, torch.float32, sa, sw)
        verify(ops, a, bw, torch.bfloat16, sa, sw)


@pytest.mark.parametrize("m,n", [(1, 200), (6, 131), (50, 96), (140, 300), (300, 264)])
@pytest.mark.parametrize("start", [0, 1, 8])
def test_result_views_and_untouched_neighbours(ops, m, n, start):
    for out_dtype in FLOATS:
        g, a, w, sa, sw = operands(m, n, 80, torch.int8, 4)
        base = torch.full((m + 3, n + 40), 9.0, dtype=out_dtype, device="cuda")
        rb = torch.randn(m, n + 17, generator=g, device="cuda").to(out_dtype)
        out = base[:m, start:start + n]
        verify(ops, a, w, out_dtype, sa, sw, residual=rb[:, start:start + n], out=out)
        left = base.clone()
        left[:m, start:start + n] = 9.0
        assert torch.all(left == 9.0)


@pytest.mark.parametrize("m,n", [(1, 4096), (30, 520), (200, 264), (2100, 2050)])
def test_residual_in_place(ops, m, n):
    g, a, w, sa, sw = operands(m, n, 256, torch.int8, 6)
    r = torch.randn(m, n, generator=g, device="cuda").bfloat16()
    want = ops.linear(a, w, a_scales=sa, w_scales=sw, residual=r)
    got = ops.linear(a, w, a_scales=sa, w_scales=sw, residual=r, out=r)
    assert got is r and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float16])
@pytest.mark.parametrize("m", [1, 5, 40, 150])
def test_nothing_to_add_up(ops, dtype, m):
    """k = 0: the activation of the bias, plus the residual."""
    a, w = torch.empty(m, 0, dtype=dtype, device="cuda"), torch.empty(21, 0, dtype=dtype, device="cuda")
    bias = torch.linspace(-3, 3, 21, device="cuda")
    verify(ops, a, w, torch.float32, bias=bias, act="gelu", residual=torch.ones(m, 21, device="cuda"))
    assert torch.all(ops.linear(a, w, out_dtype=torch.float16) == 0)


def test_no_rows(ops):
    w = torch.zeros(8, 32, dtype=torch.int8, device="cuda")
    assert ops.linear(w[:0], w).shape == (0, 8) and ops.linear(w, w[:0]).shape == (8, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 20, 200])
def test_not_a_number_stays_in_its_row(ops, dtype, m):
    g, a, w, _, _ = operands(m, 150, 100, dtype, 8)
    a[m - 1, 99] = float("nan")
    w[7, 0] = float("inf")
    got = ops.linear(a, w, out_dtype=torch.float32)
    assert torch.all(torch.isnan(got[m - 1]))
    assert not torch.isfinite(got[:, 7]).any()
    if m > 1:
        clean = [j for j in range(150) if j != 7]
        assert torch.isfinite(got[:m - 1][:, clean]).all()


@pytest.mark.parametrize("m,n,k", [(1, 131072, 64), (20000, 8, 64), (9, 70000, 32), (5000, 3000, 48)])
def test_long_sides(ops, m, n, k):
    g, a, w, sa, sw = operands(m, n, k, torch.int8, 13)
    verify(ops, a, w, torch.float32, sa, sw)


def test_results_past_32_bits(ops):
    """More than 2^31 results: the far rows land where they belong."""
    m, n = 70000, 32768
    g, a, w, sa, sw = operands(m, n, 64, torch.int8, 17)
    got = ops.linear(a, w, a_scales=sa, w_scales=sw, out_dtype=torch.float16)
    for rows in (slice(0, 300), slice(65400, 65700), slice(m - 300, m)):
        want, off = reference(a[rows], w, sa[rows], sw, None, "none", None)
        off = off + (want.abs() + off) * 2.0 ** -11 + 2.0 ** -25
        assert torch.all((got[rows].double() - want).abs() <= off)


def test_rows_of_an_index_score_as_a_search(ops, lk):
    """An int8 index's rows as the second operand: the scores are those lk_search reports for the same codes."""
    rng = np.random.default_rng(5)
    rows = rng.standard_normal((3000, 200), dtype=np.float32)
    idx = lk.DeviceIndex(200, lk.LK_I8)
    idx.append(rows)
    codes, scales = idx.read_rows()
    queries = rows[:6] + 0.1
    tmp = lk.DeviceIndex(200, lk.LK_I8)
    tmp.append(queries)
    qc, qs = tmp.read_rows()
    tmp.close()
    dev = lambda v: torch.from_numpy(v).cuda()
    scores = ops.linear(padded(dev(qc)), padded(dev(codes)), a_scales=dev(qs), w_scales=dev(scales))
    ids, want, _, _ = idx.search(queries, 5)
    idx.close()
    got = torch.gather(scores.cpu(), 1, torch.from_numpy(ids))
    np.testing.assert_allclose(got.numpy(), want, rtol=4 * E)  # dot * s * s in another order: two roundings on either side
    assert torch.equal(scores.cpu().amax(1), got[:, 0])


def test_refusals(ops, lk):
    a, w = torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.zeros(8, 32, dtype=torch.int8, device="cuda")
    f = torch.zeros(8, device="cuda")
    for kw in (dict(a=a.cpu()), dict(a=a.float()), dict(w=w.half()), dict(w=w[:, :16]), dict(w=w.cpu()), dict(a=a[0]), dict(a=a.t()), dict(act="tanh"),
               dict(a_scales=f), dict(w_scales=f.half()), dict(bias=f[:7]), dict(bias=f.half(), out_dtype=torch.float32), dict(out_dtype=torch.float64),
               dict(residual=torch.zeros(4, 7, device="cuda")), dict(out=torch.zeros(4, 8, device="cuda"), out_dtype=torch.float16),
               dict(out=torch.zeros(8, 4, device="cuda").t()), dict(out=torch.zeros(1, 8, device="cuda").expand(4, 8)),
               dict(a=a.half().requires_grad_(), w=w.half())):
        p = dict(a=a, w=w)
        p.update(kw)
        with pytest.raises(lk.LokiError):
            ops.linear(p.pop("a"), p.pop("w"), **p)


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
def test_few_slices_many_times(ops, dtype):
    """Products whose copies are all asked for at once: a stage may be used and freed before the warp that asks looks at it."""
    for m, n, k in [(17, 1000, 771), (1, 1000, 300), (40, 512, 1030), (64, 300, 200), (130, 700, 130)]:
        g, a, w, sa, sw = operands(m, n, k, dtype, k)
        first = verify(ops, a, w, torch.float32, sa, sw)
        for _ in range(100):
            again = ops.linear(a, w, a_scales=sa, w_scales=sw, out_dtype=torch.float32)
        assert torch.equal(first, again)
        ops.check_device()


def test_no_wait_has_run_out(ops):
    """All calls of this file: none gave up waiting for a copy."""
    ops.check_device()
