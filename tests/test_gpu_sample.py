"""GPU: draws (ops.sample) against a float64 statement on the host.

Whole numbers (the draw, the number kept) have to be equal: the kernel's integer sums are within vocab *
2^-64 * vocab of the exact ones relative to the largest weight (under 1e-9 here), and no seed below puts a
border that near.  The probability is a quotient of two such sums rounded to float32: 2^-24 relative for the
rounding, as much again for the float64 steps and the fixed point, plus 2^-36 of absolute resolution.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def draw_one(x, u, t=1.0, k=0, p=1.0, least=0.0):
    """(id, probability, kept) of one row by the definition."""
    if not t >= 0 or np.isnan(p) or np.isnan(least) or np.isnan(u):
        return -1, 0.0, 0
    there = np.flatnonzero(x > -np.inf)  # False for NaN
    order = there[np.lexsort((there, -x[there]))]
    if t == 0:
        k, t = 1, 1.0
    if k > 0:
        order = order[:k]
    if order.size == 0:
        return -1, 0.0, 0
    top = x[order[0]]
    with np.errstate(all="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t))
    if p < 1:
        running = np.cumsum(w)
        n = 1 + int(np.searchsorted(running, p * running[-1], side="left")) if p > 0 else 1
        order, w = order[:n], w[:n]
    n = max(1, int(np.sum(w >= min(least, 1.0))) if least > 0 else w.size)
    order, w = order[:n], w[:n]
    by_index = np.argsort(order)
    order, w = order[by_index], w[by_index]
    running = np.cumsum(w)
    at = int(np.searchsorted(running, min(max(u, 0.0), 1 - 2.0 ** -24) * running[-1], side="right"))
    at = min(at, int(np.flatnonzero(w)[-1]))
    return int(order[at]), w[at] / running[-1], n


def verify(ops, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    ids, probs, kept = ops.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    host = lambda v, d: np.full(len(u), d) if v is None else v.double().cpu().numpy()
    x = logits.double().cpu().numpy()
    want = [draw_one(*row) for row in zip(x, host(u, 0), host(temperature, 1.0), host(top_k, 0).astype(int), host(top_p, 1.0), host(min_p, 0.0))]
    assert ids.tolist() == [w[0] for w in want]
    assert kept.tolist() == [w[2] for w in want]
    np.testing.assert_allclose(probs.double().cpu().numpy(), [w[1] for w in want], rtol=2 * 2.0 ** -24, atol=2.0 ** -36)
    return ids, probs, kept


def setting(rows, seed, **off):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda: torch.rand(rows, generator=g, device="cuda")
    s = dict(temperature=0.4 + r(), top_k=torch.randint(1, 60, (rows,), generator=g, device="cuda", dtype=torch.int32),
             top_p=0.3 + 0.7 * r(), min_p=0.2 * r())
    s.update(off)
    return g, r(), s


def scores(rows, vocab, dtype, g, spread=2.5):
    return (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (4, 2), (3, 31), (5, 33), (2, 1000), (7, 1024), (3, 1025), (40, 5000), (2, 32003), (1, 131072), (150, 8200)])
def test_filters(ops, dtype, rows, vocab):
    off = [dict(), dict(top_k=None), dict(top_p=None), dict(min_p=None), dict(top_k=None, min_p=None), dict(top_p=None, min_p=None),
           dict(top_k=None, top_p=None), dict(top_k=None, top_p=None, min_p=None), dict(temperature=None, top_k=None, top_p=None, min_p=None)]
    for n, o in enumerate(off):
        g, u, s = setting(rows, 100 * vocab + n, **o)
        verify(ops, scores(rows, vocab, dtype, g), u, **s)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_on_any_stride(ops, dtype):
    g, u, s = setting(6, 8)
    base = scores(8, 3001, dtype, g)
    for start, width in ((0, 2048), (1, 2048), (3, 2997), (8, 1)):
        verify(ops, base[:6, start:start + width], u, **s)


def test_rows_behind_the_last_stay(ops):
    g, u, s = setting(5, 3)
    out = torch.full((9,), 77, dtype=torch.int64, device="cuda")
    ids, _, _ = ops.sample(scores(5, 400, torch.float32, g), u, out_ids=out[:5], **s)
    assert ids.data_ptr() == out.data_ptr() and torch.all(out[5:] == 77) and torch.all(out[:5] < 400)


@pytest.mark.parametrize("vocab", [50, 3000, 70000])
def test_ties_go_to_the_lowest_index(ops, vocab):
    """Scores of few distinct values, so that every cut falls among equals."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randint(0, 4, (12, vocab), generator=g, device="cuda").float()
    x[1] = 0.0
    x[2] = -0.0
    x[2, ::3] = 0.0  # equal to -0
    u = torch.rand(12, generator=g, device="cuda")
    k = torch.randint(1, vocab, (12,), generator=g, device="cuda", dtype=torch.int32)
    verify(ops, x, u, top_k=k)
    p = torch.rand(12, generator=g, device="cuda")
    # equal weights: p * n falls between whole numbers of entries, half an entry from either
    p = ((p * vocab).floor() + 0.5) / vocab
    verify(ops, x[1:3], u[1:3], top_p=p[1:3])
    verify(ops, x[1:3], u[1:3], top_k=k[1:3], top_p=torch.full((2,), 0.33, device="cuda"))


def test_masked_and_empty_rows(ops):
    g, u, s = setting(8, 31, top_k=None, min_p=None)
    x = scores(8, 2000, torch.float32, g)
    x[0] = float("-inf")
    x[1] = float("nan")
    x[2, 1:] = float("-inf")
    x[3, ::2] = float("nan")
    x[4, 5:] = torch.finfo(torch.float32).min
    x[5, 100:200] = float("-inf")
    x[6] = torch.finfo(torch.float32).min
    ids, probs, kept = verify(ops, x, u, **s)
    assert ids[:2].tolist() == [-1, -1] and probs[:2].tolist() == [0, 0] and kept[:2].tolist() == [0, 0]
    assert ids[2] == 0 and probs[2] == 1 and kept[2] == 1
    verify(ops, x.half(), u)
    verify(ops, x.bfloat16(), u, top_k=torch.full((8,), 3, dtype=torch.int32, device="cuda"))


def test_infinite_scores_take_all(ops):
    g, u, _ = setting(4, 6)
    x = scores(4, 900, torch.float32, g)
    x[0, 17] = x[0, 500] = float("inf")
    x[1] = float("inf")
    x[2, 899] = float("inf")
    for kw in (dict(), dict(top_p=torch.full((4,), 0.7, device="cuda")), dict(min_p=torch.full((4,), 0.1, device="cuda"))):
        ids, _, _ = verify(ops, x, u, **kw)
        assert ids[0] in (17, 500) and ids[2] == 899


def test_ends_of_the_settings(ops):
    g = torch.Generator(device="cuda").manual_seed(12)
    f = lambda *v: torch.tensor(v, device="cuda")
    x = scores(6, 700, torch.float32, g)
    x[:, 3] = x[:, 650] = x.amax(1)  # the largest twice
    inf, nan = float("inf"), float("nan")
    u = f(0.0, 1.0, -3.0, 2.0, 1 - 2.0 ** -24, 0.5)
    verify(ops, x, u)
    assert verify(ops, x, u, temperature=f(0.0, 0.0, 0.0, 0.0, 0.0, 0.0))[0].tolist() == [3] * 6
    verify(ops, x, u, temperature=f(1e-30, 1e-3, 1e3, 1e30, 3e38, inf))
    assert verify(ops, x, u, temperature=f(-1.0, nan, -inf, 1.0, 1.0, 1.0))[0][:3].tolist() == [-1] * 3
    verify(ops, x, u, top_p=f(0.0, -1.0, 1.0, 2.0, inf, nan))
    verify(ops, x, u, min_p=f(0.0, -1.0, 1.0, 2.0, inf, nan))
    verify(ops, x, u, top_k=torch.tensor([0, -5, 1, 699, 700, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    u[5] = nan
    assert verify(ops, x, u)[0][5] == -1


def test_long_rows(ops):
    g, u, s = setting(3, 4, top_k=None, min_p=None)
    verify(ops, scores(3, 1_000_003, torch.float32, g), u, **s)
    verify(ops, scores(1, 3_000_000, torch.bfloat16, g), u[:1], top_k=torch.full((1,), 1000, dtype=torch.int32, device="cuda"))


def test_numbers_for_all_rows(ops):
    g, u, _ = setting(4, 1)
    x = scores(4, 500, torch.float32, g)
    a = ops.sample(x, u, temperature=0.7, top_k=20, top_p=0.9, min_p=0.01)
    f = lambda v: torch.full((4,), v, device="cuda")
    b = ops.sample(x, u, temperature=f(0.7), top_k=f(20).int(), top_p=f(0.9), min_p=f(0.01))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_draws_follow_the_weights(ops):
    """An evenly spaced u visits every kept entry as often as its weight says, to one turn in 4,096 either way."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 2.0, 0.5, -3.0]], device="cuda")
    n = 4096
    u = (torch.arange(n, device="cuda") / n).float()
    ids, probs, kept = ops.sample(x.expand(n, 7).contiguous(), u, temperature=0.8, top_k=5)
    w = torch.exp(x[0].double() / 0.8)
    w[[3, 6]] = 0
    want = w / w.sum()
    assert torch.all(kept == 5)
    share = torch.bincount(ids, minlength=7).double() / n
    assert (share - want).abs().max() <= 1.0 / n + 1e-12
    assert torch.allclose(probs.double(), want[ids], rtol=2.0 ** -23)
    assert torch.all(ids[1:] >= ids[:-1])  # the running sum is over ascending indexes


def test_no_rows_and_no_vocabulary(ops):
    assert ops.sample(torch.empty(0, 10, device="cuda"), torch.empty(0, device="cuda"))[0].shape == (0,)
    ids, probs, kept = ops.sample(torch.empty(3, 0, device="cuda"), torch.zeros(3, device="cuda"))
    assert ids.tolist() == [-1] * 3 and probs.tolist() == [0] * 3 and kept.tolist() == [0] * 3


def test_refusals(ops, lk):
    x, u = torch.zeros(4, 32, device="cuda"), torch.zeros(4, device="cuda")
    for kw in (dict(scores=x.cpu()), dict(scores=x.double()), dict(scores=x[0]), dict(scores=x.t()), dict(u=u[:3]), dict(u=u.double()), dict(u=u.cpu()),
               dict(temperature=u[:2]), dict(top_k=u), dict(top_p=u.half()), dict(min_p=u.cpu()), dict(out_ids=u.int()),
               dict(scores=x[:1].expand(4, 32)), dict(scores=x.clone().requires_grad_())):
        a = dict(scores=x, u=u)
        a.update(kw)
        with pytest.raises(lk.LokiError):
            ops.sample(a.pop("scores"), a.pop("u"), **a)


@pytest.mark.parametrize("vocab", [9000, 140001])
@pytest.mark.parametrize("offset", [0.0, 1e4, -1e6])
@pytest.mark.parametrize("spread", [1e-3, 0.1, 30.0, 1e4])
def test_scores_of_any_size(ops, vocab, spread, offset):
    """Nearly flat rows, rows that one score rules, scores far from zero (float32 then holds few distinct ones: many ties)."""
    g, u, s = setting(5, int(vocab + spread * 7 + offset % 97), top_k=None, min_p=None)
    x = scores(5, vocab, torch.float32, g, spread) + offset
    verify(ops, x, u, **s)
    verify(ops, x, u, top_p=s["top_p"], min_p=0.1 * s["top_p"])
    verify(ops, x, u, temperature=s["temperature"], top_k=torch.randint(600, 5000, (5,), generator=g, device="cuda", dtype=torch.int32), top_p=s["top_p"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ties_across_a_long_row(ops, dtype):
    """131,072 scores of a few hundred distinct values: every cut falls among thousands of equals, spread over all CTAs of the row."""
    g = torch.Generator(device="cuda").manual_seed(40)
    x = (torch.randint(-30, 5, (4, 131072), generator=g, device="cuda") / 8.0).to(dtype)
    u = torch.rand(4, generator=g, device="cuda")
    verify(ops, x, u, top_k=torch.tensor([700, 9000, 60000, 131071], dtype=torch.int32, device="cuda"))
    verify(ops, x, u, top_p=torch.tensor([0.11, 0.37, 0.73, 0.991], device="cuda"))
    verify(ops, x, u, top_k=torch.tensor([700, 9000, 60000, 131071], dtype=torch.int32, device="cuda"), top_p=torch.full((4,), 0.613, device="cuda"))


def test_all_equal_in_a_long_row(ops):
    x = torch.full((3, 200000), -2.5, device="cuda")
    u = torch.tensor([0.0, 0.31234, 0.99], device="cuda")
    n = torch.tensor([1000, 70000, 199999], device="cuda")
    verify(ops, x, u, top_p=((n + 0.5) / 200000).float())
    verify(ops, x, u, top_k=n.int())
    verify(ops, x, u, temperature=torch.full((3,), 1e-20, device="cuda"))


def test_temperatures_in_a_long_row(ops):
    g = torch.Generator(device="cuda").manual_seed(3)
    t = torch.tensor([1e-38, 1e-6, 1e-2, 0.3, 5.0, 1e4, 1e30, 3e38], device="cuda")
    x = scores(8, 70000, torch.float32, g)
    u = torch.rand(8, generator=g, device="cuda")
    verify(ops, x, u, temperature=t)
    verify(ops, x, u, temperature=t, top_p=torch.full((8,), 0.777, device="cuda"))
    verify(ops, x, u, temperature=t, min_p=torch.full((8,), 0.3, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [20001, 131072])
@pytest.mark.parametrize("p", [0.5, 0.8, 0.9, 0.95, 0.99, 0.999])
def test_weight_on_few_entries(ops, dtype, vocab, p):
    """Peaked rows: a cut's place cannot be told well from how many entries there are at which distance."""
    g = torch.Generator(device="cuda").manual_seed(int(1000 * p) + vocab)
    t = torch.tensor([0.3, 0.5, 0.8, 1.0] * 2, device="cuda")
    verify(ops, scores(8, vocab, dtype, g, 3.0), torch.rand(8, generator=g, device="cuda"), temperature=t,
           top_p=torch.full((8,), p, device="cuda"))


@pytest.mark.parametrize("each", [20, 150, 700])
@pytest.mark.parametrize("lowest", [1.0, 4.0, 9.0])
def test_distances_at_the_ends_of_stretches(ops, each, lowest):
    """Distances just past a 128th of an octave for the upper half of the row and just short of one for the lower: a mean
    over each 128th is wrong in one direction above and in the other below."""
    g = torch.Generator(device="cuda").manual_seed(each)
    edges = torch.cat([2.0 ** e * (1 + torch.arange(128, device="cuda", dtype=torch.float64) / 128) for e in range(-3, 4)])
    edges = edges[edges < lowest]
    half = edges.numel() // 2
    d = torch.cat([edges[:half] * (1 + 1e-4), edges[half:] * (1 - 1e-4)])
    x = torch.cat([torch.zeros(1, device="cuda", dtype=torch.float64), -d.repeat(each)]).float()
    x = torch.stack([x[torch.randperm(x.numel(), generator=g, device="cuda")] for _ in range(6)])
    verify(ops, x, torch.rand(6, generator=g, device="cuda"), top_p=torch.tensor([0.05, 0.3, 0.501, 0.77, 0.96, 0.9991], device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [30011, 200000])
def test_min_p_above_and_below_the_cut(ops, dtype, vocab):
    """Both filters with weight in them, min-p from far above the top-p's cut to far below it."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x, u = scores(10, vocab, dtype, g, 1.5), torch.rand(10, generator=g, device="cuda")
    least = torch.logspace(-4, -0.3, 10, device="cuda")
    k = torch.randint(2000, vocab, (10,), generator=g, device="cuda", dtype=torch.int32)
    for p in (0.2, 0.6, 0.95):
        verify(ops, x, u, top_p=torch.full((10,), p, device="cuda"), min_p=least)
        verify(ops, x, u, top_k=k, top_p=torch.full((10,), p, device="cuda"), min_p=least)
        verify(ops, x, u, top_k=torch.full_like(k, 700), top_p=torch.full((10,), p, device="cuda"), min_p=least)
