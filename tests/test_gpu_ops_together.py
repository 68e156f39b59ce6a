"""GPU: the operators one after the other, as an answer is made, on streams and in graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def setting(rows=6, dim=768, vocab=5000, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda")
    from loki_b200 import ops
    table, table_scales, _ = ops.rms_norm_i8(randn(vocab, dim), eps=0.0)
    return dict(x=randn(rows, dim).bfloat16(), hidden=randn(rows, dim).bfloat16(), gain=(1 + 0.1 * randn(dim)).bfloat16(),
                up=(randn(2 * dim, dim) / 28).bfloat16(), down=(randn(dim, 2 * dim) / 40).bfloat16(), bias=randn(2 * dim).bfloat16(),
                table=table, table_scales=table_scales * (4.0 / dim), u=torch.rand(rows, generator=g, device="cuda"))


def answer(ops, s):
    """A layer's residual branch in 16 bits, the norm to 8 bits, the scores of a table's rows, a draw."""
    branch = ops.linear(s["x"], s["up"], bias=s["bias"], act="silu")
    hidden = ops.linear(branch, s["down"], residual=s["hidden"])
    codes, scales, total = ops.rms_norm_i8(s["x"], s["gain"], residual=hidden)
    scores = ops.linear(codes, s["table"], a_scales=scales, w_scales=s["table_scales"])
    return (hidden, codes, scales, total, scores) + ops.sample(scores, s["u"], temperature=0.9, top_k=200, top_p=0.95)


def test_an_answer(ops):
    s = setting()
    hidden, codes, scales, total, scores, ids, probs, kept = answer(ops, s)
    f = lambda t: t.double()
    b = f(s["x"]) @ f(s["up"]).t() + f(s["bias"])
    b = f((b * torch.sigmoid(b)).bfloat16())
    want_hidden = b @ f(s["down"]).t() + f(s["hidden"])
    # every element of the branch may round to either neighbour, half a bf16 step (2^-8 of its size): the sum is off by at most
    # the sum of those, and is rounded to bf16 itself
    slack = (b.abs() @ f(s["down"]).abs().t()) * 2.0 ** -7 + want_hidden.abs() * 2.0 ** -8 + 1e-5
    assert torch.all((f(hidden) - want_hidden).abs() <= slack)
    h = s["x"].float() + hidden.float()
    assert torch.equal(total, h.bfloat16())
    y = f(h) * f(s["gain"]) / torch.sqrt(f(h).square().mean(1, keepdim=True) + 1e-6)
    assert torch.all((f(codes) * f(scales)[:, None] - y).abs() <= f(scales)[:, None] * 0.5001)
    want_scores = (f(codes) @ f(s["table"]).t()) * f(scales)[:, None] * f(s["table_scales"])
    assert torch.all((f(scores) - want_scores).abs() <= want_scores.abs() * 4 * 2.0 ** -24)
    # the draw, by the definition, from the scores as they are
    setting_of = lambda v: f(torch.tensor(v, dtype=torch.float32))  # the number as the kernel gets it
    p = f(scores) / setting_of(0.9).cuda()
    for r in range(len(ids)):
        v, order = torch.sort(p[r], descending=True, stable=True)
        w = torch.exp(v - v[0])[:200]
        run = torch.cumsum(w, 0)
        n = int((run - w < setting_of(0.95).cuda() * run[-1]).sum())
        assert kept[r] == n
        mask = torch.zeros_like(p[r])
        mask[order[:n]] = w[:n]
        run = torch.cumsum(mask, 0)
        at = int((run <= f(s["u"])[r] * run[-1]).sum())
        assert ids[r] == at
        assert abs(float(probs[r]) - float(mask[at] / run[-1])) <= 2.0 ** -22 * float(probs[r])


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_same_twice_and_on_other_streams(ops):
    sets = [setting(rows=r, seed=r) for r in (1, 9, 40, 200)]
    want = [answer(ops, s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):  # all at once, again and again
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(answer(ops, s))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert same(w, g)


def test_captured_and_replayed(ops):
    s, t = setting(rows=5, seed=3), setting(rows=150, seed=4)
    want = answer(ops, s), answer(ops, t)
    graphs = []
    for v in (s, t):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = answer(ops, v)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):  # both graphs at the same time
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    assert same(graphs[0][1], want[0]) and same(graphs[1][1], want[1])
    # new inputs through the old graph
    other = setting(rows=5, seed=5)
    for name in ("x", "hidden", "u"):
        s[name].copy_(other[name])
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert same(graphs[0][1], answer(ops, s))


def test_no_allocation_by_the_calls(ops, lk):
    """With their outputs given, the calls leave the device's free memory alone."""
    s = setting()
    answer(ops, s)
    out = [torch.empty(6, 768, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda"), torch.empty(6, 768, dtype=torch.bfloat16, device="cuda"),
           torch.empty(6, 5000, device="cuda")]
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(3):
        ops.rms_norm_i8(s["x"], s["gain"], residual=s["hidden"], out_codes=out[0], out_scales=out[1], out_sum=out[2])
        ops.linear(out[0], s["table"], a_scales=out[1], w_scales=s["table_scales"], out=out[3])
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == before


def test_first_calls_of_new_sizes_in_a_capture(ops):
    """Once a function has run on the device, any of its kernels may be met in a capture first."""
    s = setting(rows=3, seed=8)
    answer(ops, s)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(700, 2048, generator=g, device="cuda").half()
    w = torch.randn(2100, 2048, generator=g, device="cuda").half()
    u = torch.rand(700, generator=g, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, scales, _ = ops.rms_norm_i8(x)
        y = ops.linear(x, w, act="gelu")
        ids, _, _ = ops.sample(y, u, top_p=0.9)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(codes, ops.rms_norm_i8(x)[0]) and torch.equal(y, ops.linear(x, w, act="gelu"))
    assert torch.equal(ids, ops.sample(y, u, top_p=0.9)[0])


def test_status_sees_side_streams(ops):
    s = setting(rows=200, seed=2)
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(20):
            out = answer(ops, s)
    ops.check_device()  # waits for that stream too
    assert same(out, answer(ops, s))
