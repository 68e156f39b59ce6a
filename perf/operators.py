"""Cases of the operators that take a model's hidden states to an answer: the root-mean-square norm
with an 8-bit output, the matrix product with its epilogue, and sampling from given random numbers.

`run` computes an operator in plain torch operations, or, where `own` is set, by the calls that a
user's program makes of `loki_b200.ops`.  `exact` gives the values of the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
_ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
_EPS = 1e-6


def _norm(name, rows, dim, dtype, residual):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "residual": residual}


def _linear(name, m, n, k, dtype, out, act, bias, residual):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "out": out, "act": act, "bias": bias, "residual": residual}


def _sample(name, rows, vocab, dtype, mode):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "mode": mode}


def listed():
    return [
        # one token's hidden state on its way into a layer: latency
        _norm("norm_token", 1, 1024, "bf16", True),
        # the pooled states of a batch of an odd width, no residual
        _norm("norm_ragged", 1000, 771, "f32", False),
        # the prompts of a batch, 8,192 tokens
        _norm("norm_prefill", 8192, 4096, "bf16", True),
        # one token through a layer's output projection: the weights are read once
        _linear("linear_token", 1, 4096, 4096, "i8", "bf16", "none", False, True),
        # a batch of single tokens through an expanding layer
        _linear("linear_batch", 48, 8192, 1024, "bf16", "bf16", "gelu", True, False),
        # eight hidden states against a table of 131,072 rows: the scores of an answer
        _linear("linear_scores", 8, 131072, 1024, "i8", "f32", "none", False, False),
        # odd sizes in every direction
        _linear("linear_ragged", 333, 1000, 771, "f16", "f16", "silu", True, True),
        # prompts through an expanding layer, 8-bit operands
        _linear("linear_expand", 4096, 8192, 4096, "i8", "bf16", "gelu_tanh", True, False),
        # prompts through a layer's output projection, 16-bit operands
        _linear("linear_project", 8192, 4096, 4096, "bf16", "bf16", "none", True, True),
        # one answer, the usual filters: latency
        _sample("sample_token", 1, 32768, "f32", "usual"),
        # a batch of answers, each with settings of its own
        _sample("sample_batch", 64, 131072, "bf16", "mixed"),
        # draws among the scores of a million rows, by nucleus alone
        _sample("sample_million", 8, 1000000, "f32", "nucleus"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "linear", "linear", "sample"))
    if op == "norm":
        dim = _spread(rng, 64, 8192)
        rows = _spread(rng, 1, max(1, min(8192, 8192 * 4096 // dim)))
        return {"op": op, "rows": rows, "dim": dim, "dtype": rng.choice(("f32", "f16", "bf16")) if rows * dim < 1 << 24 else "bf16",
                "residual": rng.random() < 0.6}
    if op == "linear":
        k = _spread(rng, 64, 8192)
        n = _spread(rng, 16, min(131072, 131072 * 1024 // k))
        m = _spread(rng, 1, max(1, min(8192, (8192 * 8192) // (2 * n), (8192 * 4096 * 4096) // (n * k))))
        return {"op": op, "m": m, "n": n, "k": k, "dtype": rng.choice(("i8", "i8", "f16", "bf16")), "out": rng.choice(("f32", "f16", "bf16")),
                "act": rng.choice(_ACTS), "bias": rng.random() < 0.6, "residual": rng.random() < 0.5}
    vocab = _spread(rng, 16, 1000000)
    rows = _spread(rng, 1, max(1, min(256, 8000000 // vocab)))
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(("f32", "f16", "bf16")), "mode": rng.choice(("usual", "mixed", "nucleus", "free"))}


def _padded(values):
    """The same values in rows that start on 16-byte boundaries, as a table of rows is kept."""
    step = 16 // values.element_size()
    wide = torch.zeros((values.shape[0], -(-values.shape[1] // step) * step), dtype=values.dtype, device=values.device)
    wide[:, : values.shape[1]] = values
    return wide[:, : values.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *size: torch.rand(size, generator=g, device="cuda")  # noqa: E731
    randn = lambda *size: torch.randn(size, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "norm":
        rows, dim, t = case["rows"], case["dim"], _T[case["dtype"]]
        wide = 0.3 + 1.5 * rand(dim) ** 4  # a few columns carry more than the others, as in hidden states
        return {"op": "norm", "x": (randn(rows, dim) * wide).to(t), "gain": (0.5 + rand(dim)).to(t),
                "residual": (randn(rows, dim) * wide * 2).to(t) if case["residual"] else None}
    if case["op"] == "linear":
        m, n, k, t, o = case["m"], case["n"], case["k"], _T[case["dtype"]], _T[case["out"]]
        s = {"op": "linear", "act": case["act"], "out": o, "a_scales": None, "w_scales": None}
        if case["dtype"] == "i8":
            s["a"] = _padded((randn(m, k) * 32).round_().clamp_(-127, 127).to(t))
            s["w"] = _padded((randn(n, k) * 32).round_().clamp_(-127, 127).to(t))
            s["a_scales"] = (0.5 + rand(m)) / 32
            s["w_scales"] = (0.5 + rand(n)) / (32 * math.sqrt(k))
        else:
            s["a"] = _padded(randn(m, k).to(t))
            s["w"] = _padded((randn(n, k) / math.sqrt(k)).to(t))
        s["bias"] = (randn(n) * 0.5).to(o) if case["bias"] else None
        s["residual"] = randn(m, n).to(o) if case["residual"] else None
        return s
    rows, vocab = case["rows"], case["vocab"]
    s = {"op": "sample", "logits": (randn(rows, vocab) * 2.5).to(_T[case["dtype"]]), "u": rand(rows),
         "temperature": None, "top_k": None, "top_p": None, "min_p": None}
    if case["mode"] in ("usual", "mixed"):
        s["temperature"] = 0.5 + rand(rows)
        s["top_k"] = torch.randint(1, 200, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["top_p"] = 0.6 + 0.4 * rand(rows)
    if case["mode"] == "mixed":  # every row its own filters, some none, some the largest logit
        kind = torch.randint(0, 6, (rows,), generator=g, device="cuda")
        s["temperature"] = torch.where(kind == 0, 0.0, s["temperature"])
        s["top_k"] = torch.where(kind >= 3, 0, s["top_k"]).to(torch.int32)
        s["top_p"] = torch.where(kind == 4, 1.0, s["top_p"])
        s["min_p"] = torch.where(kind == 5, 0.02 + 0.1 * rand(rows), 0.0)
        s["logits"] = torch.where(rand(rows, vocab) < 0.01, float("-inf"), s["logits"])  # masked entries
    if case["mode"] == "nucleus":
        s["top_p"] = 0.8 + 0.19 * rand(rows)
    return s


def run(s):
    if own:
        return _own(s)
    if s["op"] == "norm":
        return _plain_norm(s["x"], s["gain"], s["residual"])
    if s["op"] == "linear":
        return _plain_linear(s)
    return _plain_sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def _own(s):
    from loki_b200 import ops
    if s["op"] == "norm":
        codes, scales, total = ops.rms_norm_i8(s["x"], s["gain"], residual=s["residual"], eps=_EPS)
        values = torch.mul(codes, scales[:, None], out=torch.empty(codes.shape, dtype=torch.bfloat16, device=codes.device))
        return {"values": values, "scales": scales, "sum": total}
    if s["op"] == "linear":
        return ops.linear(s["a"], s["w"], a_scales=s["a_scales"], w_scales=s["w_scales"], bias=s["bias"], act=s["act"],
                          residual=s["residual"], out_dtype=s["out"])
    ids, probs, kept = ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    return {"ids": ids, "probs": probs, "kept": kept}


def _plain_norm(x, gain, residual):
    h = x.float() if residual is None else x.float() + residual.float()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS) * gain.float()
    scales = y.abs().amax(1) / 127
    codes = torch.round(y / torch.where(scales == 0, 1.0, scales)[:, None]).clamp(-127, 127)
    return {"values": (codes * scales[:, None]).to(torch.bfloat16), "scales": scales, "sum": None if residual is None else h.to(x.dtype)}


def _activation(v, act):
    if act == "relu":
        return torch.clamp_min(v, 0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain_linear(s):
    v = s["a"].float() @ s["w"].float().t()
    if s["a_scales"] is not None:
        v = v * (s["a_scales"][:, None] * s["w_scales"])
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _activation(v, s["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(s["out"])


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    """In 64 bits: the sums are long, and a draw or a cut may fall next to a border."""
    rows, vocab = logits.shape
    x = logits.double()
    x = torch.where(torch.isnan(x), float("-inf"), x)
    t = torch.ones_like(u, dtype=torch.float64) if temperature is None else temperature.double()
    k = torch.zeros_like(u, dtype=torch.int64) if top_k is None else top_k.long()
    p = torch.ones_like(t) if top_p is None else top_p.double()
    least = torch.zeros_like(t) if min_p is None else min_p.double()
    k = torch.where(t == 0, 1, k)
    t = torch.where(t == 0, 1.0, t)
    ranked, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = ranked[:, :1]
    w = torch.where(ranked == top, 1.0, torch.exp((ranked - top) / t[:, None]))
    valid = ranked > float("-inf")
    place = torch.arange(vocab, device=x.device)
    kept = valid & ((place < k[:, None]) | (k[:, None] <= 0))
    w = torch.where(kept, w, 0.0)
    running = torch.cumsum(w, 1)
    before = torch.cat([torch.zeros_like(top), running[:, :-1]], 1)
    kept = kept & ((before < p[:, None] * running[:, -1:]) | (p[:, None] >= 1)) & (w >= least[:, None]) | valid & (place == 0)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))  # back in the order of the indexes
    running = torch.cumsum(w, 1)
    total = running[:, -1:]
    count = kept.sum(1)
    ids = (running <= u.double()[:, None] * total).sum(1, keepdim=True).clamp_max(vocab - 1)
    probs = torch.gather(w, 1, ids) / total
    return {"ids": torch.where(count == 0, -1, ids[:, 0]), "probs": torch.where(count == 0, 0.0, probs[:, 0]).float(), "kept": count.to(torch.int32)}


def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["dim"], _BYTES[case["dtype"]]
        return {"bytes": n * (b * (3 if case["residual"] else 1) + 1) + case["dim"] * b + 4 * case["rows"], "flops": 8 * n}
    if case["op"] == "linear":
        m, n, k, b, o = case["m"], case["n"], case["k"], _BYTES[case["dtype"]], _BYTES[case["out"]]
        return {"bytes": (m + n) * (k * b + (4 if case["dtype"] == "i8" else 0)) + m * n * o * (2 if case["residual"] else 1) + (n * o if case["bias"] else 0),
                "flops": 2 * m * n * k}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * _BYTES[case["dtype"]] + case["rows"] * 32, "flops": 2 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (0 if s["residual"] is None else s["residual"].double())
        y = h * s["gain"].double() * (h.square().sum(1) / case["dim"] + _EPS).rsqrt()[:, None]
        step = torch.linalg.vector_norm(y, math.inf, 1) / 127
        codes = torch.where(step[:, None] > 0, (y / step[:, None]).round(), 0.0)
        return {"values": codes * step[:, None], "scales": step, "sum": None if s["residual"] is None else h}
    if case["op"] == "linear":
        v = torch.mm(s["a"].double(), s["w"].double().t())
        if s["a_scales"] is not None:
            v *= torch.outer(s["a_scales"].double(), s["w_scales"].double())
        if s["bias"] is not None:
            v += s["bias"].double()
        if case["act"] == "relu":
            v = v * (v > 0)
        elif case["act"] == "silu":
            v = v * torch.sigmoid(v)
        elif case["act"] == "gelu":
            v = v * torch.special.ndtr(v)
        elif case["act"] == "gelu_tanh":  # (1 + tanh z) / 2 = sigmoid(2 z)
            v = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))
        return v if s["residual"] is None else v + s["residual"].double()
    ids, probs, kept = [], [], []
    host = {n: None if s[n] is None else s[n].double().cpu().numpy() for n in ("logits", "u", "temperature", "top_k", "top_p", "min_p")}
    for r, x in enumerate(host["logits"]):
        t, k, p, least = (d if host[n] is None else host[n][r] for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
        there = np.flatnonzero(x > -np.inf)
        there = there[np.lexsort((there, -x[there]))]
        if t == 0:
            there, t = there[:1], 1.0
        if k > 0:
            there = there[: int(k)]
        if there.size == 0:
            ids, probs, kept = ids + [-1], probs + [0.0], kept + [0]
            continue
        w = np.exp((x[there] - x[there[0]]) / t)
        if p < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), p * w.sum()))
            there, w = there[:n], w[:n]
        n = max(1, int((w >= least).sum()))
        there, w = there[:n], w[:n]
        by_index = np.argsort(there)
        there, w = there[by_index], w[by_index]
        at = min(int(np.searchsorted(np.cumsum(w), host["u"][r] * w.sum(), side="right")), n - 1)
        ids, probs, kept = ids + [int(there[at])], probs + [w[at] / w.sum()], kept + [n]
    return {"ids": torch.tensor(ids), "probs": torch.tensor(probs, dtype=torch.float64), "kept": torch.tensor(kept, dtype=torch.int32)}
