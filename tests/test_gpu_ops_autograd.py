"""GPU: what the operators say to autograd: a tensor that carries a derivative is refused, one that is written is marked as written."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lk):
    from loki_b200 import ops
    return ops


def calls(ops):
    """name -> (function of one floating tensor, that tensor)"""
    x, gain, u = torch.randn(4, 64, device="cuda"), torch.rand(64, device="cuda"), torch.rand(4, device="cuda")
    h, w = x.half(), torch.randn(8, 64, device="cuda").half()
    codes = torch.ones(4, 64, dtype=torch.int8, device="cuda")
    table = torch.ones(8, 64, dtype=torch.int8, device="cuda")
    return {
        "x": (lambda t: ops.rms_norm_i8(t, gain), x), "gain": (lambda t: ops.rms_norm_i8(x, t), gain),
        "norm residual": (lambda t: ops.rms_norm_i8(x, gain, residual=t), x),
        "a": (lambda t: ops.linear(t, w), h), "w": (lambda t: ops.linear(h, t), w),
        "a_scales": (lambda t: ops.linear(codes, table, a_scales=t), u), "bias": (lambda t: ops.linear(h, w, bias=t), w[:, 0].contiguous()),
        "residual": (lambda t: ops.linear(h, w, residual=t), torch.ones(4, 8, device="cuda").half()),
        "scores": (lambda t: ops.sample(t, u), x), "u": (lambda t: ops.sample(x, t), u), "temperature": (lambda t: ops.sample(x, u, temperature=t), u),
        "top_p": (lambda t: ops.sample(x, u, top_p=t), u), "min_p": (lambda t: ops.sample(x, u, min_p=t), u),
    }


NAMES = ["x", "gain", "norm residual", "a", "w", "a_scales", "bias", "residual", "scores", "u", "temperature", "top_p", "min_p"]


@pytest.mark.parametrize("name", NAMES)
def test_dual_tensors_are_refused(ops, lk, name):
    call, t = calls(ops)[name]
    with fwd.dual_level():
        with pytest.raises(lk.LokiError, match="derivative"):
            call(fwd.make_dual(t, torch.ones_like(t)))
        call(t)  # one without a tangent is an ordinary tensor
    call(t)


@pytest.mark.parametrize("name", NAMES)
def test_transformed_tensors_are_refused(ops, lk, name):
    call, t = calls(ops)[name]
    first = lambda v: call(v)[0]
    with pytest.raises((lk.LokiError, RuntimeError)):
        torch.func.jvp(first, (t,), (torch.ones_like(t),))
    with pytest.raises((lk.LokiError, RuntimeError)):
        torch.func.vmap(first)(t.expand(2, *t.shape))
    with pytest.raises((lk.LokiError, RuntimeError)):
        torch.func.grad(lambda v: first(v).float().sum())(t)


def test_results_in_given_tensors_are_writes(ops):
    x, u = torch.randn(4, 64, device="cuda"), torch.rand(4, device="cuda")
    h, w = x.half(), torch.randn(8, 64, device="cuda").half()
    outs = {
        "out": (lambda t: ops.linear(h, w, out=t), torch.zeros(4, 8, device="cuda").half()),
        "out_sum": (lambda t: ops.rms_norm_i8(x, residual=x, out_sum=t), torch.zeros(4, 64, device="cuda")),
        "in place": (lambda t: ops.rms_norm_i8(x, residual=t, out_sum=t), torch.zeros(4, 64, device="cuda")),
        "out_codes": (lambda t: ops.rms_norm_i8(x, out_codes=t), torch.zeros(4, 64, dtype=torch.int8, device="cuda")),
        "out_scales": (lambda t: ops.rms_norm_i8(x, out_scales=t), torch.zeros(4, device="cuda")),
        "out_ids": (lambda t: ops.sample(x, u, out_ids=t), torch.zeros(4, dtype=torch.int64, device="cuda")),
    }
    for name, (call, t) in outs.items():
        before = t._version
        call(t)
        assert t._version > before, name
        with torch.inference_mode():  # tensors that keep no count
            call(t.clone())
    leaf = torch.ones(4, 8, device="cuda", requires_grad=True)
    saved = torch.zeros(4, 8, device="cuda")
    y = (leaf * saved).sum()
    ops.linear(h, w, out=saved, out_dtype=torch.float32)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
