"""Operators on CUDA tensors, from a model's hidden states to rows and answers.

* :func:`rms_norm_i8`  root-mean-square norm (+ residual) to int8 codes with one scale per row
* :func:`linear`       product of rows with rows, with scales, bias, activation and residual
* :func:`sample`       one draw per row of scores: temperature, top-k, top-p, min-p

They are the functions ``lk_rms_norm_i8``, ``lk_linear`` and ``lk_sample`` of ``include/lokiscan.h``,
which states the formulas; here the arguments are PyTorch tensors.  A call runs on the device of its
first tensor, on PyTorch's current stream of that device, returns without waiting and can be captured
into a CUDA graph.  Tensors are two-dimensional with contiguous rows (``stride(1) == 1``) at any row
stride; vectors are contiguous.  There is no gradient: a tensor that requires one is refused.

    codes, scales, hidden = ops.rms_norm_i8(x, gain, residual=hidden)
    scores = ops.linear(codes, table, a_scales=scales, w_scales=table_scales, out_dtype=torch.float32)
    ids, probs, kept = ops.sample(scores, u, temperature=0.8, top_p=0.9)
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import LK_EDIM, LK_EINVAL, LokiError, check, lib

_FLOATS = {torch.float32: _lib.LK_F32, torch.float16: _lib.LK_F16, torch.bfloat16: _lib.LK_BF16}
_OPERANDS = {torch.int8: _lib.LK_I8, torch.float16: _lib.LK_F16, torch.bfloat16: _lib.LK_BF16}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _refuse(status, message):
    raise LokiError(status, message)


def _ready(t, what, types, device=None, dims=2):
    """A tensor that the kernels can read: its type, its device, contiguous rows, no gradient."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(LK_EINVAL, f"{what}: a CUDA tensor is wanted (this library has no CPU path)")
    if t.dtype not in types:
        _refuse(LK_EINVAL, f"{what}: {t.dtype} is not supported here")
    if t.dim() != dims:
        _refuse(LK_EDIM, f"{what}: {dims} dimension(s) are wanted, not {t.dim()}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _refuse(LK_EINVAL, f"{what}: its rows are not contiguous")
    if dims == 2 and t.shape[0] > 1 and t.shape[1] > 0 and t.stride(0) < t.shape[1]:
        _refuse(LK_EINVAL, f"{what}: its rows overlap")
    if device is not None and t.device != device:
        _refuse(LK_EINVAL, f"{what}: it is on {t.device}, not on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(LK_EINVAL, f"{what}: it requires a gradient, which this operator does not have")
    return t


def _shaped(t, what, types, device, *shape):
    _ready(t, what, types, device, len(shape))
    if tuple(t.shape) != shape:
        _refuse(LK_EDIM, f"{what}: shape {tuple(t.shape)} where {shape} is wanted")
    return t


def _ld(t):
    """Elements between the starts of two rows; a single row's stride says nothing."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _p(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _codes(rows, dim, device):
    """rows x dim int8 in rows of a multiple of 16 bytes, the padding zero: as linear reads them best."""
    wide = (dim + 15) // 16 * 16
    if wide == dim:
        return torch.empty((rows, dim), dtype=torch.int8, device=device)
    return torch.zeros((rows, wide), dtype=torch.int8, device=device)[:, :dim]


def rms_norm_i8(x, gain=None, *, residual=None, eps: float = 1e-6, out_codes=None, out_scales=None, out_sum=None):
    """Norm of ``x (+ residual)`` in 8 bits: -> (codes [rows, dim] int8, scales [rows] float32, sum).

    ``codes * scales[:, None]`` is ``h / sqrt(mean(h ** 2) + eps) * gain`` with ``h = x + residual``,
    rounded to 8 bits; ``sum`` is ``h`` in the type of ``x`` (None without a residual).  ``gain`` is a
    vector of any of the three floating types.  ``out_sum`` may be ``x`` or ``residual`` itself.
    """
    _ready(x, "x", _FLOATS)
    rows, dim = x.shape
    dev, t = x.device, (x.dtype,)
    if gain is not None:
        _shaped(gain, "gain", _FLOATS, dev, dim)
    if residual is not None:
        _shaped(residual, "residual", t, dev, rows, dim)
    if out_sum is not None:
        _shaped(out_sum, "out_sum", t, dev, rows, dim)
    elif residual is not None:
        out_sum = torch.empty((rows, dim), dtype=x.dtype, device=dev)
    out_codes = _codes(rows, dim, dev) if out_codes is None else _shaped(out_codes, "out_codes", (torch.int8,), dev, rows, dim)
    out_scales = torch.empty(rows, dtype=torch.float32, device=dev) if out_scales is None else _shaped(out_scales, "out_scales", (torch.float32,), dev, rows)
    st = lib.lk_rms_norm_i8(dev.index, _FLOATS[x.dtype], rows, dim, x.data_ptr(), _ld(x),
                            _p(residual), 0 if residual is None else _ld(residual),
                            _p(gain), 0 if gain is None else _FLOATS[gain.dtype], eps,
                            _p(out_sum), 0 if out_sum is None else _ld(out_sum),
                            out_codes.data_ptr(), _ld(out_codes), out_scales.data_ptr(), _stream(dev))
    if st:
        check(st)
    return out_codes, out_scales, out_sum


def linear(a, w, *, a_scales=None, w_scales=None, bias=None, act: str = "none", residual=None, out_dtype=None, out=None):
    """``act(a @ w.T * a_scales[:, None] * w_scales + bias) + residual``: -> [m, n] of ``out_dtype``.

    ``a`` [m, k] and ``w`` [n, k] are both int8 (exact int32 sums; scales are float32 vectors), both
    float16 or both bfloat16 (float32 sums).  ``bias`` [n] and ``residual`` [m, n] have the type of the
    result: that of ``out``, else ``out_dtype``, else that of ``residual`` or ``bias``, else ``a``'s
    (float32 for int8).  ``out`` may be ``residual`` itself.  Rows on 16-byte boundaries run fastest.
    """
    _ready(a, "a", _OPERANDS)
    m, k = a.shape
    dev = a.device
    _ready(w, "w", (a.dtype,), dev)
    n = w.shape[0]
    if w.shape[1] != k:
        _refuse(LK_EDIM, f"w: rows of {w.shape[1]} elements, those of a have {k}")
    if act not in ACTIVATIONS:
        _refuse(LK_EINVAL, f"act: one of {', '.join(ACTIVATIONS)}, not {act!r}")
    if a_scales is not None:
        _shaped(a_scales, "a_scales", (torch.float32,), dev, m)
    if w_scales is not None:
        _shaped(w_scales, "w_scales", (torch.float32,), dev, n)
    if out is not None:
        kind = out.dtype
        if out_dtype is not None and out_dtype != kind:
            _refuse(LK_EINVAL, f"out: {kind}, but out_dtype is {out_dtype}")
    elif out_dtype is not None:
        kind = out_dtype
    elif residual is not None:
        kind = residual.dtype
    elif bias is not None:
        kind = bias.dtype
    else:
        kind = torch.float32 if a.dtype == torch.int8 else a.dtype
    if kind not in _FLOATS:
        _refuse(LK_EINVAL, f"out_dtype: {kind} is not supported here")
    if bias is not None:
        _shaped(bias, "bias", (kind,), dev, n)
    if residual is not None:
        _shaped(residual, "residual", (kind,), dev, m, n)
    out = torch.empty((m, n), dtype=kind, device=dev) if out is None else _shaped(out, "out", (kind,), dev, m, n)
    st = lib.lk_linear(dev.index, _OPERANDS[a.dtype], m, n, k, a.data_ptr(), _ld(a), _p(a_scales), w.data_ptr(), _ld(w), _p(w_scales),
                       _p(bias), ACTIVATIONS[act], _p(residual), 0 if residual is None else _ld(residual),
                       _FLOATS[kind], out.data_ptr(), _ld(out), _stream(dev))
    if st:
        check(st)
    return out


def check_device(device=0):
    """Wait for the device; raise if a bounded wait inside one of these kernels ran out since the last call."""
    index = torch.device("cuda", device).index if isinstance(device, int) else torch.device(device).index
    check(lib.lk_ops_status(index))


def _per_row(v, what, dtype, rows, device):
    """One value per row: a vector, or a number for all rows."""
    if v is None or isinstance(v, torch.Tensor):
        return v if v is None else _shaped(v, what, (dtype,), device, rows)
    return torch.full((rows,), v, dtype=dtype, device=device)


def sample(scores, u, *, temperature=None, top_k=None, top_p=None, min_p=None, out_ids=None):
    """One draw per row of ``scores`` [rows, vocab] from the random numbers ``u`` [rows] in [0, 1):
    -> (ids [rows] int64, probs [rows] float32, kept [rows] int32).

    ``temperature``, ``top_p``, ``min_p`` (float32) and ``top_k`` (int32) are vectors of one value per row, or
    numbers for all rows; None switches a filter off.  ``probs`` is the probability of the draw among the
    ``kept`` entries.  A row with nothing to draw (only NaN and -inf) gets id -1.
    """
    _ready(scores, "scores", _FLOATS)
    rows, vocab = scores.shape
    dev, f = scores.device, torch.float32
    _shaped(u, "u", (f,), dev, rows)
    temperature = _per_row(temperature, "temperature", f, rows, dev)
    top_k = _per_row(top_k, "top_k", torch.int32, rows, dev)
    top_p = _per_row(top_p, "top_p", f, rows, dev)
    min_p = _per_row(min_p, "min_p", f, rows, dev)
    ids = torch.empty(rows, dtype=torch.int64, device=dev) if out_ids is None else _shaped(out_ids, "out_ids", (torch.int64,), dev, rows)
    probs = torch.empty(rows, dtype=f, device=dev)
    kept = torch.empty(rows, dtype=torch.int32, device=dev)
    st = lib.lk_sample(dev.index, _FLOATS[scores.dtype], rows, vocab, scores.data_ptr(), _ld(scores), _p(temperature), _p(top_k),
                       _p(top_p), _p(min_p), u.data_ptr(), ids.data_ptr(), probs.data_ptr(), kept.data_ptr(), _stream(dev))
    if st:
        check(st)
    return ids, probs, kept
