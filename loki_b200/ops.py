"""Operators on CUDA tensors, from a model's hidden states to rows and answers.

* :func:`rms_norm_i8`  root-mean-square norm (+ residual) to int8 codes with one scale per row
* :func:`linear`       product of rows with rows, with scales, bias, activation and residual
* :func:`sample`       one draw per row of scores: temperature, top-k, top-p, min-p

They are the functions ``lk_rms_norm_i8``, ``lk_linear`` and ``lk_sample`` of ``include/lokiscan.h``,
which states the formulas; here the arguments are PyTorch tensors.  A call runs on the device of its
first tensor, on PyTorch's current stream of that device, returns without waiting and can be captured
into a CUDA graph.  Tensors are two-dimensional with contiguous rows (``stride(1) == 1``) at any row
stride; vectors are contiguous.  There is no gradient: a tensor that requires one, or carries a
forward-mode derivative, is refused.

    codes, scales, hidden = ops.rms_norm_i8(x, gain, residual=hidden)
    scores = ops.linear(codes, table, a_scales=scales, w_scales=table_scales, out_dtype=torch.float32)
    ids, probs, kept = ops.sample(scores, u, temperature=0.8, top_p=0.9)
"""
from __future__ import annotations

import math
import numbers

import torch
import torch.autograd.forward_ad as _forward

from . import _lib
from ._lib import LK_EDIM, LK_EINVAL, LK_ERANGE, LokiError, check, lib

_FLOATS = {torch.float32: _lib.LK_F32, torch.float16: _lib.LK_F16, torch.bfloat16: _lib.LK_BF16}
_OPERANDS = {torch.int8: _lib.LK_I8, torch.float16: _lib.LK_F16, torch.bfloat16: _lib.LK_BF16}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _refuse(status, message):
    raise LokiError(status, message)


def _why(t, what, types, index, *shape):
    """The refusal of a tensor that :func:`_matrix` or :func:`_vector` found wrong."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(LK_EINVAL, f"{what}: a CUDA tensor is wanted (this library has no CPU path)")
    if t.dtype not in types:
        _refuse(LK_EINVAL, f"{what}: {t.dtype} is not supported here")
    if t.dim() != len(shape):
        _refuse(LK_EDIM, f"{what}: {len(shape)} dimension(s) are wanted, not {t.dim()}")
    if index is not None and t.get_device() != index:
        _refuse(LK_EINVAL, f"{what}: it is on {t.device}, not on cuda:{index}")
    if any(want is not None and have != want for have, want in zip(t.shape, shape)):
        _refuse(LK_EDIM, f"{what}: shape {tuple(t.shape)} where {shape} is wanted")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _refuse(LK_EINVAL, f"{what}: its rows are not contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(LK_EINVAL, f"{what}: it requires a gradient, which this operator does not have")
    if _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None:
        _refuse(LK_EINVAL, f"{what}: it carries a forward-mode derivative, which this operator does not have")
    _refuse(LK_EINVAL, f"{what}: its rows overlap")


# The two checks below run on every call: they ask a tensor for as little as possible.

def _matrix(t, what, types, index=None, rows=None, cols=None):
    """(rows, cols, elements between rows, device) of a matrix that the kernels can read."""
    try:
        on = t.get_device()
        (r, c), (ld, one) = t.shape, t.stride()
    except (AttributeError, ValueError):
        _why(t, what, types, index, rows, cols)
    if (on < 0 or t.dtype not in types or (one != 1 and c > 1) or (index is not None and on != index) or (rows is not None and r != rows)
            or (cols is not None and c != cols) or (ld < c and r > 1) or (t.requires_grad and torch.is_grad_enabled())
            or (_forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None)):
        _why(t, what, types, index, rows, cols)
    return r, c, ld if r > 1 else max(ld, c), on  # a single row's stride says nothing


def _vector(t, what, types, index, n):
    """The address of a contiguous vector of n values; None for None."""
    if t is None:
        return None
    try:
        if (t.get_device() != index or t.dtype not in types or t.shape != (n,) or (n > 1 and t.stride() != (1,))
                or (t.requires_grad and torch.is_grad_enabled())
                or (_forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None)):
            _why(t, what, types, index, n)
    except AttributeError:
        _why(t, what, types, index, n)
    return t.data_ptr()


_stream = torch._C._cuda_getCurrentRawStream
_norm, _linear, _sample = lib.lk_rms_norm_i8, lib.lk_linear, lib.lk_sample
_F32_MAX = torch.finfo(torch.float32).max
_F32, _I32, _I64, _I8 = (torch.float32,), (torch.int32,), (torch.int64,), (torch.int8,)


_new = torch.empty_strided
_written = torch.autograd.graph.increment_version  # for tensors that the caller gives: autograd does not see the kernels' writes


def rms_norm_i8(x, gain=None, *, residual=None, eps: float = 1e-6, out_codes=None, out_scales=None, out_sum=None):
    """Norm of ``x (+ residual)`` in 8 bits: -> (codes [rows, dim] int8, scales [rows] float32, sum).

    ``codes * scales[:, None]`` is ``h / sqrt(mean(h ** 2) + eps) * gain`` with ``h = x + residual``,
    rounded to 8 bits; ``sum`` is ``h`` in the type of ``x`` (None without a residual).  ``gain`` is a
    vector of any of the three floating types.  ``out_sum`` may be ``x`` or ``residual`` itself.  Codes that
    are made here have rows on 16-byte boundaries, with whatever was there between them.
    """
    rows, dim, ldx, dev = _matrix(x, "x", _FLOATS)
    kind = x.dtype
    g = _vector(gain, "gain", _FLOATS, dev, dim)
    r = ldr = 0
    if residual is not None:
        ldr = _matrix(residual, "residual", (kind,), dev, rows, dim)[2]
        r = residual.data_ptr()
    place = x.device
    s = lds = 0
    given = ()
    if out_sum is not None:
        given = (out_sum,)
        lds = _matrix(out_sum, "out_sum", (kind,), dev, rows, dim)[2]
        s = out_sum.data_ptr()
    elif residual is not None:
        out_sum, lds = _new((rows, dim), (dim, 1), dtype=kind, device=place), dim
        s = out_sum.data_ptr()
    if out_codes is not None:
        given += (out_codes,)
        ldc = _matrix(out_codes, "out_codes", _I8, dev, rows, dim)[2]
    else:  # rows on 16-byte boundaries, as linear reads them best
        ldc = (dim + 15) // 16 * 16
        out_codes = _new((rows, dim), (ldc, 1), dtype=torch.int8, device=place)
    if out_scales is None:
        out_scales = _new((rows,), (1,), dtype=torch.float32, device=place)
        scales = out_scales.data_ptr()
    else:
        given += (out_scales,)
        scales = _vector(out_scales, "out_scales", _F32, dev, rows)
    st = _norm(dev, _FLOATS[kind], rows, dim, x.data_ptr(), ldx, r, ldr, g, 0 if g is None else _FLOATS[gain.dtype], eps,
                            s, lds, out_codes.data_ptr(), ldc, scales, _stream(dev))
    if st:
        check(st)
    if given:
        _written(given)
    return out_codes, out_scales, out_sum


def linear(a, w, *, a_scales=None, w_scales=None, bias=None, act: str = "none", residual=None, out_dtype=None, out=None):
    """``act(a @ w.T * a_scales[:, None] * w_scales + bias) + residual``: -> [m, n] of ``out_dtype``.

    ``a`` [m, k] and ``w`` [n, k] are both int8 (exact int32 sums; scales are float32 vectors), both
    float16 or both bfloat16 (float32 sums).  ``bias`` [n] and ``residual`` [m, n] have the type of the
    result: that of ``out``, else ``out_dtype``, else that of ``residual`` or ``bias``, else ``a``'s
    (float32 for int8).  ``out`` may be ``residual`` itself.  Rows on 16-byte boundaries run fastest.
    """
    m, k, lda, dev = _matrix(a, "a", _OPERANDS)
    operands = a.dtype
    n, _, ldw, _ = _matrix(w, "w", (operands,), dev, None, k)
    activation = ACTIVATIONS.get(act)
    if activation is None:
        _refuse(LK_EINVAL, f"act: one of {', '.join(ACTIVATIONS)}, not {act!r}")
    for t, what in ((out, "out"), (residual, "residual"), (bias, "bias")):
        if t is not None and not isinstance(t, torch.Tensor):
            _refuse(LK_EINVAL, f"{what}: a CUDA tensor is wanted")
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
        kind = torch.float32 if operands == torch.int8 else operands
    result = _FLOATS.get(kind)
    if result is None:
        _refuse(LK_EINVAL, f"out_dtype: {kind} is not supported here")
    r = ldr = 0
    if residual is not None:
        ldr = _matrix(residual, "residual", (kind,), dev, m, n)[2]
        r = residual.data_ptr()
    sa = None if a_scales is None else _vector(a_scales, "a_scales", _F32, dev, m)
    sw = None if w_scales is None else _vector(w_scales, "w_scales", _F32, dev, n)
    b = None if bias is None else _vector(bias, "bias", (kind,), dev, n)
    given = out is not None
    if not given:
        out, ldo = _new((m, n), (n, 1), dtype=kind, device=a.device), n
    else:
        ldo = _matrix(out, "out", (kind,), dev, m, n)[2]
    st = _linear(dev, _OPERANDS[operands], m, n, k, a.data_ptr(), lda, sa, w.data_ptr(), ldw, sw, b, activation, r, ldr,
                 result, out.data_ptr(), ldo, _stream(dev))
    if st:
        check(st)
    if given:
        _written(out)
    return out


def check_device(device=0):
    """Wait for the device (a number, a name or a ``torch.device``; the current one for ``"cuda"`` or None); raise if a
    bounded wait inside one of these kernels ran out since the last call."""
    index = device
    if not isinstance(device, int):
        named = torch.device("cuda" if device is None else device)
        if named.type != "cuda":
            _refuse(LK_EINVAL, f"device: a CUDA device is wanted, not {named}")
        index = named.index
        if index is None:
            index = torch.cuda.current_device() if torch.cuda.is_available() else 0
    check(lib.lk_ops_status(index))


def _number(v, what, types):
    """A number for all rows, as the type of the vectors can hold it."""
    if not isinstance(v, numbers.Real):
        _refuse(LK_EINVAL, f"{what}: a CUDA tensor or a number is wanted")
    if types is _I32:
        if not isinstance(v, numbers.Integral) and not (math.isfinite(v) and v == int(v)):
            _refuse(LK_EINVAL, f"{what}: {v} is not a whole number")
        if not -(1 << 31) <= v < 1 << 31:
            _refuse(LK_ERANGE, f"{what}: {v} is outside int32")
        return int(v)
    if _F32_MAX < abs(v) < math.inf:
        _refuse(LK_ERANGE, f"{what}: {v} is outside float32")
    return float(v)


def _per_row(v, what, types, scores, rows, dev):
    """(address, tensor) of one value per row: a vector, or a number for all rows."""
    if v is not None and not isinstance(v, torch.Tensor):
        v = scores.new_full((rows,), _number(v, what, types), dtype=types[0])
    return _vector(v, what, types, dev, rows), v


def sample(scores, u, *, temperature=None, top_k=None, top_p=None, min_p=None, out_ids=None):
    """One draw per row of ``scores`` [rows, vocab] from the random numbers ``u`` [rows] in [0, 1):
    -> (ids [rows] int64, probs [rows] float32, kept [rows] int32).

    ``temperature``, ``top_p``, ``min_p`` (float32) and ``top_k`` (int32) are vectors of one value per row, or
    numbers for all rows (``top_k`` a whole one; a number costs a kernel that fills a vector); None switches a filter off.  ``probs`` is the probability of the draw among the
    ``kept`` entries.  A row with nothing to draw (only NaN and -inf) gets id -1.
    """
    rows, vocab, ld, dev = _matrix(scores, "scores", _FLOATS)
    up = _vector(u, "u", _F32, dev, rows)
    t, hold_t = _per_row(temperature, "temperature", _F32, scores, rows, dev)
    k, hold_k = _per_row(top_k, "top_k", _I32, scores, rows, dev)
    p, hold_p = _per_row(top_p, "top_p", _F32, scores, rows, dev)
    mp, hold_mp = _per_row(min_p, "min_p", _F32, scores, rows, dev)
    if up is None:
        _refuse(LK_EINVAL, "u: a CUDA tensor is wanted")
    place = scores.device
    ids = _new((rows,), (1,), dtype=torch.int64, device=place) if out_ids is None else out_ids
    probs, kept = _new((rows,), (1,), dtype=torch.float32, device=place), _new((rows,), (1,), dtype=torch.int32, device=place)
    st = _sample(dev, _FLOATS[scores.dtype], rows, vocab, scores.data_ptr(), ld, t, k, p, mp, up,
                       _vector(ids, "out_ids", _I64, dev, rows), probs.data_ptr(), kept.data_ptr(), _stream(dev))
    if st:
        check(st)
    if out_ids is not None:
        _written(out_ids)
    return ids, probs, kept
