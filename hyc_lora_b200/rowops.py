"""Thin callers of the row operators' entry points: counter-based dropout, layer norm of a residual sum, token log
probabilities, each with its backward pass.

Like the functions of :mod:`packed`, these allocate outputs, fill the argument records and enqueue the kernels on the current
stream of the tensors' device; none of them synchronises, and autograd does not see through them (the modules and Functions in
``operators/`` do that).  Tensors are float32 or bfloat16 and share one device, which need not be the current one.  Leading
dimensions are rows; rows may lie apart (a slice of a wider tensor), elements of a row may not (such inputs are copied).
"""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check, lib
from .packed import _dtype_code, _require_cuda


class LayerNormOut(NamedTuple):
    y: torch.Tensor
    z: torch.Tensor       # the sum in front of the norm (the input itself where there was neither residual nor dropout)
    mean: torch.Tensor    # fp32 [rows]
    rstd: torch.Tensor    # fp32 [rows]


class TokenLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]       # fp32, the shape of the targets
    entropy: Optional[torch.Tensor]       # fp32, one per row
    top_index: Optional[torch.Tensor]     # int64 [..., top]
    top_logprob: Optional[torch.Tensor]   # fp32 [..., top]
    stats: torch.Tensor                   # fp32 [rows, 2]: largest logit, log of the sum of exp(x - largest)


# The small calls of this module are bound by their host side: the raw-stream and device queries below are torch's cheap ones
# (0.1 us each instead of 2.2 for a Stream object), allocations of one dimension go through empty_strided (1.5 us, not 2.3),
# and the argument records are packed in one go (0.15 us, not 0.6 field by field) in the layout of the ctypes records in _lib.
_DROPOUT = struct.Struct("@qqiiPqPqPPd")                       # HycDropoutArgs
_LAYER_NORM = struct.Struct("@qiiifPqPqPPPdPPPP")              # HycLayerNormArgs
_LAYER_NORM_BWD = struct.Struct("@qiiiiPqPqPqPPPPdPPPPP")      # HycLayerNormBwdArgs
_LOGPROB = struct.Struct("@PqqqqiiPqiiPPPPP")                  # HycLogprobArgs
_LOGPROB_BWD = struct.Struct("@PqqqqiiPqPPPPPPiiP")            # HycLogprobBwdArgs
_CODES = {torch.float32: _lib.HYC_F32, torch.bfloat16: _lib.HYC_BF16}

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _device_of(first: torch.Tensor, *others) -> int:
    """The index of the one CUDA device that all tensors are on."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _require_cuda(first, t)
            raise RuntimeError(f"all tensors must be on one device, got {first.device} and {t.device}")
    if index < 0:
        _require_cuda(first)
    return index


def _launch(entry, name: str, args: bytes, index: int):
    """Enqueues on the current stream of device ``index``, which is made current for the call where it is not."""
    if index == _current_device():
        code = entry(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = entry(args, _raw_stream(index))
    if code:
        check(code, name)


def _vector(n: int, dtype: torch.dtype, device) -> torch.Tensor:
    return torch.empty_strided((n,), (1,), dtype=dtype, device=device)


def _result(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor like ``x``."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: torch.Tensor):
    """(tensor to read, row stride): the tensor itself where its rows are contiguous and lie evenly, else a copy."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return t, cols
    if t.stride(-1) == 1 or cols == 1:
        if t.dim() == 2:
            return t, t.stride(0)
        if t.dim() == 3 and t.stride(0) == t.shape[1] * t.stride(1):
            return t, t.stride(1)
    return t.contiguous(), cols


def _check_rng(rng: Optional[torch.Tensor]):
    if rng is None or rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous():
        raise ValueError("rng must be a contiguous int64 tensor of two values: seed and call number")


def check_like(name: str, t: torch.Tensor, x: torch.Tensor):
    if t.shape != x.shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(x.shape)}")
    if t.dtype != x.dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {x.dtype}")


def _check_params(weight, bias, cols: int):
    if (weight is not None and (weight.dim() != 1 or weight.numel() != cols or not weight.is_contiguous())) or (
            bias is not None and (bias.dim() != 1 or bias.numel() != cols or not bias.is_contiguous())):
        raise ValueError(f"weight and bias must be contiguous vectors of {cols} values")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype} and bias {bias.dtype}: one dtype for both")


def _check_row_stats(name: str, t: torch.Tensor, numel: int):
    if t.dtype != torch.float32 or t.numel() != numel or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of {numel} values")


# ---------------------------------------------------------------------------------------------------- dropout

def rng_take(state: torch.Tensor) -> torch.Tensor:
    """A fresh ``(seed, call)`` pair from ``state`` (int64 [2] on the device), whose call number moves on by one.  Concurrent
    calls take different numbers, and so does every replay of a graph this was recorded into."""
    _check_rng(state)
    index = _device_of(state)
    used = torch.empty_like(state)
    if index == _current_device():
        code = lib.hyc_rng_take(state.data_ptr(), used.data_ptr(), _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = lib.hyc_rng_take(state.data_ptr(), used.data_ptr(), _raw_stream(index))
    check(code, "hyc_rng_take")
    return used


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + dropout(x)``: element i (row-major) is kept where word i of the generator is at least ``p``, and divided by
    ``1 - p``.  The backward pass is the same call on the gradient, without residual, with the same ``rng``."""
    _check_rng(rng)
    index = _device_of(x, rng, residual)
    if x.dim() == 0:
        raise ValueError("dropout takes tensors of at least one dimension")
    code = _CODES.get(x.dtype)
    if code is None:
        code = _dtype_code(x)
    x_stride = residual_stride = at_residual = 0
    if residual is not None:
        check_like("residual", residual, x)
    if x.is_contiguous() and (residual is None or residual.is_contiguous()):
        rows, cols = 1, x.numel()
    else:
        if residual is not None:
            residual, residual_stride = _rows(residual)
        x, x_stride = _rows(x)
        cols = x.shape[-1]
        rows = x.numel() // max(1, cols)
    if residual is not None:
        at_residual = residual.data_ptr()
    y = _result(x)
    _launch(lib.hyc_dropout, "hyc_dropout",
            _DROPOUT.pack(rows, cols, code, 0, x.data_ptr(), x_stride, at_residual, residual_stride, y.data_ptr(), rng.data_ptr(), p), index)
    return y


# ---------------------------------------------------------------------------------------------------- layer norm

def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float = 1e-5, *,
               residual: Optional[torch.Tensor] = None, p: float = 0.0, rng: Optional[torch.Tensor] = None) -> LayerNormOut:
    """Layer norm over the last dimension of ``residual + dropout(x)``; ``rng`` is needed where ``p > 0``."""
    drop = p > 0.0
    index = _device_of(x, weight, bias, residual, rng if drop else None)
    if x.dim() == 0:
        raise ValueError("layer_norm takes tensors of at least one dimension")
    cols = x.shape[-1]
    code = _CODES.get(x.dtype)
    if code is None:
        code = _dtype_code(x)
    _check_params(weight, bias, cols)
    params = code if weight is None and bias is None else _dtype_code(weight if weight is not None else bias)
    at_rng = at_residual = residual_stride = 0
    if drop:
        _check_rng(rng)
        at_rng = rng.data_ptr()
    if residual is not None:
        check_like("residual", residual, x)
        residual, residual_stride = _rows(residual)
        at_residual = residual.data_ptr()
    x, x_stride = _rows(x)
    rows = x.numel() // cols if cols else 0
    y = _result(x)
    z = torch.empty_like(y) if drop or residual is not None else None
    mean = _vector(rows, torch.float32, x.device)
    rstd = torch.empty_like(mean)
    _launch(lib.hyc_layer_norm, "hyc_layer_norm",
            _LAYER_NORM.pack(rows, cols, code, params, eps, x.data_ptr(), x_stride, at_residual, residual_stride, _at(weight), _at(bias),
                             at_rng, p, y.data_ptr(), _at(z), mean.data_ptr(), rstd.data_ptr()), index)
    return LayerNormOut(y, x if z is None else z, mean, rstd)


def layer_norm_bwd(dy: torch.Tensor, z: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor, *,
                   p: float = 0.0, rng: Optional[torch.Tensor] = None, dz: Optional[torch.Tensor] = None,
                   need_dweight: bool = True, need_dbias: bool = True, param_dtype: Optional[torch.dtype] = None):
    """``(dx, dresidual, dweight, dbias)`` of :func:`layer_norm`.  ``dz`` is a gradient that reaches the sum past the norm.
    Where ``p == 0`` dx and dresidual are one tensor.  dweight and dbias come in the weight's dtype (``param_dtype``, then
    the input's, where there is no weight)."""
    drop = p > 0.0
    index = _device_of(dy, z, weight, mean, rstd, dz, rng if drop else None)
    if dy.dim() == 0:
        raise ValueError("layer_norm_bwd takes tensors of at least one dimension")
    cols = dy.shape[-1]
    _check_params(weight, None, cols)
    check_like("z", z, dy)
    code = _CODES.get(dy.dtype)
    if code is None:
        code = _dtype_code(dy)
    kind = weight.dtype if weight is not None else param_dtype or dy.dtype
    params = _CODES.get(kind)
    if params is None:
        params = _dtype_code(torch.empty(0, dtype=kind))
    at_rng = at_dz = dz_stride = 0
    if drop:
        _check_rng(rng)
        at_rng = rng.data_ptr()
    if dz is not None:
        check_like("dz", dz, dy)
        dz, dz_stride = _rows(dz)
        at_dz = dz.data_ptr()
    dy, dy_stride = _rows(dy)
    z, z_stride = _rows(z)
    rows = dy.numel() // cols if cols else 0
    _check_row_stats("mean", mean, rows)
    _check_row_stats("rstd", rstd, rows)
    dresidual = _result(dy)
    dx = torch.empty_like(dresidual) if drop else dresidual
    dweight = dbias = partials = None
    if need_dweight:
        dweight = torch.empty_like(weight) if weight is not None else _vector(cols, kind, dy.device)
    if need_dbias:
        dbias = torch.empty_like(weight) if weight is not None else _vector(cols, kind, dy.device)
    if need_dweight or need_dbias:
        floats = lib.hyc_layer_norm_bwd_scratch_floats(rows, cols)
        if floats < 0:
            check(floats, "hyc_layer_norm_bwd_scratch_floats")
        partials = _vector(floats, torch.float32, dy.device)
    _launch(lib.hyc_layer_norm_bwd, "hyc_layer_norm_bwd",
            _LAYER_NORM_BWD.pack(rows, cols, code, params, 0, dy.data_ptr(), dy_stride, z.data_ptr(), z_stride, at_dz, dz_stride, _at(weight),
                                 mean.data_ptr(), rstd.data_ptr(), at_rng, p, dresidual.data_ptr(), dx.data_ptr() if drop else 0,
                                 _at(dweight), _at(dbias), _at(partials)), index)
    return dx, dresidual, dweight, dbias


# ---------------------------------------------------------------------------------------------------- token log probabilities

def _logit_rows(t: torch.Tensor):
    """(tensor to read, rows, seq, row stride, batch stride): one or two leading strides are taken as they are."""
    vocab = t.shape[-1]
    if not t.is_contiguous() and (t.stride(-1) == 1 or vocab == 1):
        if t.dim() == 2:
            return t, t.shape[0], max(1, t.shape[0]), t.stride(0), 0
        if t.dim() == 3:
            return t, t.shape[0] * t.shape[1], max(1, t.shape[1]), t.stride(1), t.stride(0)
    t = t.contiguous()
    rows = t.numel() // max(1, vocab)
    return t, rows, max(1, rows), vocab, 0


def _check_targets(logits, targets):
    if targets.dtype != torch.int64:
        raise TypeError(f"targets are {targets.dtype}, expected torch.int64")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, expected {tuple(logits.shape[:-1])}")
    return targets.contiguous()


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, ignore_index: int = -100,
                   entropy: bool = False, top: int = 0) -> TokenLogprobs:
    """Log probabilities of ``targets`` under ``logits`` [..., vocab], in one pass and without an fp32 copy of the logits; with
    ``entropy`` the entropy of every row, with ``top`` its best tokens (the lower index first among equals).

    A target of ``ignore_index`` gives 0; where neither entropy nor alternatives are asked for its row is not read at all.  Any
    other target outside the vocabulary gives NaN.  A row without any finite logit (all -inf) gives -inf and entropy 0."""
    device = _device_of(logits, targets)
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must have a last dimension of at least one value")
    code = _CODES.get(logits.dtype)
    if code is None:
        code = _dtype_code(logits)
    lead, dev = logits.shape[:-1], logits.device
    flat = len(lead) == 1

    def per_row():
        return _vector(lead[0], torch.float32, dev) if flat else torch.empty(lead, dtype=torch.float32, device=dev)

    logprob = h = index = best = None
    if targets is not None:
        targets = _check_targets(logits, targets)
        logprob = per_row()
    logits, rows, seq, row_stride, batch_stride = _logit_rows(logits)
    stats = torch.empty_strided((rows, 2), (2, 1), dtype=torch.float32, device=dev)
    if entropy:
        h = torch.empty_like(logprob) if logprob is not None else per_row()
    if top > 0:
        if flat:
            index = torch.empty_strided((rows, top), (top, 1), dtype=torch.int64, device=dev)
            best = torch.empty_strided((rows, top), (top, 1), dtype=torch.float32, device=dev)
        else:
            index = torch.empty((*lead, top), dtype=torch.int64, device=dev)
            best = torch.empty((*lead, top), dtype=torch.float32, device=dev)
    _launch(lib.hyc_token_logprobs, "hyc_token_logprobs",
            _LOGPROB.pack(logits.data_ptr(), rows, row_stride, batch_stride, seq, logits.shape[-1], code, _at(targets), ignore_index, top, 0,
                          _at(logprob), _at(h), stats.data_ptr(), _at(best), _at(index)), device)
    return TokenLogprobs(logprob, h, index, best, stats)


def token_logprobs_bwd(logits: torch.Tensor, stats: torch.Tensor, targets: Optional[torch.Tensor] = None,
                       d_logprob: Optional[torch.Tensor] = None, *, ignore_index: int = -100,
                       entropy: Optional[torch.Tensor] = None, d_entropy: Optional[torch.Tensor] = None,
                       top_index: Optional[torch.Tensor] = None, d_top: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient with respect to ``logits`` (their dtype, contiguous) of what arrives for the results of
    :func:`token_logprobs`; ``stats``, ``entropy`` and ``top_index`` are those results.  Each of the three may be missing."""
    device = _device_of(logits, stats, targets, d_logprob, entropy, d_entropy, top_index, d_top)
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError("logits must have a last dimension of at least one value")
    code = _dtype_code(logits)
    grad = _result(logits)
    if d_logprob is not None:
        if targets is None:
            raise ValueError("a gradient of the log probabilities needs the targets")
        targets = _check_targets(logits, targets)
    logits, rows, seq, row_stride, batch_stride = _logit_rows(logits)
    _check_row_stats("stats", stats, 2 * rows)
    if d_logprob is not None:
        d_logprob = d_logprob.contiguous()
        _check_row_stats("d_logprob", d_logprob, rows)
    if d_entropy is not None:
        if entropy is None:
            raise ValueError("a gradient of the entropies needs the entropies")
        d_entropy = d_entropy.contiguous()
        _check_row_stats("entropy", entropy, rows)
        _check_row_stats("d_entropy", d_entropy, rows)
    top = 0
    if d_top is not None:
        if top_index is None or top_index.dtype != torch.int64 or top_index.shape != d_top.shape:
            raise ValueError("a gradient of the alternatives needs their int64 indices, of the same shape")
        d_top, top_index = d_top.contiguous(), top_index.contiguous()
        top = d_top.shape[-1]
        _check_row_stats("d_top", d_top, rows * top)
    _launch(lib.hyc_token_logprobs_bwd, "hyc_token_logprobs_bwd",
            _LOGPROB_BWD.pack(logits.data_ptr(), rows, row_stride, batch_stride, seq, logits.shape[-1], code,
                              _at(targets) if d_logprob is not None else 0, ignore_index, stats.data_ptr(),
                              _at(entropy) if d_entropy is not None else 0, _at(d_logprob), _at(d_entropy), _at(d_top),
                              _at(top_index) if top else 0, top, 0, grad.data_ptr()), device)
    return grad
