"""Thin callers of the row operators' entry points: counter-based dropout, layer norm of a residual sum, token log
probabilities, each with its backward pass.

Like the functions of :mod:`packed`, these allocate outputs, fill the argument records and enqueue the kernels on the current
stream of the tensors' device; none of them synchronises, and autograd does not see through them (the modules and Functions in
``operators/`` do that).  Tensors are float32 or bfloat16 and share one device, which need not be the current one.  Leading
dimensions are rows; rows may lie apart (a slice of a wider tensor), elements of a row may not (such inputs are copied).
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from ._lib import HycDropoutArgs, HycLayerNormArgs, HycLayerNormBwdArgs, HycLogprobArgs, HycLogprobBwdArgs, check, lib
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
# (0.1 us each instead of 2.2 for a Stream object), and allocations of one dimension go through empty_strided (1.5 us, not 2.3).
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


def _launch(entry, name: str, args, index: int):
    """Enqueues on the current stream of device ``index``, which is made current for the call where it is not."""
    if index == _current_device():
        code = entry(C.byref(args), _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = entry(C.byref(args), _raw_stream(index))
    if code:
        check(code, name)


def _vector(n: int, dtype: torch.dtype, device) -> torch.Tensor:
    return torch.empty_strided((n,), (1,), dtype=dtype, device=device)


def _result(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor like ``x``."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


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


def _like(name: str, t: torch.Tensor, x: torch.Tensor):
    if t.shape != x.shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(x.shape)}")
    if t.dtype != x.dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {x.dtype}")


def _check_params(weight, bias, cols: int):
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (cols,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous vector of {cols} values")
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
    a = HycDropoutArgs()
    a.dtype = _dtype_code(x)
    if residual is not None:
        _like("residual", residual, x)
        if x.is_contiguous() and residual.is_contiguous():
            a.rows, a.cols = 1, x.numel()
        else:
            residual, a.residual_stride = _rows(residual)
        a.residual = residual.data_ptr()
    elif x.is_contiguous():
        a.rows, a.cols = 1, x.numel()
    if not a.rows:
        x, a.x_stride = _rows(x)
        a.cols = x.shape[-1]
        a.rows = x.numel() // max(1, a.cols)
    y = _result(x)
    a.x, a.y, a.rng, a.p = x.data_ptr(), y.data_ptr(), rng.data_ptr(), p
    _launch(lib.hyc_dropout, "hyc_dropout", a, index)
    return y


# ---------------------------------------------------------------------------------------------------- layer norm

def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float = 1e-5, *,
               residual: Optional[torch.Tensor] = None, p: float = 0.0, rng: Optional[torch.Tensor] = None) -> LayerNormOut:
    """Layer norm over the last dimension of ``residual + dropout(x)``; ``rng`` is needed where ``p > 0``."""
    index = _device_of(x, weight, bias, residual, rng if p > 0.0 else None)
    if x.dim() == 0:
        raise ValueError("layer_norm takes tensors of at least one dimension")
    cols = x.shape[-1]
    _check_params(weight, bias, cols)
    a = HycLayerNormArgs()
    a.dtype = _dtype_code(x)
    a.param_dtype = a.dtype if weight is None and bias is None else _dtype_code(weight if weight is not None else bias)
    if p > 0.0:
        _check_rng(rng)
        a.rng = rng.data_ptr()
    if residual is not None:
        _like("residual", residual, x)
        residual, a.residual_stride = _rows(residual)
        a.residual = residual.data_ptr()
    x, a.x_stride = _rows(x)
    rows = x.numel() // max(1, cols)
    y = _result(x)
    z = torch.empty_like(y) if residual is not None or p > 0.0 else None
    mean = _vector(rows, torch.float32, x.device)
    rstd = torch.empty_like(mean)
    a.rows, a.cols, a.eps, a.p = rows, cols, eps, p
    a.x, a.weight, a.bias, a.y, a.z = x.data_ptr(), _at(weight), _at(bias), y.data_ptr(), _at(z)
    a.mean, a.rstd = mean.data_ptr(), rstd.data_ptr()
    _launch(lib.hyc_layer_norm, "hyc_layer_norm", a, index)
    return LayerNormOut(y, x if z is None else z, mean, rstd)


def layer_norm_bwd(dy: torch.Tensor, z: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor, *,
                   p: float = 0.0, rng: Optional[torch.Tensor] = None, dz: Optional[torch.Tensor] = None,
                   need_dweight: bool = True, need_dbias: bool = True, param_dtype: Optional[torch.dtype] = None):
    """``(dx, dresidual, dweight, dbias)`` of :func:`layer_norm`.  ``dz`` is a gradient that reaches the sum past the norm.
    Where ``p == 0`` dx and dresidual are one tensor.  dweight and dbias come in the weight's dtype (``param_dtype``, then
    the input's, where there is no weight)."""
    index = _device_of(dy, z, weight, mean, rstd, dz, rng if p > 0.0 else None)
    if dy.dim() == 0:
        raise ValueError("layer_norm_bwd takes tensors of at least one dimension")
    cols = dy.shape[-1]
    _check_params(weight, None, cols)
    _like("z", z, dy)
    a = HycLayerNormBwdArgs()
    a.dtype = _dtype_code(dy)
    kind = weight.dtype if weight is not None else param_dtype or dy.dtype
    a.param_dtype = _dtype_code(torch.empty(0, dtype=kind)) if weight is None and kind != dy.dtype else _dtype_code(weight) if weight is not None else a.dtype
    if p > 0.0:
        _check_rng(rng)
        a.rng = rng.data_ptr()
    if dz is not None:
        _like("dz", dz, dy)
        dz, a.dz_stride = _rows(dz)
        a.dz = dz.data_ptr()
    dy, a.dy_stride = _rows(dy)
    z, a.z_stride = _rows(z)
    rows = dy.numel() // max(1, cols)
    _check_row_stats("mean", mean, rows)
    _check_row_stats("rstd", rstd, rows)
    dresidual = _result(dy)
    dx = torch.empty_like(dresidual) if p > 0.0 else dresidual
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
    a.rows, a.cols, a.p = rows, cols, p
    a.dy, a.z, a.weight, a.mean, a.rstd = dy.data_ptr(), z.data_ptr(), _at(weight), mean.data_ptr(), rstd.data_ptr()
    a.dresidual, a.dx = dresidual.data_ptr(), dx.data_ptr() if p > 0.0 else None
    a.dweight, a.dbias, a.partials = _at(dweight), _at(dbias), _at(partials)
    _launch(lib.hyc_layer_norm_bwd, "hyc_layer_norm_bwd", a, index)
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
    a = HycLogprobArgs()
    a.dtype = _dtype_code(logits)
    lead, dev = logits.shape[:-1], logits.device
    flat = len(lead) == 1

    def per_row():
        return _vector(lead[0], torch.float32, dev) if flat else torch.empty(lead, dtype=torch.float32, device=dev)

    logprob = h = index = best = None
    if targets is not None:
        targets = _check_targets(logits, targets)
        logprob = per_row()
        a.targets, a.logprob = targets.data_ptr(), logprob.data_ptr()
    logits, a.rows, a.seq, a.row_stride, a.batch_stride = _logit_rows(logits)
    a.logits, a.vocab, a.ignore_index, a.top = logits.data_ptr(), logits.shape[-1], ignore_index, top
    stats = torch.empty_strided((a.rows, 2), (2, 1), dtype=torch.float32, device=dev)
    a.stats = stats.data_ptr()
    if entropy:
        h = torch.empty_like(logprob) if logprob is not None else per_row()
        a.entropy = h.data_ptr()
    if top > 0:
        if flat:
            index = torch.empty_strided((lead[0], top), (top, 1), dtype=torch.int64, device=dev)
            best = torch.empty_strided((lead[0], top), (top, 1), dtype=torch.float32, device=dev)
        else:
            index = torch.empty((*lead, top), dtype=torch.int64, device=dev)
            best = torch.empty((*lead, top), dtype=torch.float32, device=dev)
        a.top_index, a.top_logprob = index.data_ptr(), best.data_ptr()
    _launch(lib.hyc_token_logprobs, "hyc_token_logprobs", a, device)
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
    a = HycLogprobBwdArgs()
    a.dtype = _dtype_code(logits)
    grad = _result(logits)
    if d_logprob is not None:
        if targets is None:
            raise ValueError("a gradient of the log probabilities needs the targets")
        targets = _check_targets(logits, targets)
    logits, a.rows, a.seq, a.row_stride, a.batch_stride = _logit_rows(logits)
    rows = a.rows
    _check_row_stats("stats", stats, 2 * rows)
    if d_logprob is not None:
        d_logprob = d_logprob.contiguous()
        _check_row_stats("d_logprob", d_logprob, rows)
        a.targets, a.d_logprob = targets.data_ptr(), d_logprob.data_ptr()
    if d_entropy is not None:
        if entropy is None:
            raise ValueError("a gradient of the entropies needs the entropies")
        d_entropy = d_entropy.contiguous()
        _check_row_stats("entropy", entropy, rows)
        _check_row_stats("d_entropy", d_entropy, rows)
        a.entropy, a.d_entropy = entropy.data_ptr(), d_entropy.data_ptr()
    if d_top is not None:
        if top_index is None or top_index.dtype != torch.int64 or top_index.shape != d_top.shape:
            raise ValueError("a gradient of the alternatives needs their int64 indices, of the same shape")
        d_top, top_index = d_top.contiguous(), top_index.contiguous()
        a.top = d_top.shape[-1]
        _check_row_stats("d_top", d_top, rows * a.top)
        a.top_index, a.d_top = top_index.data_ptr(), d_top.data_ptr()
    a.logits, a.vocab, a.ignore_index, a.stats, a.grad = logits.data_ptr(), logits.shape[-1], ignore_index, stats.data_ptr(), grad.data_ptr()
    _launch(lib.hyc_token_logprobs_bwd, "hyc_token_logprobs_bwd", a, device)
    return grad
