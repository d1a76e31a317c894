"""``torch.nn.functional.layer_norm`` over the last dimension on this package's kernels.

Same call shape as the function the planner's programs name (``hap.rs:1637-1660``): the fx target
can be swapped without touching the arguments.  Rows of up to 2048 float32 / bfloat16 elements
(a multiple of 8) with an elementwise weight take the fused kernels (one read of ``x`` forward; one
read of ``x`` and ``dy`` backward, deterministic parameter gradients); any other call is handed to
torch's own CUDA implementation unchanged.
"""
from __future__ import annotations

import functools

import torch
import torch.nn.functional as F

from . import _native as N
from .comm import _differentiated, _launch, _on_device, _once

_DTYPES = {torch.float32: N.F32, torch.bfloat16: N.BF16}


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        E = x.shape[-1]
        xc = x.contiguous()
        rows = xc.numel() // E
        y = torch.empty_like(xc)
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        w = weight.contiguous()
        b = None if bias is None else bias.contiguous()
        with torch.cuda.device(x.device):
            N.check(N.lib.hapx_layer_norm_forward(xc.data_ptr(), w.data_ptr(), 0 if b is None else b.data_ptr(), y.data_ptr(),
                                                  mean.data_ptr(), rstd.data_ptr(), _DTYPES[x.dtype], rows, E, float(eps),
                                                  torch.cuda.current_stream().cuda_stream))
        ctx.save_for_backward(xc, w, mean, rstd)
        ctx.has_bias = bias is not None
        ctx.x_shape = x.shape
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, w, mean, rstd = ctx.saved_tensors
        E = xc.shape[-1]
        rows = xc.numel() // E
        dyc = dy.contiguous()
        dx = torch.empty_like(xc)
        need_w, need_b = ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        dw = torch.empty_like(w) if need_w else None
        db = torch.empty_like(w) if need_b else None
        blocks = N.lib.hapx_layer_norm_backward_blocks(rows, E)
        partial = torch.empty(2 * E * blocks, dtype=torch.float32, device=xc.device)
        with torch.cuda.device(xc.device):
            N.check(N.lib.hapx_layer_norm_backward(xc.data_ptr(), dyc.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                                   dx.data_ptr(), 0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(),
                                                   partial.data_ptr(), _DTYPES[xc.dtype], rows, E,
                                                   torch.cuda.current_stream().cuda_stream))
        return dx, dw, db, None


class _LayerNormFork(torch.autograd.Function):
    """(x, layer_norm(x)): the input handed through next to its normalised form, so that the gradient arriving
    through the residual connection and the gradient of the normalised branch meet in ONE backward kernel
    (``dx = layer_norm_backward(dy) + d_residual``) instead of in an addition kernel of autograd's."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y = _LayerNorm.forward(ctx, x, weight, bias, eps)
        return x.view_as(x), y

    @staticmethod
    def backward(ctx, d_residual, dy):
        xc, w, mean, rstd = ctx.saved_tensors
        if dy is None:                       # the normalised branch took no part in the loss
            return d_residual, None, None, None
        E = xc.shape[-1]
        rows = xc.numel() // E
        dyc = dy.contiguous()
        add = None if d_residual is None else d_residual.contiguous()
        dx = torch.empty_like(xc)
        need_w, need_b = ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        dw = torch.empty_like(w) if need_w else None
        db = torch.empty_like(w) if need_b else None
        blocks = N.lib.hapx_layer_norm_backward_blocks(rows, E)
        partial = torch.empty(2 * E * blocks, dtype=torch.float32, device=xc.device)
        with torch.cuda.device(xc.device):
            N.check(N.lib.hapx_layer_norm_backward_add(xc.data_ptr(), dyc.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                                       0 if add is None else add.data_ptr(), dx.data_ptr(),
                                                       0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(),
                                                       partial.data_ptr(), _DTYPES[xc.dtype], rows, E,
                                                       torch.cuda.current_stream().cuda_stream))
        return dx.view(ctx.x_shape), dw, db, None


def _fusable(input, shape, weight, bias) -> bool:
    E = input.shape[-1] if input.dim() else 0
    return (input.is_cuda and len(shape) == 1 and shape[0] == E and weight is not None and input.dtype in _DTYPES
            and weight.dtype == input.dtype and (bias is None or bias.dtype == input.dtype)
            and E % 8 == 0 and 8 <= E <= 2048 and input.numel() > 0)


def layer_norm(input: torch.Tensor, normalized_shape, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not _fusable(input, shape, weight, bias):
        return F.layer_norm(input, shape, weight, bias, eps)
    return _LayerNorm.apply(input, weight, bias, eps)


def layer_norm_fork(input: torch.Tensor, normalized_shape, weight=None, bias=None, eps: float = 1e-5):
    """``(input, layer_norm(input, ...))`` for the pre-LN residual pattern ``x + f(layer_norm(x))``: use the first
    result where the program used ``x`` on the residual path.  Same values as :func:`layer_norm`; the backward pass
    adds the residual path's gradient inside the normalisation's backward kernel."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not _fusable(input, shape, weight, bias) or not input.is_contiguous():
        return input, layer_norm(input, shape, weight, bias, eps)
    return _LayerNormFork.apply(input, weight, bias, eps)


# ---- the input kept for the backward pass in 8 bits ---------------------------------------------------
def _ptr(t):
    return None if t is None else t.data_ptr()


def _kept8(rows: int, E: int):
    """Pitch of a row of e4m3 bytes; where the scales and the statistics start behind them; bytes in all."""
    pitch = (E + 15) // 16 * 16
    scales = rows * pitch
    stats = scales + 4 * rows * ((E + 127) // 128)
    return pitch, scales, stats, stats + 8 * rows


def _norm8_forward(x, w, b, eps, keep):
    """y, and - ``keep`` - one block of bytes for the backward pass: the input as e4m3 bytes, its scales, mean and rstd."""
    E = x.shape[-1]
    rows = x.numel() // E
    xc = x.contiguous()
    y = torch.empty_like(xc)
    pitch, scales_at, stats_at, size = _kept8(rows, E)
    kept = saved = scales = mean = rstd = None
    if keep:
        kept = x.new_empty(size, dtype=torch.uint8)
        saved = kept.data_ptr()
        scales, mean, rstd = saved + scales_at, saved + stats_at, saved + stats_at + 4 * rows
    _launch(x.device, N.lib.hapx_layer_norm8_forward, xc.data_ptr(), _ptr(w), _ptr(b), y.data_ptr(), mean, rstd, saved, pitch, scales,
            _DTYPES[x.dtype], rows, E, eps)
    return y, kept


def _norm8_save(ctx, x, weight, bias, eps):
    w = None if weight is None else weight.contiguous()
    y, kept = _norm8_forward(x, w, None if bias is None else bias.contiguous(), eps, True)
    ctx.save_for_backward(kept, w)
    _, ctx.need_w, ctx.need_b, _ = ctx.needs_input_grad
    return y


@functools.lru_cache(maxsize=4096)
def _norm8_workspace(device, rows, E) -> int:
    with _on_device(device):
        return N.lib.hapx_layer_norm8_backward_workspace(rows, E)


def _norm8_backward(ctx, dy, add):
    kept, w = ctx.saved_tensors
    E, device, dtype = dy.shape[-1], dy.device, dy.dtype
    rows = dy.numel() // E
    dy = dy.contiguous()
    add = None if add is None else add.contiguous()
    dx = torch.empty_like(dy)
    dw = dy.new_empty(E) if ctx.need_w else None
    db = dy.new_empty(E) if ctx.need_b else None
    pitch, scales_at, stats_at, _ = _kept8(rows, E)
    saved = kept.data_ptr()
    work = None
    if ctx.need_w or ctx.need_b:
        work = dy.new_empty(_norm8_workspace(device, rows, E), dtype=torch.uint8)
    _launch(device, N.lib.hapx_layer_norm8_backward, saved, pitch, saved + scales_at, dy.data_ptr(), _ptr(w), saved + stats_at,
            saved + stats_at + 4 * rows, _ptr(add), dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(work), _DTYPES[dtype], rows, E)
    return dx, dw, db, None


class _LayerNorm8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        return _norm8_save(ctx, x, weight, bias, eps)

    @staticmethod
    @_once
    def backward(ctx, dy):
        return _norm8_backward(ctx, dy, None)


class _LayerNormFork8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.set_materialize_grads(False)
        return x.view_as(x), _norm8_save(ctx, x, weight, bias, eps)

    @staticmethod
    @_once
    def backward(ctx, d_residual, dy):
        if dy is None:                       # the normalised branch took no part in the loss
            return d_residual, None, None, None
        return _norm8_backward(ctx, dy, d_residual)


def _check8(what, input, shape, weight, bias):
    if not input.is_cuda:
        raise RuntimeError(f"{what}: hap_b200 has no CPU path; tensor is on {input.device}")
    if input.dtype not in _DTYPES:
        raise TypeError(f"{what}: bfloat16 or float32 only, got {input.dtype}")
    if len(shape) != 1 or input.dim() < 1 or input.shape[-1] != shape[0] or shape[0] < 1:
        raise ValueError(f"{what}: normalises the last dimension only, got normalized_shape {shape} for an input of shape {tuple(input.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != input.dtype or t.shape != shape or t.device != input.device):
            raise ValueError(f"{what}: the {name} must be {shape}, {input.dtype}, on {input.device}; got {tuple(t.shape)}, {t.dtype}, on {t.device}")


def layer_norm8(input: torch.Tensor, normalized_shape, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """:func:`layer_norm` over the last dimension (of any extent up to 2^20) that keeps its input for the backward pass as
    e4m3 values with one scale per 128 columns (:mod:`hap_b200.block8`) and two floats per row, instead of the input
    itself.  The result is layer_norm's to the order of its float32 sums; the gradients are layer_norm's at the rounded
    input, normalised with the statistics of the input itself.  No forward-mode derivative: a tangent is refused."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    _check8("layer_norm8", input, shape, weight, bias)
    if _differentiated(input, weight, bias):
        return _LayerNorm8.apply(input, weight, bias, eps)
    return _norm8_forward(input, None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous(), eps, False)[0]


def layer_norm_fork8(input: torch.Tensor, normalized_shape, weight=None, bias=None, eps: float = 1e-5):
    """:func:`layer_norm_fork` on :func:`layer_norm8`: ``(input, layer_norm8(input, ...))`` with the residual path's
    gradient added inside the normalisation's backward kernel."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    _check8("layer_norm_fork8", input, shape, weight, bias)
    if _differentiated(input, weight, bias):
        return _LayerNormFork8.apply(input, weight, bias, eps)
    return input, layer_norm8(input, shape, weight, bias, eps)
