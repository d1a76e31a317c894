"""``torch.nn.functional.layer_norm`` over the last dimension on this package's kernels.

Same call shape as the function the planner's programs name (``hap.rs:1637-1660``): the fx target
can be swapped without touching the arguments.  Rows of up to 2048 float32 / bfloat16 elements
(a multiple of 8) with an elementwise weight take the fused kernels (one read of ``x`` forward; one
read of ``x`` and ``dy`` backward, deterministic parameter gradients); any other call is handed to
torch's own CUDA implementation unchanged.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _native as N
from .comm import _on_device, _stream

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
    return 0 if t is None else t.data_ptr()


def _norm8_forward(ctx, x, weight, bias, eps, keep):
    E = x.shape[-1]
    xc = x.contiguous()
    rows = xc.numel() // E
    pitch = (E + 15) // 16 * 16
    y = torch.empty_like(xc)
    saved = scales = stats = mean = rstd = None
    if keep and any(ctx.needs_input_grad[:3]):
        stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
        mean, rstd = stats[0], stats[1]
        saved = torch.empty((rows, pitch), dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty((rows, (E + 127) // 128), dtype=torch.float32, device=x.device)
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    with _on_device(x.device):
        N.check(N.lib.hapx_layer_norm8_forward(xc.data_ptr(), _ptr(w), _ptr(b), y.data_ptr(), _ptr(mean), _ptr(rstd), _ptr(saved), pitch,
                                               _ptr(scales), _DTYPES[x.dtype], rows, E, float(eps), _stream(x.device)))
    ctx.save_for_backward(saved, scales, stats, w)
    ctx.has_bias = bias is not None
    return y


def _norm8_backward(ctx, dy, add):
    saved, scales, stats, w = ctx.saved_tensors
    E = dy.shape[-1]
    rows = dy.numel() // E
    dyc = dy.contiguous()
    add = None if add is None else add.contiguous()
    dx = torch.empty_like(dyc)
    dw = torch.empty(E, dtype=dy.dtype, device=dy.device) if w is not None and ctx.needs_input_grad[1] else None
    db = torch.empty(E, dtype=dy.dtype, device=dy.device) if ctx.has_bias and ctx.needs_input_grad[2] else None
    work = None
    if dw is not None or db is not None:
        work = torch.empty(N.lib.hapx_layer_norm8_backward_workspace(rows, E) // 4, dtype=torch.float32, device=dy.device)
    with _on_device(dy.device):
        N.check(N.lib.hapx_layer_norm8_backward(saved.data_ptr(), saved.shape[1], scales.data_ptr(), dyc.data_ptr(), _ptr(w), stats[0].data_ptr(),
                                                stats[1].data_ptr(), _ptr(add), dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(work), _DTYPES[dy.dtype], rows, E,
                                                _stream(dy.device)))
    return dx, dw, db, None, None


class _LayerNorm8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        return _norm8_forward(ctx, x, weight, bias, eps, keep)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _norm8_backward(ctx, dy, None)


class _LayerNormFork8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        ctx.set_materialize_grads(False)
        y = _norm8_forward(ctx, x, weight, bias, eps, keep)
        return x.view_as(x), y

    @staticmethod
    @once_differentiable
    def backward(ctx, d_residual, dy):
        if dy is None:                       # the normalised branch took no part in the loss
            return d_residual, None, None, None, None
        return _norm8_backward(ctx, dy, d_residual)


def _check8(what, input, shape, weight, bias):
    if not input.is_cuda:
        raise RuntimeError(f"{what}: hap_b200 has no CPU path; tensor is on {input.device}")
    if input.dtype not in _DTYPES:
        raise TypeError(f"{what}: bfloat16 or float32 only, got {input.dtype}")
    if len(shape) != 1 or input.dim() < 1 or input.shape[-1] != shape[0] or shape[0] < 1:
        raise ValueError(f"{what}: normalises the last dimension only, got normalized_shape {shape} for an input of shape {tuple(input.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.dtype != input.dtype or tuple(t.shape) != shape or t.device != input.device):
            raise ValueError(f"{what}: the {name} must be {shape}, {input.dtype}, on {input.device}; got {tuple(t.shape)}, {t.dtype}, on {t.device}")


def layer_norm8(input: torch.Tensor, normalized_shape, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """:func:`layer_norm` over the last dimension (of any extent) that keeps its input for the backward pass as e4m3
    values with one scale per 128 columns (:mod:`hap_b200.block8`) and two floats per row, instead of the input
    itself.  The result is layer_norm's; the gradients are layer_norm's at the rounded input, normalised with the
    statistics of the input itself."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    _check8("layer_norm8", input, shape, weight, bias)
    return _LayerNorm8.apply(input, weight, bias, eps, torch.is_grad_enabled())


def layer_norm_fork8(input: torch.Tensor, normalized_shape, weight=None, bias=None, eps: float = 1e-5):
    """:func:`layer_norm_fork` on :func:`layer_norm8`: ``(input, layer_norm8(input, ...))`` with the residual path's
    gradient added inside the normalisation's backward kernel."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    _check8("layer_norm_fork8", input, shape, weight, bias)
    return _LayerNormFork8.apply(input, weight, bias, eps, torch.is_grad_enabled())
