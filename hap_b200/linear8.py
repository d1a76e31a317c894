"""``F.linear`` with all three products in 8-bit floating point: the training form of the block-scaled product.

Same call shape as :func:`hap_b200.linear.linear` (the ``torch.nn.functional.linear`` nodes of the synthesized program,
``hap.rs:1030-1037``).  The tensors keep their types: bfloat16 or float32 in, the same out; what is multiplied is their
8-bit form (:mod:`hap_b200.block8`), made inside the call:

    y  = x8 w8^T + b       x8 in 1 x 128 blocks along in_features, w8 in 128 x 128 blocks
    dx = g8 w8             g8 in 1 x 128 blocks along out_features, the same w8
    dW = g8t^T x8t         g and x in 128 x 1 blocks along the tokens
    db = sum g             from g itself

x8t is written by the pass that makes x8 and is all the forward pass keeps of x: one byte per element and one
per 128 instead of two or four bytes per element.  The weight's 8-bit transposed form is kept too (one byte per
weight).  A weight that does not change (evaluation, frozen layers) is quantised once with
:func:`hap_b200.block8.quantize_weight` and passed as it is.

Blocks start where the tensor starts.  So a shard of a weight that is not cut at multiples of 128 is rounded otherwise
than the whole weight, and so are x and g where the cut runs through their contraction; y and dx of a token do not depend
on how the batch is cut, dW does (by the roundings of x8t and g8t).
"""
from __future__ import annotations

import functools
from typing import Optional, Union

import torch

from . import _native as N
from .block8 import Block8, _CODES, _up
from .comm import _differentiated, _launch, _on_device, _once


@functools.lru_cache(maxsize=4096)
def _forward_workspace(device, m, n, k, prepared, keep_x) -> int:
    with _on_device(device):
        return N.lib.hapx_linear8_forward_workspace(m, n, k, prepared, keep_x)


@functools.lru_cache(maxsize=4096)
def _backward_workspace(device, m, n, k, dx, dw, db) -> int:
    with _on_device(device):
        return N.lib.hapx_linear8_backward_workspace(m, n, k, dx, dw, db)


def _kept_bytes(rows: int, cols: int):
    """Bytes of an 8-bit matrix and of its scales, rounded up so that pieces laid one after another stay aligned."""
    return _up(rows * _up(cols, 16), 256), _up(cols, 512) // 512 * _up(rows, 128) * 4


def _rows(t: torch.Tensor):
    """The matrix of a tensor's last dimension (a copy only when its rows do not lie at one pitch) and that pitch."""
    cols = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(t.numel() // cols, cols)
    if t.is_contiguous():
        return t, cols
    if t.shape[0] > 1 and t.stride(0) < cols or cols > 1 and t.stride(1) != 1:
        return t.contiguous(), cols
    return t, t.stride(0) if t.shape[0] > 1 else cols


def _forward(x, weight, bias, prepared, keep_x, keep_w):
    """y and the block of kept bytes (x8t, its scales, w8t, its scales; None when neither is asked for)."""
    device, dtype = x.device, x.dtype
    k = x.shape[-1]
    m = x.numel() // k
    x2, ldx = _rows(x)
    if prepared is None:
        n = weight.shape[0]
        w, ldw = _rows(weight)
        w_ptr, w8_ptr, w8s_ptr = w.data_ptr(), None, None
    else:
        n = prepared.rows
        ldw, w_ptr, w8_ptr, w8s_ptr = 0, None, prepared.values.data_ptr(), prepared.scales.data_ptr()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    y = x.new_empty((*x.shape[:-1], n))
    if m == 0:
        keep_x = False
    kept = xt = xts = wt = wts = None
    if keep_x or keep_w:
        (xv, xs), (wv, ws_) = _kept_bytes(k, m) if keep_x else (0, 0), _kept_bytes(k, n) if keep_w else (0, 0)
        kept = x.new_empty(xv + xs + wv + ws_, dtype=torch.uint8)
        base = kept.data_ptr()
        if keep_x:
            xt, xts = base, base + xv
        if keep_w:
            wt, wts = base + xv + xs, base + xv + xs + wv
    need = _forward_workspace(device, m or 1, n, k, prepared is not None, keep_x)
    work = x.new_empty(need, dtype=torch.uint8) if need else None
    _launch(device, N.lib.hapx_linear8_forward, y.data_ptr(), x2.data_ptr(), ldx, w_ptr, ldw, w8_ptr, w8s_ptr,
            bias.data_ptr() if bias is not None else None, _CODES[dtype], m, n, k, xt, xts, wt, wts, work.data_ptr() if need else None, need)
    return y, kept


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, prepared):
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        y, kept = _forward(x, weight, bias, prepared, need_w, need_x and prepared is None)
        t = prepared.transposed if prepared is not None and need_x else None
        ctx.save_for_backward(kept, *((t.values, t.scales) if t is not None else ()))
        ctx.meta = (x.shape, y.shape[-1], need_x, need_w, need_b)
        return y

    @staticmethod
    @_once
    def backward(ctx, g):
        kept, *prepared_t = ctx.saved_tensors
        x_shape, n, need_x, need_w, need_b = ctx.meta
        device, dtype = g.device, g.dtype
        k = x_shape[-1]
        m = g.numel() // n
        g2, ldg = _rows(g)
        dx = g.new_empty(x_shape) if need_x else None
        dw = g.new_empty((n, k)) if need_w else None
        db = g.new_empty(n) if need_b else None
        xt = xts = wt = wts = None
        xv, xs = _kept_bytes(k, m) if need_w and m else (0, 0)
        if need_w and m:
            xt, xts = kept.data_ptr(), kept.data_ptr() + xv
        if prepared_t:
            wt, wts = prepared_t[0].data_ptr(), prepared_t[1].data_ptr()
        elif need_x:
            wt = kept.data_ptr() + xv + xs
            wts = wt + _kept_bytes(k, n)[0]
        need = _backward_workspace(device, m or 1, n, k, need_x, need_w, need_b)
        work = g.new_empty(need, dtype=torch.uint8)
        _launch(device, N.lib.hapx_linear8_backward, dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None,
                db.data_ptr() if need_b else None, g2.data_ptr(), ldg, _CODES[dtype], m, n, k, wt, wts, xt, xts, work.data_ptr(), need)
        return dx, dw, db, None


def _check_prepared(w8: Block8, transposed: bool) -> None:
    """The kernels take a prepared weight's pitch as its row rounded up to 16 bytes, as ``quantize_weight`` makes it."""
    forms = [w8]
    if transposed:
        t = w8.transposed
        if t is None:
            raise ValueError("linear8: the input's gradient needs the weight's transposed form: block8.quantize_weight(w, transposed=True)")
        if t.rows != w8.cols or t.cols != w8.rows:
            raise ValueError(f"linear8: {t} is not the transposed form of {w8}")
        forms.append(t)
    for q in forms:
        if q.values.shape[1] != _up(q.cols, 16):
            raise ValueError(f"linear8: the weight's rows lie {q.values.shape[1]} bytes apart, {_up(q.cols, 16)} are expected")


def linear8(input: torch.Tensor, weight: Union[torch.Tensor, Block8], bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``F.linear(input, weight, bias)`` on CUDA bfloat16 or float32 tensors of any extents, with the products in 8-bit
    floating point (see the module).  ``weight``: a tensor of the input's type, or a :class:`hap_b200.block8.Block8`
    from :func:`hap_b200.block8.quantize_weight` - then nothing is computed for a weight gradient, and a gradient of
    the input needs the weight's transposed form (``quantize_weight(w, transposed=True)``).  No forward-mode derivative: a
    tangent is refused."""
    if not input.is_cuda:
        raise RuntimeError(f"linear8: hap_b200 has no CPU path; tensor is on {input.device}")
    dtype, shape = input.dtype, input.shape
    if dtype not in _CODES:
        raise TypeError(f"linear8: operands must be bfloat16 or float32, got {dtype}")
    if not shape or shape[-1] < 1:
        raise ValueError(f"linear8: at least one input feature is expected, got shape {tuple(shape)}")
    prepared = None
    if isinstance(weight, Block8):
        prepared, weight = weight, None
        _check_prepared(prepared, input.requires_grad and torch.is_grad_enabled())
        fout, fin, device = prepared.rows, prepared.cols, prepared.device
    else:
        if weight.dim() != 2 or weight.shape[0] < 1:
            raise ValueError(f"linear8: the weight must be (out_features, in_features), got shape {tuple(weight.shape)}")
        if weight.dtype != dtype:
            raise TypeError(f"linear8: mixed operand dtypes {dtype} and {weight.dtype}")
        (fout, fin), device = weight.shape, weight.device
    if fin != shape[-1]:
        raise ValueError(f"linear8: input features {shape[-1]} != weight in_features {fin}")
    if device != input.device:
        raise ValueError(f"linear8: input is on {input.device}, weight on {device}")
    if bias is not None:
        if bias.dtype != dtype:
            raise TypeError(f"linear8: mixed operand dtypes {dtype} and {bias.dtype}")
        if bias.shape != (fout,) or bias.device != device:
            raise ValueError(f"linear8: the bias must be ({fout},) on {device}, got {tuple(bias.shape)} on {bias.device}")
    if _differentiated(input, weight, bias):
        return _Linear8.apply(input, weight, bias, prepared)
    return _forward(input, weight, bias, prepared, False, False)[0]
