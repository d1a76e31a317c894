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
"""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from . import block8
from .block8 import Block8, _CODES, _empty, _run
from .comm import _on_device, _stream


def _pack(*forms):
    """Tensors and plain values of some Block8 operands, for ctx."""
    tensors, meta = [], []
    for f in forms:
        if f is None:
            tensors += [None, None]
            meta.append(None)
        else:
            tensors += [f.values, f.scales]
            meta.append((f.rows, f.cols))
    return tensors, meta


def _unpack(tensors, meta):
    return [None if m is None else Block8(tensors[2 * i], tensors[2 * i + 1], *m) for i, m in enumerate(meta)]


def _bias_grad(partial: torch.Tensor, rows: int, cols: int, dtype) -> torch.Tensor:
    db = torch.empty(cols, dtype=dtype, device=partial.device)
    with _on_device(partial.device):
        N.check(N.lib.hapx_block8_colsum_join(db.data_ptr(), _CODES[dtype], partial.data_ptr(), rows, cols, _stream(partial.device)))
    return db


class _Linear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, prepared, keep):
        rows, fin = x.numel() // x.shape[-1], x.shape[-1]
        x2 = block8._matrix(x.reshape(rows, fin), "linear8")
        need_x, need_w, need_b = (keep and n for n in ctx.needs_input_grad[:3])
        need_w = need_w and prepared is None
        if prepared is None:
            w8 = block8.quantize_weight(weight, transposed=need_x)
        else:
            w8 = prepared
        x8t = None
        if rows:
            x8 = _empty(rows, fin, x.device)
            x8t = _empty(fin, rows, x.device) if need_w else None
            _run(x2, False, x8, x8t)
            y = block8.matmul(x8, w8, bias, x.dtype)
        else:
            y = torch.empty((0, w8.rows), dtype=x.dtype, device=x.device)
        tensors, ctx.forms = _pack(x8t, w8.transposed if need_x else None)
        ctx.save_for_backward(*tensors)
        ctx.needs = (need_x, need_w, need_b and bias is not None)
        ctx.fout, ctx.x_shape, ctx.dtype = w8.rows, x.shape, x.dtype
        return y.view(*x.shape[:-1], w8.rows)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        need_x, need_w, need_b = ctx.needs
        x8t, w8t = _unpack(ctx.saved_tensors, ctx.forms)
        fout, fin = ctx.fout, ctx.x_shape[-1]
        rows = g.numel() // fout
        dx = dw = db = None
        if rows == 0:
            if need_x:
                dx = torch.empty(ctx.x_shape, dtype=ctx.dtype, device=g.device)
            if need_w:
                dw = torch.zeros((fout, fin), dtype=ctx.dtype, device=g.device)
            if need_b:
                db = torch.zeros(fout, dtype=ctx.dtype, device=g.device)
            return dx, dw, db, None, None
        g2 = block8._matrix(g.reshape(rows, fout), "linear8 backward")
        # one read of g: its rows for dx, its columns for dW, partial column sums for db
        g8 = _empty(rows, fout, g.device) if need_x or not need_w else None
        g8t = _empty(fout, rows, g.device) if need_w else None
        partial = torch.empty((block8._blocks(rows), fout), dtype=torch.float32, device=g.device) if need_b else None
        _run(g2, False, g8, g8t, partial)
        if need_x:
            dx = block8.matmul(g8, w8t, None, ctx.dtype).view(ctx.x_shape)
        if need_w:
            dw = block8.matmul(g8t, x8t, None, ctx.dtype)
        if need_b:
            db = _bias_grad(partial, rows, fout, ctx.dtype)
        return dx, dw, db, None, None


def linear8(input: torch.Tensor, weight: Union[torch.Tensor, Block8], bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``F.linear(input, weight, bias)`` on CUDA bfloat16 or float32 tensors of any extents, with the products in 8-bit
    floating point (see the module).  ``weight``: a tensor of the input's type, or a :class:`hap_b200.block8.Block8`
    from :func:`hap_b200.block8.quantize_weight` - then nothing is computed for a weight gradient, and a gradient of
    the input needs the weight's transposed form (``quantize_weight(w, transposed=True)``)."""
    if not input.is_cuda:
        raise RuntimeError(f"linear8: hap_b200 has no CPU path; tensor is on {input.device}")
    if input.dtype not in _CODES:
        raise TypeError(f"linear8: operands must be bfloat16 or float32, got {input.dtype}")
    if input.dim() < 1 or input.shape[-1] < 1:
        raise ValueError(f"linear8: at least one input feature is expected, got shape {tuple(input.shape)}")
    prepared = weight if isinstance(weight, Block8) else None
    if prepared is not None:
        if input.requires_grad and torch.is_grad_enabled() and prepared.transposed is None:
            raise ValueError("linear8: the input's gradient needs the weight's transposed form: block8.quantize_weight(w, transposed=True)")
        fout, fin, device = prepared.rows, prepared.cols, prepared.device
        weight = None
    else:
        if weight.dim() != 2 or weight.shape[0] < 1:
            raise ValueError(f"linear8: the weight must be (out_features, in_features), got shape {tuple(weight.shape)}")
        if weight.dtype != input.dtype:
            raise TypeError(f"linear8: mixed operand dtypes {input.dtype} and {weight.dtype}")
        (fout, fin), device = weight.shape, weight.device
    if fin != input.shape[-1]:
        raise ValueError(f"linear8: input features {input.shape[-1]} != weight in_features {fin}")
    if device != input.device:
        raise ValueError(f"linear8: input is on {input.device}, weight on {device}")
    if bias is not None:
        if bias.dtype != input.dtype:
            raise TypeError(f"linear8: mixed operand dtypes {input.dtype} and {bias.dtype}")
        if tuple(bias.shape) != (fout,) or bias.device != input.device:
            raise ValueError(f"linear8: the bias must be ({fout},) on {input.device}, got {tuple(bias.shape)} on {bias.device}")
    return _Linear8.apply(input, weight, bias, prepared, torch.is_grad_enabled())
