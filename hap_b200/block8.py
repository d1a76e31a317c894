"""8-bit blocks: matrices of e4m3 values with one power-of-two scale per block of 128, and their product.

:func:`quantize` turns a bfloat16 / float32 matrix into a :class:`Block8` whose blocks are 128 consecutive elements
of a row (activations, gradients); :func:`quantize_weight` one whose blocks are 128 x 128 tiles, which serve the
matrix and its transpose alike (weights: the forward product contracts over the columns, the input gradient over
the rows).  :func:`matmul` multiplies two of them along their rows, ``a @ b.T``, on the tensor cores with float32
sums.  :func:`hap_b200.linear8.linear8` is built from these.

A block's scale is the smallest power of two that brings its largest magnitude to 448 at most, so scaling is exact
and a value's only error is its rounding to the nearest e4m3 number: 2^-4 relative for magnitudes down to 2^-14 of
the block's largest.  Infinities and NaN become NaN (e4m3 has no infinity) and are left out of the maximum.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native as N
from .comm import _on_device, _stream

BLOCK = 128
_CODES = {torch.bfloat16: N.BF16, torch.float32: N.F32}


def _up(n: int, to: int) -> int:
    return (n + to - 1) // to * to


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _scale_bytes(rows: int, cols: int) -> int:
    return _up(cols, 512) // 512 * _blocks(rows) * 512


class Block8:
    """``rows x cols`` e4m3 values (``values``, float8_e4m3fn, contiguous, rows padded to a multiple of 16 bytes) and one
    power-of-two scale per 128 columns of a row (``scales``, bytes in the order the tensor cores read them;
    :meth:`scale_matrix` decodes them).  ``transposed`` is the same matrix with rows and columns exchanged, where the
    maker was asked for both."""

    __slots__ = ("values", "scales", "rows", "cols", "transposed")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, rows: int, cols: int, transposed: Optional["Block8"] = None):
        # the kernels take extents and pitch from here: what does not hold them is refused, not read past its end
        if rows < 0 or cols < 1:
            raise ValueError(f"Block8: {rows} x {cols} is no matrix")
        if values.dtype != torch.float8_e4m3fn or scales.dtype != torch.uint8:
            raise TypeError(f"Block8: values are float8_e4m3fn and scales uint8, got {values.dtype} and {scales.dtype}")
        if values.dim() != 2 or values.shape[0] != rows or values.shape[1] < cols or values.shape[1] % 16 or not values.is_contiguous():
            raise ValueError(f"Block8: the values of {rows} x {cols} are {rows} rows of a multiple of 16 bytes, contiguous; got {tuple(values.shape)}")
        if scales.numel() != _scale_bytes(rows, cols) or not scales.is_contiguous():
            raise ValueError(f"Block8: the scales of {rows} x {cols} are {_scale_bytes(rows, cols)} contiguous bytes, got {tuple(scales.shape)}")
        if scales.device != values.device:
            raise ValueError(f"Block8: values are on {values.device}, scales on {scales.device}")
        if transposed is not None and (transposed.rows != cols or transposed.cols != rows or transposed.device != values.device):
            raise ValueError(f"Block8: {transposed} is not the transposed form of {rows} x {cols} on {values.device}")
        self.values, self.scales, self.rows, self.cols, self.transposed = values, scales, rows, cols, transposed

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def device(self):
        return self.values.device

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.scales.numel()

    def scale_matrix(self) -> torch.Tensor:
        """The scales as float32, (rows, blocks of 128 columns)."""
        s = self.scales.view(_up(self.cols, 512) // 512, _blocks(self.rows), 32, 4, 4).permute(1, 3, 2, 0, 4)       # [row / 128][row / 32][row % 32][block / 4][block % 4]
        s = s.reshape(_blocks(self.rows) * BLOCK, _up(self.cols, 512) // 128)[:self.rows, :_blocks(self.cols)]
        return torch.ldexp(torch.ones(s.shape, device=s.device), s.to(torch.int32) - 127)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The matrix as it is represented (exact in bfloat16 too, as e4m3 has four significant bits; what a scale of 2^120 or
        one near 2^-126 takes out of the type's range is rounded there)."""
        if dtype not in _CODES:
            raise TypeError(f"block8: bfloat16 or float32 only, got {dtype}")
        out = torch.empty((self.rows, self.cols), dtype=dtype, device=self.device)
        with _on_device(self.device):
            N.check(N.lib.hapx_block8_dequantize(out.data_ptr(), _CODES[dtype], self.values.data_ptr(), self.values.shape[1],
                                                 self.scales.data_ptr(), self.rows, self.cols, _stream(self.device)))
        return out

    def __repr__(self):
        return f"Block8({self.rows} x {self.cols}, {self.device})"


def _matrix(x: torch.Tensor, what: str) -> torch.Tensor:
    if not x.is_cuda:
        raise RuntimeError(f"{what}: hap_b200 has no CPU path; tensor is on {x.device}")
    if x.dtype not in _CODES:
        raise TypeError(f"{what}: bfloat16 or float32 only, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError(f"{what}: a matrix is expected, got shape {tuple(x.shape)}")
    if x.shape[1] < 1:
        raise ValueError(f"{what}: rows of at least one element are expected")
    x = x.detach()
    if x.shape[0] > 1 and x.stride(0) < x.shape[1] or x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x


def _empty(rows: int, cols: int, device, transposed: Optional[Block8] = None) -> Block8:
    values = torch.empty((rows, _up(cols, 16)), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty(_scale_bytes(rows, cols), dtype=torch.uint8, device=device)
    return Block8(values, scales, rows, cols, transposed)


def _run(x: torch.Tensor, square: bool, q: Optional[Block8], qt: Optional[Block8]) -> None:
    """One pass of the quantiser over ``x`` into ``q`` (as it stands) and / or ``qt`` (transposed)."""
    rows, cols = x.shape
    ldx = x.stride(0) if rows > 1 else cols
    a = (q.values.data_ptr(), q.values.shape[1], q.scales.data_ptr()) if q is not None else (None, 0, None)
    b = (qt.values.data_ptr(), qt.values.shape[1], qt.scales.data_ptr()) if qt is not None else (None, 0, None)
    with _on_device(x.device):
        N.check(N.lib.hapx_block8_quantize(x.data_ptr(), _CODES[x.dtype], rows, cols, ldx, int(square), *a, *b, None,
                                           _stream(x.device)))


def quantize(x: torch.Tensor, rows: bool = True, columns: bool = False):
    """``x`` (rows x cols) in 1 x 128 blocks.  ``rows``: blocks along the rows, a :class:`Block8` of x.  ``columns``:
    blocks along the columns, a :class:`Block8` of x transposed (cols x rows).  Both forms come from one read of x;
    with both the result is the pair ``(rows form, columns form)``.  Not differentiable."""
    if not rows and not columns:
        raise ValueError("block8.quantize: nothing asked for")
    x = _matrix(x, "block8.quantize")
    if columns and x.shape[0] < 1:
        raise ValueError("block8.quantize: the columns of an empty matrix have no blocks")
    q = _empty(x.shape[0], x.shape[1], x.device) if rows else None
    qt = _empty(x.shape[1], x.shape[0], x.device) if columns else None
    _run(x, False, q, qt)
    return (q, qt) if rows and columns else (q if rows else qt)


def quantize_weight(w: torch.Tensor, transposed: bool = False) -> Block8:
    """``w`` (out_features x in_features) in 128 x 128 blocks, the layout :func:`hap_b200.linear8.linear8` takes for a
    weight that does not change from call to call.  ``transposed`` adds the transposed copy that the input gradient
    contracts over (``.transposed``, the same values and scales)."""
    w = _matrix(w, "block8.quantize_weight")
    if w.shape[0] < 1:
        raise ValueError("block8.quantize_weight: rows of at least one element are expected")
    qt = _empty(w.shape[1], w.shape[0], w.device) if transposed else None
    q = _empty(w.shape[0], w.shape[1], w.device, qt)
    _run(w, True, q, qt)
    return q


def matmul(a: Block8, b: Block8, bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a @ b.T (+ bias)``: a (m x k), b (n x k), m x n out.  Products and scales are multiplied on the tensor cores and
    summed there in float32; one rounding to ``out_dtype``.  ``bias``: n values of ``out_dtype``.  Not differentiable."""
    if a.cols != b.cols:
        raise ValueError(f"block8.matmul: contraction lengths differ ({a.cols} and {b.cols})")
    if a.device != b.device:
        raise ValueError(f"block8.matmul: operands are on {a.device} and {b.device}")
    if out_dtype not in _CODES:
        raise TypeError(f"block8.matmul: the output is bfloat16 or float32, got {out_dtype}")
    if bias is not None:
        if bias.dtype != out_dtype:
            raise TypeError(f"block8.matmul: bias is {bias.dtype}, the output {out_dtype}")
        if bias.numel() != b.rows or bias.device != a.device:
            raise ValueError(f"block8.matmul: {b.rows} bias values on {a.device} are expected")
        bias = bias.detach().contiguous()
    m, n, k = a.rows, b.rows, a.cols
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    with _on_device(a.device):
        need = N.lib.hapx_block8_matmul_workspace(m, n, k)
        ws = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None
        N.check(N.lib.hapx_block8_matmul(out.data_ptr(), _CODES[out_dtype], a.values.data_ptr(), a.values.shape[1], a.scales.data_ptr(),
                                         b.values.data_ptr(), b.values.shape[1], b.scales.data_ptr(),
                                         bias.data_ptr() if bias is not None else None, m, n, k, ws.data_ptr() if need else None, need,
                                         _stream(a.device)))
    return out
