"""8-bit blocks and the operators built on them, restated in float64 on the CPU from their definitions: a block's scale
is the smallest power of two that brings its largest finite magnitude to 448 at most (not below 2^-126; 1 for a block
of zeros), a value is the nearest e4m3 number (3 fraction bits, exponents from -6 up, ties to even) of x / scale, and
what is not finite is NaN."""
import math

import torch

BLOCK = 128


def scale_of(big: float) -> float:
    if big == 0.0:
        return 1.0
    mant, exp = math.frexp(big / 448.0)          # big / 448 = mant 2^exp, mant in [0.5, 1)
    e = exp - 1 if mant == 0.5 else exp
    return math.ldexp(1.0, max(e, -126))


def round_e4m3(v: torch.Tensor) -> torch.Tensor:
    _, ex = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (ex - 1).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(v), torch.round(v / step) * step, torch.full_like(v, math.nan))


def _block(part: torch.Tensor):
    finite = part[torch.isfinite(part)].abs()
    s = scale_of(float(finite.max()) if finite.numel() else 0.0)
    return round_e4m3(part / s) * s, s


def quantize(x: torch.Tensor, square: bool = False):
    """Values (as what they stand for) and scales [column block, row or row block] of a matrix."""
    x = x.double()
    r, c = x.shape
    step = BLOCK if square else 1
    out = torch.empty_like(x)
    scales = torch.empty((-(-c // BLOCK), -(-r // step)), dtype=torch.float64)
    for i in range(0, r, step):
        for j in range(0, c, BLOCK):
            part, s = _block(x[i:i + step, j:j + BLOCK])
            out[i:i + step, j:j + BLOCK] = part
            scales[j // BLOCK, i // step] = s
    return out, scales


def fast_rows(x: torch.Tensor) -> torch.Tensor:
    """quantize(x)[0] for finite x without the loop over rows."""
    x = x.double()
    out = torch.empty_like(x)
    for j in range(0, x.shape[1], BLOCK):
        part = x[:, j:j + BLOCK]
        big = part.abs().amax(1, keepdim=True)
        mant, exp = torch.frexp(big / 448.0)
        e = torch.where(mant == 0.5, exp - 1, exp).clamp(min=-126)
        s = torch.where(big > 0, torch.ldexp(torch.ones_like(big), e), torch.ones_like(big))
        out[:, j:j + BLOCK] = round_e4m3(part / s) * s
    return out


def linear8(x, w, b, g):
    """y, dx, dw, db (float64) and, for each, the sum of magnitudes its float32 sum runs over."""
    xr, wq = fast_rows(x), quantize(w, square=True)[0]
    gr, gc, xc = fast_rows(g), fast_rows(g.t()), fast_rows(x.t())
    y, ys = xr @ wq.t(), xr.abs() @ wq.abs().t()
    if b is not None:
        y, ys = y + b.double(), ys + b.double().abs()
    return ((y, ys), (gr @ wq, gr.abs() @ wq.abs()), (gc @ xc.t(), gc.abs() @ xc.abs().t()), (g.double().sum(0), g.double().abs().sum(0)))


def runs(x: torch.Tensor) -> torch.Tensor:
    """x with every 128 consecutive elements (row-major) as one block."""
    flat = x.double().reshape(-1)
    pad = torch.cat([flat, flat.new_zeros(-flat.numel() % BLOCK)]).reshape(-1, BLOCK)
    return fast_rows(pad).reshape(-1)[:flat.numel()].reshape(x.shape)


def gelu(x):
    return 0.5 * x * torch.special.erfc(-x / math.sqrt(2.0))


def gelu_slope(x):
    return 0.5 * torch.special.erfc(-x / math.sqrt(2.0)) + x * torch.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)


def layer_norm8(x, w, b, g, eps=1e-5, add=None, kept=None):
    """y, dx, dw, db in float64; the backward pass normalises `kept` (x in 1 x 128 blocks) with the statistics of x."""
    x, g = x.double(), g.double()
    kept = fast_rows(x) if kept is None else kept
    w1 = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd * w1
    if b is not None:
        y = y + b.double()
    z = (kept - mean) * rstd
    gw = g * w1
    dx = rstd * (gw - gw.mean(1, keepdim=True) - z * (gw * z).mean(1, keepdim=True))
    if add is not None:
        dx = dx + add.double()
    return y, dx, (g * z).sum(0), g.sum(0)
