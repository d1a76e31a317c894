"""The cases by which the 8-bit training operators are timed and compared.

Four operators, each in the form a training or serving program calls it:

* ``linear8``      - ``F.linear`` forward and backward with every product in 8-bit floating point (e4m3), one
                     power-of-two scale per block of 128: 1 x 128 blocks of activations and gradients along the
                     contraction, 128 x 128 blocks of the weight;
* ``linear8_eval`` - the same forward product with a weight that was laid out once (serving, evaluation);
* ``act8``         - the FFN's activation, forward and backward, with its input kept for the backward pass in 8 bits
                     (gelu) or one bit (relu);
* ``norm8``        - layer_norm forward and backward with its input kept for the backward pass in 8 bits.

``run`` with ``own`` false computes them from elementary torch operations in 32 bits; with ``own`` true it makes the
calls a user of the framework makes.
"""
import math

import torch

own = False

BLOCK = 128
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------
def listed():
    return [
        # attention input projection of the Transformer LM: 32 sequences of 256 tokens, 768 -> 3 x 768
        {"name": "linear8_qkv", "op": "linear8", "tokens": 8192, "fin": 768, "fout": 2304, "bias": True, "dtype": "bf16"},
        # its vocabulary projection, the largest product of a step
        {"name": "linear8_vocab", "op": "linear8", "tokens": 8192, "fin": 768, "fout": 33280, "bias": True, "dtype": "bf16"},
        # the two-layer MLP of the float32 parity configuration: one rank's 38 of 64 samples
        {"name": "linear8_mlp_f32", "op": "linear8", "tokens": 38, "fin": 1024, "fout": 4096, "bias": True, "dtype": "f32"},
        # an uneven shard in every extent: a column-parallel cut that is no multiple of the block, an odd token count
        {"name": "linear8_ragged", "op": "linear8", "tokens": 5001, "fin": 1000, "fout": 1237, "bias": False, "dtype": "bf16"},
        # one token through a projection whose weight was quantised when the model was loaded
        {"name": "eval_one_token", "op": "linear8_eval", "tokens": 1, "fin": 768, "fout": 2304, "bias": True, "dtype": "bf16"},
        # a small evaluation batch through an expert-sized projection
        {"name": "eval_batch", "op": "linear8_eval", "tokens": 64, "fin": 1024, "fout": 4096, "bias": False, "dtype": "bf16"},
        # the ViT's attention output projection over 64 images of 197 patches
        {"name": "eval_vit", "op": "linear8_eval", "tokens": 12608, "fin": 768, "fout": 768, "bias": True, "dtype": "bf16"},
        # the activations of the MoE layer's experts: 16 x 32 x 20 slots of 4096 hidden units
        {"name": "act8_gelu", "op": "act8", "rows": 10240, "cols": 4096, "act": "gelu", "dtype": "bf16"},
        # a small ragged activation in float32
        {"name": "act8_relu_odd", "op": "act8", "rows": 333, "cols": 515, "act": "relu", "dtype": "f32"},
        # the norms of the Transformer LM
        {"name": "norm8_lm", "op": "norm8", "rows": 8192, "cols": 768, "bias": True, "dtype": "bf16"},
        # three images of the ViT
        {"name": "norm8_vit", "op": "norm8", "rows": 591, "cols": 768, "bias": True, "dtype": "bf16"},
        # a wide norm in float32 without a bias
        {"name": "norm8_wide_f32", "op": "norm8", "rows": 4000, "cols": 2040, "bias": False, "dtype": "f32"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear8", "linear8", "linear8_eval", "linear8_eval", "act8", "norm8"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("linear8", "linear8_eval"):
        tokens = _log_int(rng, 1, 16384)
        fin, fout = _log_int(rng, 16, 4096), _log_int(rng, 16, 33280)
        most = 8192 * 768 * 33280 // (2 if dtype == "f32" else 1)
        tokens = max(1, min(tokens, most // (fin * fout)))
        return {"op": op, "tokens": tokens, "fin": fin, "fout": fout, "bias": rng.random() < 0.5, "dtype": dtype}
    if op == "act8":
        rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 8, 8192)
        return {"op": op, "rows": max(1, min(rows, 10240 * 4096 // cols)), "cols": cols, "act": rng.choice(["gelu", "relu"]), "dtype": dtype}
    cols = _log_int(rng, 8, 8192)
    return {"op": op, "rows": max(1, min(_log_int(rng, 1, 16384), 8192 * 2048 // cols)), "cols": cols, "bias": rng.random() < 0.5, "dtype": dtype}


# ---- inputs -----------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(dev).manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dt)

    s = {"case": case}
    if case["op"] in ("linear8", "linear8_eval"):
        t, fin, fout = case["tokens"], case["fin"], case["fout"]
        # a normalised activation with a few strong channels, as the projections of a trained model see it
        gain = torch.exp(0.7 * torch.randn(fin, generator=gen, device=dev))
        x = (torch.randn(t, fin, generator=gen, device=dev) * gain).to(dt)
        w = normal(fout, fin, scale=fin ** -0.5)
        b = normal(fout, scale=0.1) if case["bias"] else None
        if case["op"] == "linear8":
            # gradients whose size differs from token to token
            size = torch.exp(1.5 * torch.randn(t, 1, generator=gen, device=dev)) * 1e-3
            g = (torch.randn(t, fout, generator=gen, device=dev) * size).to(dt)
            s.update(x=x, w=w, b=b, g=g)
        else:
            if own:
                from hap_b200 import block8
                s.update(x=x, w=block8.quantize_weight(w), b=b)
            else:
                q, e = _plain_quantize(w.float(), square=True)
                s.update(x=x, w=(q, e), b=b)
    elif case["op"] == "act8":
        s.update(x=normal(case["rows"], case["cols"]), g=normal(case["rows"], case["cols"], scale=0.01))
    else:
        r, c = case["rows"], case["cols"]
        s.update(x=normal(r, c, scale=2.0) + torch.tensor(0.25, dtype=dt, device=dev), w=1 + normal(c, scale=0.2),
                 b=normal(c, scale=0.2) if case["bias"] else None, g=normal(r, c, scale=0.01))
    if own and case["op"] != "linear8_eval":
        for k in ("x", "w", "b"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    return s


# ---- the plain forms, 32 bits -------------------------------------------------------------------------
def _blocks(x, square):
    """x (rows, cols) as blocks, zero-extended: (rows, nb, 128), or (nr, 128, nc, 128) for square ones."""
    r, c = x.shape
    pc = -c % BLOCK
    pr = -r % BLOCK if square else 0
    x = torch.nn.functional.pad(x, (0, pc, 0, pr))
    return x.reshape(-1, BLOCK, (c + pc) // BLOCK, BLOCK) if square else x.reshape(r, -1, BLOCK)


def _plain_quantize(x, square=False):
    """e4m3 values and block exponents: the smallest power of two that brings the block's largest magnitude to 448 at
    most, and values rounded to the nearest e4m3 number."""
    v = _blocks(x, square)
    dims = (1, 3) if square else (2,)
    big = v.abs().amax(dim=dims, keepdim=True)
    mant, exp = torch.frexp(big)
    e = torch.where(mant > 0.875, exp - 8, exp - 9).clamp_(min=-126)
    e = torch.where(big > 0, e, torch.zeros_like(e))
    q = (v * torch.ldexp(torch.ones_like(big), -e)).to(torch.float8_e4m3fn)
    return q, e


def _plain_values(q, e, r, c):
    v = q.float() * torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)
    v = v.reshape(-1, v.shape[-1] * v.shape[-2]) if v.dim() == 4 else v.reshape(v.shape[0], -1)
    return v[:r, :c]


def _plain_q(x, square=False):
    return _plain_values(*_plain_quantize(x, square), *x.shape)


def _plain_linear8(s):
    x, w, b, g = s["x"], s["w"], s["b"], s["g"]
    dt = x.dtype
    xf, wf, gf = x.float(), w.float(), g.float()
    wq = _plain_q(wf, square=True)
    y = _plain_q(xf) @ wq.t()
    if b is not None:
        y = y + b.float()
    dx = _plain_q(gf) @ wq
    # the weight gradient contracts over the tokens: its operands are quantised along them
    dw = _plain_q(gf.t().contiguous()) @ _plain_q(xf.t().contiguous()).t()
    out = [y.to(dt), dx.to(dt), dw.to(dt)]
    if b is not None:
        out.append(gf.sum(0, dtype=torch.float64).to(dt))
    return out


def _plain_eval(s):
    x, (q, e), b, case = s["x"], s["w"], s["b"], s["case"]
    y = _plain_q(x.float()) @ _plain_values(q, e, case["fout"], case["fin"]).t()
    if b is not None:
        y = y + b.float()
    return [y.to(x.dtype)]


def _plain_act8(s):
    x, g = s["x"], s["g"]
    xf, gf = x.float(), g.float()
    if s["case"]["act"] == "relu":
        on = xf > 0
        return [(xf * on).to(x.dtype), (gf * on).to(x.dtype)]
    y = xf * 0.5 * (1.0 + torch.erf(xf * 0.7071067811865476))
    # blocks of 128 consecutive elements in memory
    h = _plain_q(xf.reshape(1, -1)).reshape(xf.shape)
    slope = 0.5 * (1.0 + torch.erf(h * 0.7071067811865476)) + h * torch.exp(-0.5 * h * h) * 0.3989422804014327
    return [y.to(x.dtype), (gf * slope).to(x.dtype)]


def _plain_norm8(s):
    x, w, b, g = s["x"], s["w"], s["b"], s["g"]
    xf, wf, gf = x.float(), w.float(), g.float()
    mean = xf.mean(1, keepdim=True)
    rstd = torch.rsqrt(((xf - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    y = (xf - mean) * rstd * wf
    if b is not None:
        y = y + b.float()
    z = (_plain_q(xf) - mean) * rstd            # the normalised rows as the backward pass sees them
    gw = gf * wf
    dx = rstd * (gw - gw.mean(1, keepdim=True) - z * (gw * z).mean(1, keepdim=True))
    out = [y.to(x.dtype), dx.to(x.dtype), (gf * z).sum(0, dtype=torch.float64).to(x.dtype)]
    if b is not None:
        out.append(gf.sum(0, dtype=torch.float64).to(x.dtype))
    return out


# ---- one pass -----------------------------------------------------------------------------------------
def _own(s):
    import hap_b200
    op = s["case"]["op"]
    if op == "linear8_eval":
        with torch.no_grad():
            return [hap_b200.linear8(s["x"], s["w"], s["b"])]
    if op == "linear8":
        y = hap_b200.linear8(s["x"], s["w"], s["b"])
        leaves = [s["x"], s["w"]]
    elif op == "act8":
        y = hap_b200.dropout.act_dropout8(s["x"], s["case"]["act"], 0.0)
        leaves = [s["x"]]
    else:
        y = hap_b200.layer_norm8(s["x"], (s["case"]["cols"],), s["w"], s["b"], 1e-5)
        leaves = [s["x"], s["w"]]
    if s.get("b") is not None:
        leaves.append(s["b"])
    return [y.detach(), *torch.autograd.grad(y, leaves, s["g"])]


def run(state):
    if own:
        return _own(state)
    return {"linear8": _plain_linear8, "linear8_eval": _plain_eval, "act8": _plain_act8, "norm8": _plain_norm8}[state["case"]["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------
def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear8":
        t, i, o = case["tokens"], case["fin"], case["fout"]
        # x, w, g read; y, dx, dw written; bias and its gradient; three products
        return {"bytes": es * (2 * t * i + 2 * t * o + 2 * i * o + (2 * o if case["bias"] else 0)), "flops": 6 * t * i * o}
    if case["op"] == "linear8_eval":
        t, i, o = case["tokens"], case["fin"], case["fout"]
        scales = 4 * math.ceil(i / BLOCK) * math.ceil(o / BLOCK)
        return {"bytes": es * (t * i + t * o + (o if case["bias"] else 0)) + i * o + scales, "flops": 2 * t * i * o}
    n = case["rows"] * case["cols"]
    if case["op"] == "act8":
        return {"bytes": 4 * es * n, "flops": (30 if case["act"] == "gelu" else 2) * n}
    return {"bytes": 4 * es * n + es * case["cols"] * (4 if case["bias"] else 2), "flops": 20 * n}


# ---- the definition in 64 bits --------------------------------------------------------------------------
def _exact_round(v):
    """v (64 bits) to the nearest e4m3 number, ties to even: three fraction bits, exponents from -6 up."""
    _, ex = torch.frexp(v)                                   # |v| = m 2^ex, m in [0.5, 1)
    step = torch.ldexp(torch.ones_like(v), (ex - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def _exact_along(x, dim):
    """Blocks of 128 along `dim`."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[dim], BLOCK):
        part = x.narrow(dim, lo, min(BLOCK, x.shape[dim] - lo))
        out.narrow(dim, lo, part.shape[dim]).copy_(_exact_block(part, part.abs().amax(dim, keepdim=True)))
    return out


def _exact_block(part, big):
    # the smallest e with big <= 448 * 2^e, at least -126
    e = torch.ceil(torch.log2(torch.where(big > 0, big, torch.full_like(big, 448.0)) / 448.0))
    e = torch.where(big > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where(big <= 448.0 * torch.exp2(e - 1), torch.where(big > 0, e - 1, e), e).clamp(min=-126.0)
    s = torch.exp2(e)
    return _exact_round(part / s) * s


def _exact_square(w):
    out = torch.empty_like(w)
    for r in range(0, w.shape[0], BLOCK):
        rows = w[r:r + BLOCK]
        for c in range(0, w.shape[1], BLOCK):
            part = rows[:, c:c + BLOCK]
            out[r:r + BLOCK, c:c + BLOCK] = _exact_block(part, part.abs().amax().reshape(1, 1))
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    x, g, b = s["x"].double(), s.get("g"), s.get("b")
    g = None if g is None else g.double()
    b = None if b is None else b.double()
    if case["op"] == "linear8":
        w = _exact_square(s["w"].double())
        y = _exact_along(x, 1) @ w.t()
        out = [y if b is None else y + b, _exact_along(g, 1) @ w, _exact_along(g, 0).t() @ _exact_along(x, 0)]
        return out + ([] if b is None else [g.sum(0)])
    if case["op"] == "linear8_eval":
        q, e = s["w"]
        w = (q.double() * torch.exp2(e.double())).reshape(-1, q.shape[2] * BLOCK)[:case["fout"], :case["fin"]]
        y = _exact_along(x, 1) @ w.t()
        return [y if b is None else y + b]
    if case["op"] == "act8":
        if case["act"] == "relu":
            return [x.clamp(min=0), torch.where(x > 0, g, torch.zeros_like(g))]
        n = x.numel()
        flat = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
        flat[:n] = x.reshape(-1)
        rows = flat.reshape(-1, BLOCK)
        h = _exact_block(rows, rows.abs().amax(1, keepdim=True)).reshape(-1)[:n].reshape(x.shape)
        phi = lambda t: 0.5 * torch.special.erfc(-t / math.sqrt(2.0))
        return [x * phi(x), g * (phi(h) + h * torch.exp(-h * h / 2) / math.sqrt(2.0 * math.pi))]
    w = s["w"].double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5)
    y = (x - mean) * rstd * w
    z = (_exact_along(x, 1) - mean) * rstd
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - z * (gw * z).mean(1, keepdim=True))
    out = [y if b is None else y + b, dx, (g * z).sum(0)]
    return out + ([] if b is None else [g.sum(0)])
