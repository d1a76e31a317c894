"""The 8-bit operators against oracle/block8_math.py (float64).

Tolerances.  Quantised values and scales are exact: scaling by a power of two rounds nothing, so 32 and 64 bits round to
the same e4m3 number.  A float32 sum of n terms in any order, each addition off by at most 2^-23 (rounded or cut), is
off by at most n 2^-23 times the sum of magnitudes; joining blocks with their scales adds two roundings.  The result is
then rounded once: half a step, eps / 2 of the value."""
import pytest
import torch

from oracle import block8_math as B

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, slack):
    """|got - want| <= slack + half a rounding step of got's type (and the smallest normal number)."""
    g, want = got.detach().cpu().double(), want.double()
    bound = slack + half_step(got.dtype) * (want.abs() + slack) + torch.finfo(got.dtype).tiny
    worst = ((g - want).abs() / bound).max() if g.numel() else torch.tensor(0.0)
    assert g.shape == want.shape and bool(((g - want).abs() <= bound).all()), f"off by {float(worst):.2f} of the bound"


def sum_slack(magnitudes, n):
    return magnitudes * (n + 4) * 2.0 ** -23


def per_row(scales, rows):
    """The oracle's scales [column block, row or row block] as (rows, column blocks)."""
    return (scales if scales.shape[1] == rows else scales.repeat_interleave(128, 1)[:, :rows]).t()


# ---- quantiser ----------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 128), (3, 129), (128, 128), (129, 127), (300, 515), (17, 1000), (257, 64), (1000, 33)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_is_exact(dtype, shape):
    from hap_b200 import block8
    x = (torch.randn(shape, generator=gen(sum(shape))) * torch.exp(2 * torch.randn(shape[0], 1, generator=gen(1)))).to(dtype)
    x[shape[0] // 2] = 0
    rows, cols = block8.quantize(x.to(DEV), rows=True, columns=True)
    sq = block8.quantize_weight(x.to(DEV), transposed=True)
    for got, want in ((rows, B.quantize(x)), (cols, B.quantize(x.t())), (sq, B.quantize(x, True)), (sq.transposed, B.quantize(x.t(), True))):
        values, scales = want
        assert torch.equal(got.dequantize(F32).cpu().double(), values)
        assert torch.equal(got.dequantize(BF).cpu().double(), values)
        assert torch.equal(got.scale_matrix().cpu().double(), per_row(scales, got.rows))
    # one form at a time gives the same
    assert torch.equal(block8.quantize(x.to(DEV)).dequantize(), rows.dequantize())
    assert torch.equal(block8.quantize(x.to(DEV), rows=False, columns=True).dequantize(), cols.dequantize())
    assert torch.equal(block8.quantize_weight(x.to(DEV)).dequantize(), sq.dequantize())


def test_quantize_special_values():
    from hap_b200 import block8
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(8, 256)
    x[0, :4] = torch.tensor([448.0, -448.0, 447.0, 1.0])
    x[1, :4] = torch.tensor([448.1, 2.0 ** -9, -0.0, 3.0])
    x[2, 0], x[2, 1], x[2, 200] = nan, 5.0, 7.0
    x[3, 0], x[3, 1], x[3, 2] = inf, -inf, 3.0
    x[4] = nan
    x[5, :3] = torch.tensor([1e-45, 1e-40, 2e-38])
    x[6, :3] = torch.tensor([3.3e38, -1e30, 1e38])
    x[7, 130] = 1.1754944e-38
    rows, cols = block8.quantize(x.to(DEV), rows=True, columns=True)
    for got, (values, scales) in ((rows, B.quantize(x)), (cols, B.quantize(x.t())), (block8.quantize_weight(x.to(DEV)), B.quantize(x, True))):
        # dequantize rounds to float32: 3.3e38 / 2^120 = 248.3 is nearest to 256 on its grid (steps of 16), and 256 * 2^120 = 2^128
        # is above float32's largest number, an infinity there
        torch.testing.assert_close(got.dequantize().cpu(), values.float(), rtol=0, atol=0, equal_nan=True)
        assert torch.equal(got.scale_matrix().cpu().double(), per_row(scales, got.rows))
    assert torch.equal(torch.isnan(rows.dequantize().cpu()), ~torch.isfinite(x))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_strided_and_offset_inputs(dtype):
    from hap_b200 import block8
    base = torch.randn(70, 301, generator=gen(5)).to(dtype).to(DEV)
    for x in (base[:, :200], base[3:, 1:270], base.t(), base[::2, 5:9], base[:1, 7:8]):
        want = B.quantize(x.cpu())[0]
        assert torch.equal(block8.quantize(x).dequantize().cpu().double(), want)
        assert torch.equal(block8.quantize(x, rows=False, columns=True).dequantize().cpu().double(), B.quantize(x.cpu().t())[0])
    empty = block8.quantize(torch.empty(0, 40, dtype=dtype, device=DEV))
    assert empty.shape == (0, 40) and empty.dequantize().shape == (0, 40)


# ---- product ------------------------------------------------------------------------------------------
PRODUCTS = [(1, 1, 1), (1, 768, 768), (3, 5, 129), (64, 256, 128), (127, 129, 255), (128, 128, 128), (129, 300, 1000), (300, 1237, 77),
            (1000, 640, 513), (513, 264, 2048), (40, 2304, 1024)]


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_matmul(out, square, m, n, k):
    from hap_b200 import block8
    a = torch.randn(m, k, generator=gen(m)) * torch.exp(torch.randn(m, 1, generator=gen(2)))
    b = torch.randn(n, k, generator=gen(n)) * torch.exp(torch.randn(n, 1, generator=gen(3)))
    bias = torch.randn(n, generator=gen(4)).to(out)
    aq, bq = block8.quantize(a.to(DEV)), (block8.quantize_weight if square else block8.quantize)(b.to(DEV))
    av, bv = B.fast_rows(a), B.quantize(b, square)[0]
    want, size = av @ bv.t(), av.abs() @ bv.abs().t()
    close(block8.matmul(aq, bq, None, out), want, sum_slack(size, k))
    got = block8.matmul(aq, bq, bias.to(DEV), out)
    close(got, want + bias.double(), sum_slack(size + bias.double().abs(), k + 1))
    assert torch.equal(got, block8.matmul(aq, bq, bias.to(DEV), out))          # the same bits every time


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("m,n,k", [(2600, 1000, 16384), (2305, 513, 16389), (40000, 300, 1000), (4096, 1024, 8192), (513, 2049, 2000), (8200, 1027, 4096)])
def test_matmul_of_long_operands_is_exact(out, m, n, k):
    """Whole numbers up to 6 quantise without error and their sums stay below 2^24: every order of addition gives the same."""
    from hap_b200 import block8
    a = torch.randint(-6, 7, (m, k), device=DEV, dtype=torch.int8).float()
    b = torch.randint(-6, 7, (n, k), device=DEV, dtype=torch.int8).float()
    bias = torch.randint(-500, 501, (n,), device=DEV).to(out)
    want = (a.double() @ b.double().t() + bias.double()).to(out)
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(block8.matmul(block8.quantize(a), block8.quantize(b), bias, out), want)


@pytest.mark.parametrize("m", [100, 300])
def test_long_float32_sums_do_not_drift(m):
    """Positive terms, so that every step that cuts instead of rounding errs in the same direction.  Accumulators run over
    512 terms (16 steps of 32, each off by 2^-22 of the sum at most: one cut where the terms are aligned, one of the
    result); their sums are added rounding to nearest, 2^-24 each."""
    from hap_b200 import block8
    k = 16384
    a, b = (block8.quantize(torch.rand(rows, k, generator=gen(rows)).to(DEV) + 0.1) for rows in (m, 48))
    want = a.dequantize().double() @ b.dequantize().double().t()
    got = block8.matmul(a, b, None, F32).double()
    assert float(((got - want).abs() / want).max()) <= 16 * 2.0 ** -22 + k / 512 * 2.0 ** -24


def test_float32_weight_gradient_over_many_tokens():
    """The same bound through linear8's backward pass."""
    import hap_b200
    from hap_b200 import block8
    t = 16384
    x, g = (torch.rand(t, n, generator=gen(n)).to(DEV) + 0.1 for n in (64, 300))
    w = leaf(torch.rand(300, 64, generator=gen(1)))
    (dw,) = torch.autograd.grad(hap_b200.linear8(x, w), w, g)
    want = block8.quantize(g, False, True).dequantize().double() @ block8.quantize(x, False, True).dequantize().double().t()
    assert float(((dw.double() - want).abs() / want).max()) <= 16 * 2.0 ** -22 + t / 512 * 2.0 ** -24


def test_matmul_of_integers_is_exact_and_nan_stays_in_its_row():
    from hap_b200 import block8
    a = torch.randint(-8, 9, (200, 384), generator=gen(0)).float()
    b = torch.randint(-8, 9, (150, 384), generator=gen(1)).float()
    got = block8.matmul(block8.quantize(a.to(DEV)), block8.quantize(b.to(DEV)), None, F32).cpu()
    assert torch.equal(got, a @ b.t())
    a[17, 200] = float("nan")
    got = block8.matmul(block8.quantize(a.to(DEV)), block8.quantize_weight(b.to(DEV)), None, F32).cpu()
    assert bool(torch.isnan(got[17]).all()) and int(torch.isnan(got).sum()) == 150


# ---- linear8 ------------------------------------------------------------------------------------------
LINEARS = [(1, 16, 24), (1, 1, 1), (7, 130, 129), (38, 1024, 512), (256, 768, 768), (515, 1000, 237), (2048, 96, 640)]


def linear_inputs(rows, fin, fout, dtype):
    x = (torch.randn(rows, fin, generator=gen(rows)) * torch.exp(0.7 * torch.randn(fin, generator=gen(1)))).to(dtype)
    w = (torch.randn(fout, fin, generator=gen(fin)) * fin ** -0.5).to(dtype)
    b = torch.randn(fout, generator=gen(2)).to(dtype)
    g = (torch.randn(rows, fout, generator=gen(3)) * torch.exp(torch.randn(rows, 1, generator=gen(4))) * 1e-3).to(dtype)
    return x, w, b, g


def leaf(t, dev=DEV):
    return t.detach().to(dev).requires_grad_(True)


def check_linear(got, want, rows, fin, fout):
    for t, (v, size), n in zip(got, want, (fin + 1, fout, rows, rows)):
        if t is not None:
            close(t, v, sum_slack(size, n))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,fin,fout", LINEARS)
@pytest.mark.parametrize("bias", [True, False])
def test_linear8_forward_backward(dtype, rows, fin, fout, bias):
    import hap_b200
    x, w, b, g = linear_inputs(rows, fin, fout, dtype)
    b = b if bias else None
    want = B.linear8(x, w, b, g)
    xg, wg, bg = leaf(x), leaf(w), (leaf(b) if bias else None)
    y = hap_b200.linear8(xg, wg, bg)
    assert y.dtype == dtype and y.shape == (rows, fout)
    y.backward(g.to(DEV))
    check_linear((y, xg.grad, wg.grad, bg.grad if bias else None), want, rows, fin, fout)


def test_linear8_gradients_against_differences():
    """On operands that 8 bits hold exactly the operator is bilinear: differences of the loss are its gradients."""
    import hap_b200
    ints = lambda *s, seed: torch.randint(-3, 4, s, generator=gen(seed)).float()
    x, w, b, g = ints(150, 200, seed=0), ints(130, 200, seed=1), ints(130, seed=2), ints(150, 130, seed=3)
    xg, wg, bg = leaf(x), leaf(w), leaf(b)
    loss = lambda a, c, d: float((hap_b200.linear8(a, c, d).detach().double() * g.to(DEV).double()).sum())
    hap_b200.linear8(xg, wg, bg).backward(g.to(DEV))
    base = loss(xg, wg, bg)
    for i, (t, grad) in enumerate(((x, xg.grad), (w, wg.grad), (b, bg.grad))):
        d = ints(*t.shape, seed=10 + i)
        moved = [v.to(DEV) for v in (x, w, b)]
        moved[i] = (t + d).to(DEV)
        assert loss(*moved) - base == float((grad.cpu().double() * d.double()).sum())


def test_linear8_layouts_and_partial_gradients():
    import hap_b200
    x, w, b, g = linear_inputs(24 * 9, 136, 200, BF)
    want = B.linear8(x, w, b, g)
    # sequence-first memory seen batch-first, a column-major weight, a strided gradient
    x3 = x.view(24, 9, 136).transpose(0, 1)
    xg, wg, bg = leaf(x3), leaf(w.t().contiguous().t()), leaf(b)
    y = hap_b200.linear8(xg, wg, bg)
    assert y.shape == (9, 24, 200)
    y.backward(g.view(24, 9, 200).transpose(0, 1).to(DEV))
    xb, gb = x3.reshape(-1, 136), g.view(24, 9, 200).transpose(0, 1).reshape(-1, 200)
    check_linear((y.reshape(-1, 200), xg.grad.reshape(-1, 136), wg.grad, bg.grad), B.linear8(xb, w, b, gb), 216, 136, 200)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True)):
        leaves = [t.to(DEV).requires_grad_(n) for t, n in zip((x, w, b), needs)]
        y = hap_b200.linear8(*leaves)
        y.backward(g.to(DEV))
        check_linear([y] + [t.grad for t in leaves], want, 216, 136, 200)
        assert [t.grad is not None for t in leaves] == list(needs)
    # a vector, and an expanded gradient (the gradient of a sum)
    xv = leaf(x[0])
    yv = hap_b200.linear8(xv, w.to(DEV), b.to(DEV))
    assert yv.shape == (200,)
    yv.sum().backward()
    check_linear((yv[None], xv.grad[None]), B.linear8(x[:1], w, b, torch.ones(1, 200))[:2], 1, 136, 200)


def test_linear8_without_tokens():
    import hap_b200
    x, w, b = leaf(torch.empty(0, 3, 40, dtype=BF)), leaf(torch.ones(24, 40, dtype=BF)), leaf(torch.ones(24, dtype=BF))
    y = hap_b200.linear8(x, w, b)
    assert y.shape == (0, 3, 24)
    y.sum().backward()
    assert x.grad.shape == x.shape and float(w.grad.abs().max()) == 0.0 and float(b.grad.abs().max()) == 0.0


def test_linear8_prepared_weight():
    import hap_b200
    from hap_b200 import block8
    x, w, b, g = linear_inputs(77, 300, 130, BF)
    want = B.linear8(x, w, b, g)
    w8 = block8.quantize_weight(w.to(DEV))
    with torch.no_grad():
        y = hap_b200.linear8(x.to(DEV), w8, b.to(DEV))
    check_linear((y,), want, 77, 300, 130)
    assert torch.equal(y, hap_b200.linear8(x.to(DEV), w.to(DEV), b.to(DEV)))
    with pytest.raises(ValueError, match="transposed"):
        hap_b200.linear8(leaf(x), w8, b.to(DEV))
    xg, bg = leaf(x), leaf(b)
    hap_b200.linear8(xg, block8.quantize_weight(w.to(DEV), transposed=True), bg).backward(g.to(DEV))
    check_linear((y, xg.grad, None, bg.grad), want, 77, 300, 130)
    bg = leaf(b)
    hap_b200.linear8(x.to(DEV), w8, bg).backward(g.to(DEV))                  # only the bias learns
    check_linear((None, None, None, bg.grad), want, 77, 300, 130)
    # a weight in 1 x 128 blocks serves too
    w1 = block8.quantize(w.to(DEV))
    y1 = hap_b200.linear8(x.to(DEV), w1)
    xv, wv = B.fast_rows(x), B.fast_rows(w)
    close(y1, xv @ wv.t(), sum_slack(xv.abs() @ wv.abs().t(), 300))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,fin,fout", [(1, 768, 2304), (1, 1, 1), (2, 130, 77), (3, 5000, 64), (8, 1000, 129), (8, 4096, 40), (9, 768, 768), (33, 129, 300),
                                           (64, 1024, 512), (65, 100, 200), (100, 640, 33), (128, 513, 264), (129, 256, 192), (40, 8192, 64), (20, 8192, 64), (1, 25000, 40)])
def test_linear8_few_tokens_prepared_weight(dtype, rows, fin, fout):
    """Every way the tokens reach the product (a warp per output, converted inside the product, quantised before it) gives
    the result of the plain call; rows with infinities and NaN, strided rows."""
    import hap_b200
    from hap_b200 import block8
    x, w, b, g = linear_inputs(rows, fin, fout, dtype)
    want = B.linear8(x, w, b, g)[:1]
    w8 = block8.quantize_weight(w.to(DEV))
    y = hap_b200.linear8(x.to(DEV), w8, b.to(DEV))
    check_linear((y,), want, rows, fin, fout)
    wide = torch.zeros(rows, 2 * fin + 3, dtype=dtype, device=DEV)
    wide[:, 1:1 + fin] = x.to(DEV)
    assert torch.equal(hap_b200.linear8(wide[:, 1:1 + fin], w8, b.to(DEV)), y)
    x[rows // 2, fin // 2] = float("inf")
    x[0, 0] = float("nan")
    y = hap_b200.linear8(x.to(DEV), w8).cpu()
    bad = torch.isnan(x).any(1) | torch.isinf(x).any(1)
    assert bool(torch.isnan(y[bad]).all()) and bool(torch.isfinite(y[~bad]).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [3, 4, 7, 32])
def test_linear8_few_tokens_wide_weight(dtype, rows):
    """Several tiles per thread block, whose first operand is converted far quicker than the weight arrives: the ring of
    stages goes round often, and every call gives the same bits."""
    import hap_b200
    from hap_b200 import block8
    x = torch.randint(-6, 7, (rows, 768), device=DEV).to(dtype)
    w = torch.randint(-6, 7, (33280, 768), device=DEV).float()
    want = (x.double() @ w.double().t()).to(dtype)
    w8 = block8.quantize_weight(w)
    flush = torch.empty(256 << 20, device=DEV, dtype=torch.uint8)
    with torch.no_grad():
        for i in range(60):
            if i % 2:
                flush.zero_()
            assert torch.equal(hap_b200.linear8(x, w8), want)


def test_linear8_uses_the_same_leaf_twice_and_keeps_its_graph():
    import hap_b200
    x, w, b, g = linear_inputs(60, 96, 96, F32)
    xg, wg = leaf(x), leaf(w)
    y = hap_b200.linear8(hap_b200.linear8(xg, wg), wg)
    first = torch.autograd.grad(y, [xg, wg], g.to(DEV), retain_graph=True)
    again = torch.autograd.grad(y, [xg, wg], g.to(DEV))
    for a, c in zip(first, again):
        assert torch.equal(a, c) and float(a.abs().max()) > 0
    mid = hap_b200.linear8(xg.detach(), wg.detach()).requires_grad_(True)
    w1, w2 = leaf(w), leaf(w)
    dmid, d2 = torch.autograd.grad(hap_b200.linear8(mid, w2), [mid, w2], g.to(DEV))
    (d1,) = torch.autograd.grad(hap_b200.linear8(xg.detach(), w1), [w1], dmid)
    assert torch.equal(first[1], d1 + d2) or torch.equal(first[1], d2 + d1)


def test_linear8_large_offsets():
    """An output of more than 2^31 elements: the last rows and columns are where they belong."""
    import hap_b200
    from hap_b200 import block8
    rows, fin, fout = 70000, 16, 33000
    x = torch.zeros(rows, fin, dtype=BF, device=DEV)
    w = torch.zeros(fout, fin, dtype=BF, device=DEV)
    x[-300:] = torch.randn(300, fin, generator=gen(0)).to(BF).to(DEV)
    w[-200:] = torch.randn(200, fin, generator=gen(1)).to(BF).to(DEV)
    y = hap_b200.linear8(x, block8.quantize_weight(w))
    assert y.numel() > 2 ** 31
    xv, wv = B.fast_rows(x[-300:].cpu()), B.quantize(w.cpu()[32640:], True)[0]           # from a whole block of 128 weight rows on
    close(y[-300:, 32640:], xv @ wv.t(), sum_slack(xv.abs() @ wv.abs().t(), fin))
    assert float(y[:-300].abs().max()) == 0.0


def test_linear8_refusals():
    import hap_b200
    from hap_b200 import block8
    x, w = torch.ones(4, 8, device=DEV), torch.ones(5, 8, device=DEV)
    for args, err in (((x.half(), w.half()), TypeError), ((x, w.to(BF)), TypeError), ((x, w[:, :7]), ValueError), ((x, w, w[0]), ValueError),
                      ((x, w, torch.ones(5, device=DEV, dtype=BF)), TypeError), ((x, w, torch.ones(5)), ValueError), ((x, w.cpu()), ValueError),
                      ((x, w[0]), ValueError), ((x[:, :0], w[:, :0]), ValueError), ((x, w[:0]), ValueError), ((x[0, 0], w), ValueError),
                      ((x, block8.quantize(w[:, :7])), ValueError)):
        with pytest.raises(err):
            hap_b200.linear8(*args)
    for bad in (x[0], x[:, :0]):
        with pytest.raises(ValueError):
            block8.quantize(bad)
    with pytest.raises(ValueError):
        block8.quantize(x[:0], rows=False, columns=True)
    with pytest.raises(ValueError):
        block8.quantize_weight(w[:0])
    y = hap_b200.linear8(leaf(x.cpu()), w)
    (dx,) = torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable, create_graph=True)
    assert not dx.requires_grad or dx.grad_fn is not None
    with pytest.raises(RuntimeError):
        dx.sum().backward()                                      # no second derivative: refused, not wrong


def saved_bytes(fn):
    total = 0

    def pack(t):
        nonlocal total
        total += t.numel() * t.element_size()
        return t
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        fn()
    return total


def test_what_is_kept_for_the_backward_pass():
    import hap_b200
    rows, fin, fout = 512, 1024, 256
    x, w = leaf(torch.randn(rows, fin).to(BF)), torch.randn(fout, fin).to(BF).to(DEV)
    n = rows * fin
    assert saved_bytes(lambda: hap_b200.linear8(x.detach(), leaf(w))) == n + n // 128                          # the input, 8 bits
    assert saved_bytes(lambda: hap_b200.linear8(x, w)) == fin * fout + fin * 4                  # the weight: out_features 256 are two blocks of four
    assert saved_bytes(lambda: hap_b200.dropout.act_dropout8(x, "gelu", 0.1)) == n + 4 * n // 128
    assert saved_bytes(lambda: hap_b200.dropout.act_dropout8(x, "relu", 0.1)) == n // 8
    assert saved_bytes(lambda: hap_b200.layer_norm8(x, (fin,))) == n + 4 * n // 128 + 8 * rows
    with torch.no_grad():
        assert saved_bytes(lambda: hap_b200.layer_norm8(x, (fin,))) == 0


# ---- activation ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1,), (3,), (128,), (129,), (5, 7, 33), (333, 515), (1000, 1024)])
@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_act_dropout8(dtype, shape, act, p):
    from hap_b200 import dropout as D
    x = (torch.randn(shape, generator=gen(len(shape))) * 2).to(dtype)
    g = torch.randn(shape, generator=gen(9)).to(dtype)
    D.manual_seed(5)
    D.advance()
    xg = leaf(x)
    y = D.act_dropout8(xg, act, p)
    k = (D.keep_mask(x.numel(), p, 1).cpu().double().view(shape) if p else torch.ones(shape, dtype=torch.float64)) / (1.0 - p)
    y.backward(g.to(DEV))
    v, h, gd = x.double(), B.runs(x), g.double()
    if act == "relu":
        close(y, v.clamp(min=0) * k, v.abs() * k * 2.0 ** -23)
        close(xg.grad, torch.where(v > 0, gd, torch.zeros_like(gd)) * k, gd.abs() * k * 2.0 ** -23)
        return
    # erfc amplifies the rounding of its argument by 2 z^2 = v^2; expf is off by 2 + 1.2 |v^2 / 2| steps
    close(y, B.gelu(v) * k, B.gelu(v).abs() * k * (2 * v * v + 32) * 2.0 ** -24)
    size = 0.5 * torch.special.erfc(-h / 2 ** 0.5) + h.abs() * torch.exp(-h * h / 2) * 0.4
    close(xg.grad, gd * k * B.gelu_slope(h), gd.abs() * k * size * (2 * h * h + 32) * 2.0 ** -23)


def test_act_dropout8_layouts_and_values():
    from hap_b200 import dropout as D
    # a permuted dense tensor is walked in memory order and keeps its strides; the gradient arrives in another layout
    x = torch.randn(6, 10, 96, generator=gen(0)).to(BF)
    xg = x.to(DEV).permute(1, 0, 2).requires_grad_(True)
    y = D.act_dropout8(xg, "gelu", 0.0)
    assert y.stride() == xg.stride()
    y.backward(torch.ones(10, 6, 96, dtype=BF, device=DEV))
    close(xg.grad, B.gelu_slope(B.runs(x)).permute(1, 0, 2), torch.full((10, 6, 96), 1e-5, dtype=torch.float64))
    # views that are not dense are copied; infinities and NaN
    v = torch.tensor([float("inf"), -float("inf"), float("nan"), 3.0, -3.0, 0.0, -0.0, 1e-30])
    xs = torch.stack([v, torch.zeros(8)], 1)[:, 0].to(DEV).requires_grad_(True)
    for act in ("relu", "gelu"):
        y = D.act_dropout8(xs, act, 0.0)
        want = torch.relu(v) if act == "relu" else B.gelu(v.double())      # x Phi(x): inf at inf, NaN at -inf
        assert torch.equal(torch.isnan(y).cpu(), torch.isnan(want)) and float(y.detach()[0]) == float("inf")
        (d,) = torch.autograd.grad(y, xs, torch.ones_like(y))
        if act == "relu":
            assert torch.equal(d.cpu(), (v > 0).float())
        else:
            assert bool(torch.isfinite(d[3:]).all()) and bool(torch.isnan(d[:3]).all())
    assert D.act_dropout8(torch.empty(0, 5, device=DEV), "gelu", 0.0).shape == (0, 5)
    with pytest.raises(ValueError, match="relu"):
        D.act_dropout8(xs, "silu", 0.0)
    with pytest.raises(ValueError, match="p must"):
        D.act_dropout8(xs, "relu", 1.0)
    with pytest.raises(TypeError):
        D.act_dropout8(xs.half(), "relu", 0.0)


def test_gelu_gradient_against_differences():
    """At inputs that 8 bits hold exactly the kept input is the input: the gradient is the function's own."""
    from hap_b200 import dropout as D
    x = torch.arange(-64, 64).float() / 16 * 1.0
    x = B.runs(x).float()
    xg = leaf(x)
    D.act_dropout8(xg, "gelu", 0.0).sum().backward()
    h = 1e-5
    diff = (B.gelu(x.double() + h) - B.gelu(x.double() - h)) / (2 * h)
    close(xg.grad, diff, torch.full((128,), 1e-6, dtype=torch.float64))      # h^2 / 6 gelu''' + the float32 bound of the slope


# ---- layer_norm8 --------------------------------------------------------------------------------------
def norm_bounds(x, w, b, g, kept, want, rows):
    """Bounds on y, dx, dw, db: a lane adds E / 32 terms and 5 shuffles; mean and variance carry that many roundings."""
    x, g = x.double(), g.double()
    E = x.shape[1]
    n = E / 32 + 16
    w1 = torch.ones(E, dtype=torch.float64) if w is None else w.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    za = (torch.maximum(x.abs(), kept.abs()) + x.abs().mean(1, keepdim=True)) * rstd
    gw = (g * w1).abs()
    slack = n * 2.0 ** -21
    return (slack * za * (1 + za.square().mean(1, keepdim=True).sqrt()) * w1.abs() + (0 if b is None else b.double().abs() * 2.0 ** -23),
            slack * rstd * (gw + gw.mean(1, keepdim=True) + za * (gw * za).mean(1, keepdim=True)),
            (g.abs() * za).sum(0) * (slack + rows * 2.0 ** -23), g.abs().sum(0) * rows * 2.0 ** -23)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,E", [(1, 1), (1, 8), (5, 33), (3, 129), (591, 768), (130, 2048), (64, 1288), (33, 5000), (200, 127), (2000, 256), (70, 400),
                                    (9, 1000), (40, 4096), (5, 8192), (70, 9001), (3, 20000)])
@pytest.mark.parametrize("affine", ["both", "weight", "none"])
def test_layer_norm8(dtype, rows, E, affine):
    import hap_b200
    x = (torch.randn(rows, E, generator=gen(rows + E)) * 2 + 0.25).to(dtype)
    w = (torch.rand(E, generator=gen(1)) + 0.5).to(dtype) if affine != "none" else None
    b = torch.randn(E, generator=gen(2)).to(dtype) if affine == "both" else None
    g = torch.randn(rows, E, generator=gen(3)).to(dtype)
    kept = B.fast_rows(x)
    want = B.layer_norm8(x, w, b, g)
    bounds = norm_bounds(x, w, b, g, kept, want, rows)
    xg, wg, bg = leaf(x), leaf(w) if w is not None else None, leaf(b) if b is not None else None
    y = hap_b200.layer_norm8(xg, (E,), wg, bg, 1e-5)
    y.backward(g.to(DEV))
    for got, v, bound in zip((y, xg.grad, wg.grad if w is not None else None, bg.grad if b is not None else None), want, bounds):
        if got is not None:
            close(got, v, bound)
    with torch.no_grad():
        assert torch.equal(y, hap_b200.layer_norm8(xg, E, wg, bg))
    again = leaf(x)
    hap_b200.layer_norm8(again, (E,), wg, bg).backward(g.to(DEV))
    assert torch.equal(again.grad, xg.grad)


def test_layer_norm8_gradient_against_differences():
    import hap_b200
    x = B.fast_rows(torch.randn(4, 200, generator=gen(0)))            # held exactly by 8 bits
    w, g = torch.rand(200, generator=gen(1)).double() + 0.5, torch.randn(4, 200, generator=gen(2)).double()
    d = torch.randn(4, 200, generator=gen(3)).double()
    xg, wg = leaf(x.float()), leaf(w.float())
    hap_b200.layer_norm8(xg, 200, wg).backward(g.float().to(DEV))
    h = 1e-5
    f = lambda v, u: float((B.layer_norm8(v, u, None, g.float())[0] * g.float().double()).sum())
    diff = (f(x + h * d, w.float().double()) - f(x - h * d, w.float().double())) / (2 * h)
    got = float((xg.grad.cpu().double() * d).sum())
    assert abs(got - diff) <= 1e-5 * float((xg.grad.cpu().double() * d).abs().sum())
    diff = (f(x, w.float().double() + h * d[0]) - f(x, w.float().double() - h * d[0])) / (2 * h)
    assert abs(float((wg.grad.cpu().double() * d[0]).sum()) - diff) <= 1e-5 * float((wg.grad.cpu().double() * d[0]).abs().sum())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(40, 3, 768), (9, 2, 65), (5, 2, 3000), (3, 2, 9001)])
def test_layer_norm_fork8(dtype, shape):
    from hap_b200.norm import layer_norm8, layer_norm_fork8
    E, rows = shape[-1], shape[0] * shape[1]
    x = torch.randn(shape, generator=gen(0)).to(dtype)
    w, b = (torch.rand(E, generator=gen(1)) + 0.5).to(dtype), torch.randn(E, generator=gen(2)).to(dtype)
    dres, dy = torch.randn(shape, generator=gen(3)).to(dtype), torch.randn(shape, generator=gen(4)).to(dtype)
    x2, g2 = x.view(rows, E), dy.view(rows, E)
    want = B.layer_norm8(x2, w, b, g2, add=dres.view(rows, E))
    bounds = norm_bounds(x2, w, b, g2, B.fast_rows(x2), want, rows)
    for view in (lambda t: t, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):        # dense and permuted
        xg, wg, bg = leaf(view(x)), leaf(w), leaf(b)
        res, y = layer_norm_fork8(xg, (E,), wg, bg)
        assert res.data_ptr() == xg.data_ptr() and torch.equal(y, layer_norm8(xg.detach(), (E,), wg.detach(), bg.detach()))
        torch.autograd.backward([res, y], [view(dres).to(DEV), view(dy).to(DEV)])
        close(xg.grad.reshape(rows, E), want[1], bounds[1] + dres.view(rows, E).double().abs() * 2.0 ** -23)
        close(wg.grad, want[2], bounds[2])
        close(bg.grad, want[3], bounds[3])
    xg = leaf(x)
    (layer_norm_fork8(xg, (E,), w.to(DEV))[0] * dres.to(DEV)).sum().backward()                   # only the residual path used
    assert torch.equal(xg.grad.cpu(), dres)
    xg = leaf(x)
    layer_norm_fork8(xg, (E,), w.to(DEV))[1].backward(dy.to(DEV))
    plain = leaf(x)
    layer_norm8(plain, (E,), w.to(DEV)).backward(dy.to(DEV))
    assert torch.equal(xg.grad, plain.grad)


def test_layer_norm8_refusals_and_empty():
    import hap_b200
    x = torch.ones(3, 4, 8, device=DEV)
    for args in ((x, (4, 8)), (x, (7,)), (x, (8,), torch.ones(7, device=DEV)), (x, (8,), torch.ones(8, device=DEV, dtype=BF)),
                 (x, (8,), None, torch.ones(8))):
        with pytest.raises(ValueError):
            hap_b200.layer_norm8(*args)
    with pytest.raises(TypeError):
        hap_b200.layer_norm8(x.half(), 8)
    e = leaf(torch.empty(0, 8))
    w = leaf(torch.ones(8))
    hap_b200.layer_norm8(e, 8, w).sum().backward()
    assert e.grad.shape == (0, 8) and torch.equal(w.grad.cpu(), torch.zeros(8))


# ---- together -----------------------------------------------------------------------------------------
def test_ffn_block_step_by_step():
    """x + dropout(W2 gelu(W1 layer_norm(x))) forward and backward: every operator is checked at the inputs and
    gradients it saw in the run."""
    import hap_b200
    from hap_b200 import dropout as D
    from hap_b200.norm import layer_norm_fork8
    rows, E, H = 333, 136, 520
    x = torch.randn(rows, E, generator=gen(0)).to(BF)
    P = [t.to(BF) for t in (torch.rand(E, generator=gen(1)) + 0.5, torch.randn(E, generator=gen(2)) * 0.1,
                            torch.randn(H, E, generator=gen(3)) * E ** -0.5, torch.randn(H, generator=gen(4)) * 0.1,
                            torch.randn(E, H, generator=gen(5)) * H ** -0.5, torch.randn(E, generator=gen(6)) * 0.1)]
    xg, p = leaf(x), [leaf(t) for t in P]
    D.manual_seed(11)
    D.advance()
    res, h = layer_norm_fork8(xg, (E,), p[0], p[1])
    u = hap_b200.linear8(h, p[2], p[3])
    a = D.act_dropout8(u, "gelu", 0.0)
    o = hap_b200.linear8(a, p[4], p[5])
    out = D.dropout_add(o, res, 0.1)
    for t in (res, h, u, a, o):
        t.retain_grad()
    g = torch.randn(rows, E, generator=gen(7)).to(BF)
    out.backward(g.to(DEV))
    c = lambda t: t.detach().cpu()
    check_linear((u, h.grad, p[2].grad, p[3].grad), B.linear8(c(h), P[2], P[3], c(u.grad)), rows, E, H)
    check_linear((o, a.grad, p[4].grad, p[5].grad), B.linear8(c(a), P[4], P[5], c(o.grad)), rows, H, E)
    slope = B.gelu_slope(B.runs(c(u)))
    close(u.grad, c(a.grad).double() * slope, c(a.grad).double().abs() * 1e-5)
    want = B.layer_norm8(x, P[0], P[1], c(h.grad), add=c(res.grad))
    bounds = norm_bounds(x, P[0], P[1], c(h.grad), B.fast_rows(x), want, rows)
    close(h, want[0], bounds[0])
    close(xg.grad, want[1], bounds[1] + c(res.grad).double().abs() * 2.0 ** -23)
    close(p[0].grad, want[2], bounds[2])


def lm_worker(layers=2, dtype=BF):
    import hap_b200
    from hap_b200 import fxpass, plan
    from hap_b200.spmd import ProcessWorker
    torch.manual_seed(3)
    model = plan.TransformerLM(vocab=520, d_model=128, nheads=2, d_ffn=264, nlayers=layers, seqlen=40).to(dtype).to(DEV)
    hap_b200.collectives.set_default_comm(hap_b200.single_comm(torch.device(DEV), stage_bytes=1 << 20, heap_bytes=8 << 20))
    graph = plan.emit_lm(model, "dp", [1.0], 0, 5, dropout_p=0.1)
    fxpass.fuse_elementwise(graph)
    fxpass.fuse_residual_norm(graph)
    changed = fxpass.use_block8(graph)
    assert changed == {"linear": 2 * layers + 1, "multi_head_attention_forward": layers, "act_dropout": layers, "layer_norm": 1,
                       "layer_norm_fork": 2 * layers}
    return model, ProcessWorker(torch.fx.GraphModule(model, graph), lr=1e-3)


def test_language_model_step_eager_and_captured():
    """The whole 8-bit program through the step driver; a step replayed from a CUDA graph gives the eager step's bits."""
    import hap_b200
    g = gen(0)
    batches = [(torch.randint(0, 520, (5, 40), generator=g).to(DEV), torch.randint(0, 520, (5, 40), generator=g).to(DEV)) for _ in range(3)]
    results = []
    for captured in (False, True):
        model, worker = lm_worker()
        step = worker.step
        if captured:
            start = [p.detach().clone() for p in model.parameters()]
            step = worker.capture(*batches[0])
            with torch.no_grad():
                for p, s in zip(model.parameters(), start):
                    p.copy_(s)
        hap_b200.dropout.manual_seed(1)
        results.append([float(step(*b)) for b in batches[:1]])
        assert all(torch.isfinite(p).all() for p in model.parameters())
        del step, worker
    assert results[0] == results[1]


def test_linear8_in_two_captured_graphs_and_on_other_streams():
    """Two graphs captured from the same operator replayed at the same time, and an eager call beside them, keep to
    their own memory."""
    import hap_b200
    x, w, b, g = (t.to(DEV) for t in linear_inputs(700, 520, 264, BF))
    xs = [x, x * 2]
    outs, graphs = [], []

    def step(v):
        lv, lw, lb = v.detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y = hap_b200.linear8(lv, lw, lb)
        return (y.detach(), *torch.autograd.grad(y, (lv, lw, lb), g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[t.clone() for t in step(v)] for v in xs]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for v in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(v))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        eager = step(x)
    torch.cuda.synchronize()
    for got, ref in ((outs[0], want[0]), (outs[1], want[1]), (eager, want[0])):
        for a, c in zip(got, ref):
            assert torch.equal(a, c)


def test_attention_projections_on_linear8():
    import hap_b200
    from hap_b200.attention import attention, multi_head_attention_forward8
    L, n, E, H = 20, 3, 128, 2
    x = torch.randn(L, n, E, generator=gen(0)).to(BF).to(DEV)
    iw, ib = (torch.randn(3 * E, E, generator=gen(1)) * E ** -0.5).to(BF).to(DEV), torch.randn(3 * E, generator=gen(2)).to(BF).to(DEV)
    ow, ob = (torch.randn(E, E, generator=gen(3)) * E ** -0.5).to(BF).to(DEV), torch.randn(E, generator=gen(4)).to(BF).to(DEV)
    out, weights = multi_head_attention_forward8(x, x, x, E, H, iw, ib, out_proj_weight=ow, out_proj_bias=ob, attn_mask="causal")
    want = hap_b200.linear8(attention(hap_b200.linear8(x, iw, ib), H, "causal"), ow, ob)
    assert weights is None and torch.equal(out, want)
    with pytest.raises(NotImplementedError):
        multi_head_attention_forward8(x, x.clone(), x, E, H, iw, ib, out_proj_weight=ow, out_proj_bias=ob)
