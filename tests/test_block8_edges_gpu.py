"""The 8-bit operators at the ends of what they accept: the largest extents, scales far apart, values near the largest
float32 number, NaN and infinities, forward-mode differentiation, operands that do not fit together; and whole steps
replayed from CUDA graphs."""
import pytest
import torch

from oracle import block8_math as B
from tests.test_block8_gpu import BF, DEV, F32, check_linear, close, gen, half_step, leaf, linear_inputs, lm_worker, norm_bounds, sum_slack

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """A kernel whose bounded wait ran out raises a flag; its output may look whole all the same."""
    import hap_b200
    yield
    hap_b200.linear_ops.gemm_status()


@pytest.mark.parametrize("rows", [1, 2])
def test_prepared_weight_with_the_most_output_features(rows):
    """out_features 2^31 - 256, where a row number plus the grid's stride is above 2^31 - 1.  in_features 1: y = x w."""
    import hap_b200
    from hap_b200 import block8
    n = 2 ** 31 - 256
    last = torch.arange(1, 9, dtype=F32)
    raw = torch.zeros(n, 16, dtype=torch.uint8, device=DEV)                                               # 34 GB
    raw[:, 0] = 0x38                                                                                      # 1.0
    raw[-8:, 0] = last.to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
    raw[2 ** 30, 0] = 0xC4                                                                                # -3.0
    scales = torch.full((-(-n // 128) * 512,), 127, dtype=torch.uint8, device=DEV)                        # 2^0 everywhere
    x = torch.tensor([[2.0], [-4.0]], dtype=BF, device=DEV)[:rows]
    y = hap_b200.linear8(x, block8.Block8(raw.view(torch.float8_e4m3fn), scales, n, 1))
    del raw, scales
    assert y.shape == (rows, n)
    for r in range(rows):
        xr = float(x[r, 0])
        assert torch.equal(y[r, -8:].float().cpu(), xr * last) and float(y[r, 2 ** 30]) == -3.0 * xr
        y[r, -8:] = y[r, 2 ** 30] = xr
        low, high = torch.aminmax(y[r])
        assert float(low) == float(high) == xr
    del y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 2, 3, 33, 200])
@pytest.mark.parametrize("ex,ew", [(-120, 120), (115, -110), (-118, 125), (100, -120), (-60, -60), (10, 100)])
def test_scales_far_apart(rows, ex, ew):
    """Either operand's scale alone takes the sums out of float32, both together do not: every path by which tokens reach a
    prepared weight multiplies them as one power of two."""
    import hap_b200
    from hap_b200 import block8
    k, n = 300, 40
    x, w = (torch.randint(-448, 449, shape, generator=gen(sum(shape))).double() / 64 for shape in ((rows, k), (n, k)))
    x, w = (x * 2.0 ** ex).float(), (w * 2.0 ** ew).float()                    # exact: 10 bits, normal numbers
    xv, wv = B.fast_rows(x), B.quantize(w, square=True)[0]
    y = hap_b200.linear8(x.to(DEV), block8.quantize_weight(w.to(DEV)))
    close(y, xv @ wv.t(), sum_slack(xv.abs() @ wv.abs().t(), k))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_gelu_gradient_of_the_largest_numbers(dtype):
    """From 248 * 2^120 on the kept value is 256 * 2^120, which float32 does not hold; the slope there is 1 (or 0) all the same."""
    from hap_b200 import dropout as D
    x = torch.tensor([3.2e38, 3.3e38, 3.38e38, torch.finfo(dtype).max, 1.0, 0.0, 3e37, 2.0 ** 111]).to(dtype).repeat(20)
    for sign in (1.0, -1.0):
        xg = (sign * x).to(DEV).requires_grad_(True)
        g = torch.full_like(x, 0.75)
        D.act_dropout8(xg, "gelu", 0.0).backward(g.to(DEV))
        close(xg.grad, 0.75 * B.gelu_slope(B.runs(sign * x)), torch.full(x.shape, 2.0 ** -20, dtype=torch.float64))


def test_replayed_steps_train_like_eager_ones():
    """Three steps of the 8-bit program, eager and replayed from a graph, from the same parameters and optimizer state: the
    losses, every updated parameter and both moments have the same bits."""
    import hap_b200
    g = gen(0)
    batches = [tuple(torch.randint(0, 520, (5, 40), generator=g).to(DEV) for _ in range(2)) for _ in range(3)]
    runs = []
    for captured in (False, False, True):
        model, worker = lm_worker()
        opt, step = worker.optimizer, worker.step
        state = [*model.parameters(), *opt.exp_avg, *opt.exp_avg_sq, opt.state]
        if captured:
            start = [t.detach().clone() for t in state]
            step = worker.capture(*batches[0])
            with torch.no_grad():
                for t, s in zip(state, start):
                    t.copy_(s)
        hap_b200.dropout.manual_seed(1)
        losses = [float(step(*b)) for b in batches]
        # every parameter had a gradient (a norm's weight of 1 may not move: a step of 1e-3 is below 2^-9, half its rounding)
        assert all(float(m.float().abs().max()) > 0 for m in opt.exp_avg)
        runs.append((losses, [t.detach().clone() for t in state]))
        del step, worker
    for losses, state in runs[1:]:
        assert losses == runs[0][0]
        for a, b in zip(state, runs[0][1]):
            assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


@pytest.mark.parametrize("which", ["gelu", "relu", "fork", "linear"])
def test_two_graphs_of_each_operator_replayed_beside_an_eager_call(which):
    """Forward and backward (dropout on) captured twice and replayed on two streams at once, with an eager call beside them."""
    import hap_b200
    from hap_b200 import block8
    from hap_b200 import dropout as D
    from hap_b200.norm import layer_norm_fork8
    x, w, b, g = (t.to(DEV) for t in linear_inputs(700, 520, 264, BF))
    gx, wv, bv = x.flip(0), w[0].clone(), w[1].clone()
    w8 = block8.quantize_weight(w, transposed=True)

    def step(v):
        v, lw, lb = (t.detach().requires_grad_(True) for t in (v, wv, bv))
        if which == "fork":
            res, y = layer_norm_fork8(v, (520,), lw, lb)
            return (y.detach(), *torch.autograd.grad([res, y], (v, lw, lb), [gx, gx]))
        if which == "linear":
            y = hap_b200.linear8(v, w8, b)
            return (y.detach(), *torch.autograd.grad(y, v, g))
        y = D._ActDropout8.apply(v, D._ACTS[which], 0.25, 7)             # the same call id, so the same mask, in every call
        return (y.detach(), *torch.autograd.grad(y, v, gx))
    xs = [x, x * 2]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[t.clone() for t in step(v)] for v in xs]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(float(t.float().abs().max()) > 0 for t in want[0])
    graphs, outs = [], []
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


# ---- next to the operators in their own types ---------------------------------------------------------
@pytest.mark.parametrize("dtype,apart", [(F32, 2.0 ** -20), (BF, 2.0 ** -18)])
def test_activation_forward_next_to_act_dropout(dtype, apart):
    """relu has the same bits.  gelu = x Phi(x) has two forms of Phi.  float32: 0.5 (1 + erff): two steps of erff, the rounding of
    its argument (z erf'(z) <= 0.49) and of the sum, 2^-23 together; act_dropout8's tail of at most 1/2: its fit 1e-7 relative,
    ex2 and rcp 2^-22 each, the rounding of u and u^2 (2 u^2 ln2 2^-24, largest times the tail at v = 1: 2^-25), eight of the
    polynomial: 2^-21 together.  bfloat16: 7.5e-8 of the rational erf, 2.1e-6 = 4.1e-6 / 2 of the fit, and the same roundings."""
    from hap_b200 import dropout as D
    x = torch.cat([torch.linspace(-14, 14, 1 << 18), torch.randn(1 << 18, generator=gen(0)) * 2]).to(dtype).to(DEV)
    for p in (0.0, 0.25):
        for act in ("relu", "gelu"):
            D.manual_seed(4), D.advance()
            first = D.act_dropout(x, act, p)
            D.manual_seed(4), D.advance()
            b = D.act_dropout8(x, act, p)
            if act == "relu":
                assert torch.equal(first, b)
            else:
                close(b, first.cpu().double(), (x.abs().cpu().double() * apart / (1 - p) + half_step(dtype) * first.abs().cpu().double()))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,E", [(591, 768), (130, 2048), (70, 400), (9, 1000)])
def test_norm_forward_next_to_layer_norm(dtype, rows, E):
    """The same numbers with sums in another order: each is within its bound of the exact one."""
    import hap_b200
    x = (torch.randn(rows, E, generator=gen(rows)) * 2 + 0.25).to(dtype)
    w, b, g = (torch.rand(E, generator=gen(1)) + 0.5).to(dtype), torch.randn(E, generator=gen(2)).to(dtype), torch.zeros(rows, E)
    slack = norm_bounds(x, w, b, g, B.fast_rows(x), None, rows)[0]
    a, c = (f(x.to(DEV), (E,), w.to(DEV), b.to(DEV)) for f in (hap_b200.layer_norm, hap_b200.layer_norm8))
    close(c, a.cpu().double(), 2 * slack + half_step(dtype) * a.cpu().double().abs())


# ---- what is not finite -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,E", [(40, 33), (70, 768), (12, 2048), (5, 9001)])
def test_norm_rows_that_are_not_finite(dtype, rows, E):
    """A row with an infinity or a NaN is NaN in y and dx, as torch's, and makes dw NaN; the other rows and db do not see it."""
    import hap_b200
    x = torch.randn(rows, E, generator=gen(0)).to(dtype)
    w, b, g = (torch.rand(E, generator=gen(1)) + 0.5).to(dtype), torch.randn(E, generator=gen(2)).to(dtype), torch.randn(rows, E, generator=gen(3)).to(dtype)
    bad = x.clone()
    bad[1, E // 2], bad[2, 0], bad[3, E - 1], bad[3, 1] = float("nan"), float("inf"), -float("inf"), float("inf")

    def run(v):
        v, lw, lb = leaf(v), leaf(w), leaf(b)
        y = hap_b200.layer_norm8(v, E, lw, lb)
        return (y.detach(), *torch.autograd.grad(y, (v, lw, lb), g.to(DEV)))
    want, got = run(x), run(bad)
    ok = torch.tensor([r not in (1, 2, 3) for r in range(rows)], device=DEV)
    for i in (0, 1):
        assert bool(torch.isnan(got[i][~ok]).all()) and torch.equal(got[i][ok], want[i][ok])
    assert bool(torch.isnan(got[2]).all()) and torch.equal(got[3], want[3])
    assert bool(torch.isnan(torch.nn.functional.layer_norm(bad.to(DEV), (E,), w.to(DEV), b.to(DEV))[~ok]).all())


# ---- gradients through a prepared weight and through the attention block -------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows,fin,fout", [(1, 16, 24), (2, 130, 77), (33, 129, 300), (130, 1000, 40), (515, 96, 1000), (300, 768, 768)])
def test_input_gradient_through_a_prepared_weight(dtype, rows, fin, fout):
    import hap_b200
    from hap_b200 import block8
    x, w, b, g = linear_inputs(rows, fin, fout, dtype)
    want = B.linear8(x, w, b, g)
    w8 = block8.quantize_weight(w.to(DEV), transposed=True)
    xg, bg = leaf(x), leaf(b)
    y = hap_b200.linear8(xg, w8, bg)
    y.backward(g.to(DEV))
    check_linear((y, xg.grad, None, bg.grad), want, rows, fin, fout)
    again = leaf(x)
    hap_b200.linear8(again, w.to(DEV)).backward(g.to(DEV))                     # a weight that is quantised in the call
    assert torch.equal(again.grad, xg.grad)


def test_attention_block_gradients():
    """Every gradient of multi_head_attention_forward8 has the bits of the three operators called one by one, and the two
    projections are checked at the inputs and gradients that they saw."""
    import hap_b200
    from hap_b200.attention import attention, multi_head_attention_forward8
    L, n, E, H = 24, 3, 128, 2
    P = [t.to(BF) for t in (torch.randn(L, n, E, generator=gen(0)), torch.randn(3 * E, E, generator=gen(1)) * E ** -0.5, torch.randn(3 * E, generator=gen(2)),
                            torch.randn(E, E, generator=gen(3)) * E ** -0.5, torch.randn(E, generator=gen(4)))]
    g = torch.randn(L, n, E, generator=gen(5)).to(BF)
    a = [leaf(t) for t in P]
    out, weights = multi_head_attention_forward8(a[0], a[0], a[0], E, H, a[1], a[2], out_proj_weight=a[3], out_proj_bias=a[4], attn_mask="causal")
    out.backward(g.to(DEV))
    c = [leaf(t) for t in P]
    qkv = hap_b200.linear8(c[0], c[1], c[2])
    att = attention(qkv, H, "causal")
    qkv.retain_grad(), att.retain_grad()
    one_by_one = hap_b200.linear8(att, c[3], c[4])
    one_by_one.backward(g.to(DEV))
    assert weights is None and torch.equal(out, one_by_one)
    for s, t in zip(a, c):
        assert torch.equal(s.grad, t.grad) and float(s.grad.float().abs().max()) > 0
    flat = lambda t: t.detach().cpu().reshape(L * n, -1)
    check_linear((flat(qkv), flat(a[0].grad), a[1].grad, a[2].grad), B.linear8(flat(P[0]), P[1], P[2], flat(qkv.grad)), L * n, E, 3 * E)
    check_linear((flat(out), flat(att.grad), a[3].grad, a[4].grad), B.linear8(flat(att), P[3], P[4], flat(g)), L * n, E, E)


# ---- shards -------------------------------------------------------------------------------------------
def test_blocks_start_where_the_tensor_starts():
    """A shard cut at a multiple of 128 has the whole weight's blocks; any other cut has blocks, and so scales, of its own."""
    from hap_b200 import block8
    w = (torch.randn(700, 500, generator=gen(0)) * torch.exp(torch.randn(700, 1, generator=gen(1)))).to(DEV)
    whole = block8.quantize_weight(w).dequantize()
    for cut in (128, 384):
        assert torch.equal(block8.quantize_weight(w[cut:]).dequantize(), whole[cut:]) and torch.equal(block8.quantize_weight(w[:, :cut]).dequantize(), whole[:, :cut])
    shard = block8.quantize_weight(w[100:]).dequantize()
    assert not torch.equal(shard, whole[100:]) and torch.equal(shard.cpu().double(), B.quantize(w[100:].cpu(), square=True)[0])
    rows = block8.quantize(w).dequantize()
    assert torch.equal(block8.quantize(w[100:]).dequantize(), rows[100:])                       # 1 x 128 blocks do not see the rows above


@pytest.mark.parametrize("plan", ["dp", "dp_zero", "tp"])
def test_program_on_uneven_virtual_ranks(plan):
    """The language model on two virtual ranks with uneven shards, in bf16 and on the 8-bit operators.  A rounding to e4m3 is off by
    2^-4 / sqrt 3 rms at most; a gradient passes 2 operands of at most 18 products (9 forward, 9 back) and 7 kept inputs, 43
    independent roundings: sqrt(43) 2^-4 / sqrt 3 = 0.24 of its norm.  A shard in the wrong place would be off by 1."""
    import hap_b200
    from hap_b200 import fxpass
    from hap_b200.spmd import LockstepWorld
    from tests import spmd_common as C
    tok, tgt = (t.to(DEV) for t in C.lm_batch())
    comm = hap_b200.local_comm(2, DEV, stage_bytes=16 << 20, heap_bytes=32 << 20)
    try:
        grads, worlds = [], []
        for block8 in (False, True):
            modules = C.lm_rank_modules(C.lm_model(BF), plan, hap_b200.plan.default_namespace(), device=DEV)
            for m in modules:
                fxpass.fuse_elementwise(m.graph), fxpass.fuse_residual_norm(m.graph)
                if block8:
                    changed = fxpass.use_block8(m.graph)
                    assert changed["linear"] == 5 and changed["multi_head_attention_forward"] == 2
                m.recompile()
            world = LockstepWorld(modules, hap_b200.LocalCollectives(comm))
            losses = world.forward([(tok, tgt)] * 2)
            torch.stack(losses).sum().backward()
            grads.append([torch.cat([p.grad.float().flatten() for p in m.parameters()]) for m in modules])
            worlds.append(world)
        for a, b in zip(*grads):
            assert bool(torch.isfinite(b).all()) and float((a - b).norm()) <= 0.24 * float(a.norm())
            assert float((a - b).norm()) > 0
        world = worlds[1]
        for _ in range(2):
            loss = world.step([(tok, tgt)] * 2)
            assert bool(torch.isfinite(loss))
        if plan == "dp":                                           # replicas stay replicas
            for p, q in zip(*(m.parameters() for m in world.modules)):
                assert torch.equal(p, q)
        comm.check()
    finally:
        comm.destroy()
