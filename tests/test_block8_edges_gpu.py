"""The 8-bit operators at the ends of what they accept: the largest extents, scales far apart, values near the largest
float32 number, NaN and infinities, forward-mode differentiation, operands that do not fit together; and whole steps
replayed from CUDA graphs."""
import pytest
import torch

from oracle import block8_math as B
from tests.test_block8_gpu import BF, DEV, F32, close, gen, leaf, linear_inputs, lm_worker, sum_slack

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
