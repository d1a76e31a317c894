"""The 8-bit operators at the ends of what they accept: the largest extents, scales far apart, values near the largest
float32 number, NaN and infinities, forward-mode differentiation, operands that do not fit together; and whole steps
replayed from CUDA graphs."""
import pytest
import torch

from oracle import block8_math as B
from tests.test_block8_gpu import BF, DEV, F32, close, gen, sum_slack

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
