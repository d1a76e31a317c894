"""8-bit blocks without a GPU: the oracle against torch's own e4m3 conversion, refusals of the Python layer and of the
C entry points, and the fx pass that moves a program onto the 8-bit operators."""
import pytest
import torch

import hap_b200
from hap_b200 import _native as N
from hap_b200 import block8, fxpass, plan
from oracle import block8_math as B


def test_oracle_rounds_like_torch():
    v = torch.cat([torch.arange(-448, 449, dtype=torch.float64) / 1.0, torch.arange(-4000, 4001, dtype=torch.float64) / 2 ** 14])
    assert torch.equal(B.round_e4m3(v), v.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("big,scale", [(0.0, 1.0), (448.0, 1.0), (448.5, 2.0), (447.0, 1.0), (224.0, 0.5), (224.5, 1.0), (1e-45, 2.0 ** -126),
                                       (3.0e38, 2.0 ** 120), (1.75, 2.0 ** -8), (1.76, 2.0 ** -7)])
def test_oracle_scale(big, scale):
    assert B.scale_of(big) == scale


def _ints(*shape, low=-7, high=8, seed=0):
    return torch.randint(low, high, shape, generator=torch.Generator().manual_seed(seed)).float()


def test_oracle_keeps_small_integers():
    x = _ints(5, 300)
    assert torch.equal(B.quantize(x)[0], x.double()) and torch.equal(B.fast_rows(x), x.double())
    assert torch.equal(B.quantize(x, square=True)[0], x.double())


def test_cpu_tensors_are_refused():
    x, w = torch.ones(2, 8), torch.ones(4, 8)
    for call in (lambda: block8.quantize(x), lambda: block8.quantize_weight(w), lambda: hap_b200.linear8(x, w),
                 lambda: hap_b200.dropout.act_dropout8(x, "gelu", 0.0), lambda: hap_b200.layer_norm8(x, (8,)),
                 lambda: hap_b200.norm.layer_norm_fork8(x, 8)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_quantize_with_nothing_to_do_is_refused():
    with pytest.raises(ValueError, match="nothing asked for"):
        block8.quantize(torch.ones(2, 8), rows=False)


def _block8(rows, cols):
    return block8.Block8(torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.uint8).view(torch.float8_e4m3fn),
                         torch.full((-(-cols // 512) * -(-rows // 128) * 512,), 127, dtype=torch.uint8), rows, cols)


def test_scale_matrix_decodes_the_order_of_the_tensor_cores():
    b = _block8(300, 700)                                               # 3 groups of rows, 6 blocks of columns in 2 groups of 4
    assert b.scales.numel() == N.lib.hapx_block8_scale_bytes(300, 700) == 2 * 3 * 512 and b.nbytes == 300 * 704 + 6 * 512
    for r, kb in ((0, 0), (31, 1), (32, 2), (127, 3), (128, 4), (299, 5), (170, 3)):
        b.scales.fill_(127)
        b.scales[((kb // 4) * 3 + r // 128) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + kb % 4] = 130
        want = torch.ones(300, 6)
        want[r, kb] = 8.0
        assert torch.equal(b.scale_matrix(), want)
    assert _block8(0, 40).scale_matrix().shape == (0, 1) and N.lib.hapx_block8_scale_bytes(0, 40) == 0


def test_matmul_refusals():
    a, b = _block8(3, 40), _block8(5, 40)
    with pytest.raises(ValueError, match="contraction"):
        block8.matmul(a, _block8(5, 41))
    with pytest.raises(TypeError, match="output"):
        block8.matmul(a, b, out_dtype=torch.float16)
    with pytest.raises(TypeError, match="bias"):
        block8.matmul(a, b, torch.zeros(5), torch.bfloat16)
    with pytest.raises(ValueError, match="bias"):
        block8.matmul(a, b, torch.zeros(4), torch.float32)


def test_c_entries_refuse_before_any_launch():
    """Pointers below are never dereferenced: every call is answered by the checks of its arguments."""
    p, q = 4096, 4097                                                    # a 16-byte aligned and an odd address
    quant = N.lib.hapx_block8_quantize
    assert quant(p, N.F16, 4, 8, 8, 0, p, 16, p, None, 0, None, None, None) == N.ERR_DTYPE
    assert quant(p, N.BF16, 4, 8, 7, 0, p, 16, p, None, 0, None, None, None) == N.ERR_EXTENT      # pitch below the row
    assert quant(p, N.BF16, -1, 8, 8, 0, p, 16, p, None, 0, None, None, None) == N.ERR_EXTENT
    assert quant(p, N.BF16, 4, 8, 8, 0, p, 8, p, None, 0, None, None, None) == N.ERR_EXTENT       # pitch not of 16 bytes
    assert quant(p, N.BF16, 4, 8, 8, 0, q, 16, p, None, 0, None, None, None) == N.ERR_EXTENT
    assert quant(p, N.BF16, 40, 8, 8, 0, None, 0, None, p, 32, p, None, None) == N.ERR_EXTENT     # pitch below the column
    assert quant(p, N.BF16, 4, 8, 8, 0, None, 0, None, q, 16, p, None, None) == N.ERR_EXTENT
    assert quant(p, N.BF16, 4, 8, 8, 0, None, 0, None, None, 0, None, None, None) == N.ERR_ARGUMENT
    assert quant(p, N.BF16, 4, 8, 8, 0, p, 16, None, None, 0, None, None, None) == N.ERR_ARGUMENT
    assert quant(None, N.BF16, 4, 8, 8, 0, p, 16, p, None, 0, None, None, None) == N.ERR_ARGUMENT
    assert quant(p, N.BF16, 1 << 40, 1 << 40, 1 << 40, 0, p, 1 << 40, p, None, 0, None, None, None) == N.ERR_EXTENT
    assert quant(None, N.BF16, 0, 8, 8, 0, None, 0, None, None, 0, None, None, None) == N.OK      # an empty matrix
    assert N.lib.hapx_block8_dequantize(p, N.F64, p, 16, p, 4, 8, None) == N.ERR_DTYPE
    assert N.lib.hapx_block8_dequantize(p, N.F32, p, 4, p, 4, 8, None) == N.ERR_EXTENT
    assert N.lib.hapx_block8_dequantize(None, N.F32, p, 16, p, 4, 8, None) == N.ERR_ARGUMENT
    assert N.lib.hapx_block8_colsum_join(p, N.F16, p, 4, 8, None) == N.ERR_DTYPE
    assert N.lib.hapx_block8_colsum_join(None, N.F32, p, 4, 8, None) == N.ERR_ARGUMENT
    mm = N.lib.hapx_block8_matmul
    assert mm(p, N.F16, p, 16, p, p, 16, p, None, 4, 4, 8, None, 0, None) == N.ERR_DTYPE
    assert mm(p, N.BF16, p, 16, p, p, 16, p, None, 4, 4, -8, None, 0, None) == N.ERR_EXTENT
    assert mm(p, N.BF16, p, 16, p, p, 16, p, None, 4, 4, 0, None, 0, None) == N.ERR_EXTENT
    assert mm(p, N.BF16, p, 16, p, p, 16, p, None, 1 << 31, 4, 8, None, 0, None) == N.ERR_EXTENT
    assert mm(p, N.BF16, p, 16, p, p, 12, p, None, 4, 4, 8, None, 0, None) == N.ERR_EXTENT
    assert mm(p, N.BF16, q, 16, p, p, 16, p, None, 4, 4, 8, None, 0, None) == N.ERR_EXTENT
    assert mm(p, N.BF16, p, 16, q, p, 16, p, None, 4, 4, 8, None, 0, None) == N.ERR_EXTENT
    assert mm(None, N.BF16, p, 16, p, p, 16, p, None, 4, 4, 8, None, 0, None) == N.ERR_ARGUMENT
    assert mm(p, N.BF16, None, 16, p, p, 16, p, None, 4, 4, 8, None, 0, None) == N.ERR_ARGUMENT
    assert mm(None, N.BF16, None, 0, None, None, 0, None, None, 0, 4, 8, None, 0, None) == N.OK
    act = N.lib.hapx_act_dropout8
    assert act(p, p, p, p, N.F16, 8, 2, 0.0, 0, None) == N.ERR_DTYPE
    assert act(p, p, p, p, N.F32, -1, 2, 0.0, 0, None) == N.ERR_EXTENT
    assert act(p, p, p, p, N.F32, 8, 3, 0.0, 0, None) == N.ERR_ARGUMENT
    assert act(p, p, p, p, N.F32, 8, 2, 1.0, 0, None) == N.ERR_ARGUMENT
    assert act(p, p, None, p, N.F32, 8, 2, 0.0, 0, None) == N.ERR_ARGUMENT
    assert act(p, q, p, p, N.F32, 8, 2, 0.0, 0, None) == N.ERR_EXTENT
    assert N.lib.hapx_act_dropout8_backward(p, p, None, p, N.F32, 8, 2, 0.0, 0, None) == N.ERR_ARGUMENT
    assert N.lib.hapx_act_dropout8_backward(p, p, q, p, N.F32, 8, 2, 0.0, 0, None) == N.ERR_EXTENT
    ln = N.lib.hapx_layer_norm8_forward
    assert ln(p, p, p, p, p, p, p, 16, p, N.F16, 4, 8, 1e-5, None) == N.ERR_DTYPE
    assert ln(p, p, p, p, p, p, p, 16, p, N.F32, 4, 0, 1e-5, None) == N.ERR_EXTENT
    assert ln(p, p, p, p, p, p, p, 8, p, N.F32, 4, 8, 1e-5, None) == N.ERR_EXTENT
    assert ln(p, p, p, p, None, p, p, 16, p, N.F32, 4, 8, 1e-5, None) == N.ERR_ARGUMENT
    bw = N.lib.hapx_layer_norm8_backward
    assert bw(p, 16, p, p, p, p, p, None, p, p, None, None, N.F32, 4, 8, None) == N.ERR_ARGUMENT        # no workspace
    assert bw(None, 16, p, p, p, p, p, None, p, None, None, None, N.F32, 4, 8, None) == N.ERR_ARGUMENT
    assert bw(p, 8, p, p, p, p, p, None, p, None, None, None, N.F32, 4, 8, None) == N.ERR_EXTENT
    assert N.lib.hapx_last_error()


def test_use_block8_moves_a_program():
    model = plan.TransformerLM(vocab=64, d_model=64, nheads=1, d_ffn=128, nlayers=2, seqlen=8)
    graph = plan.emit_lm(model, "dp", [1.0], 0, 4, dropout_p=0.1)
    fxpass.fuse_elementwise(graph)
    fxpass.fuse_residual_norm(graph)
    changed = fxpass.use_block8(graph, skip=lambda n: n.target is hap_b200.linear and "dec_w" in str(n.args[1].args))
    assert changed == {"linear": 4, "multi_head_attention_forward": 2, "act_dropout": 2, "layer_norm": 1, "layer_norm_fork": 4}
    names = [n.target.__name__ for n in graph.nodes if n.op == "call_function"]
    assert names.count("linear8") == 4 and names.count("linear") == 1 and names.count("act_dropout8") == 2
    from hap_b200.spmd import _program_has_dropout
    assert _program_has_dropout(torch.fx.GraphModule(model, graph))
    again = fxpass.use_block8(graph, products=False)
    assert not any(again.values()) and set(again) == {"act_dropout", "layer_norm", "layer_norm_fork"}
