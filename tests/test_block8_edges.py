"""The 8-bit operators without a GPU: operands that do not fit together, derivatives that are not there."""
import sys

import pytest
import torch

from hap_b200 import block8
from tests.test_block8 import _block8


def test_blocks_that_do_not_hold_their_matrix_are_refused():
    values, scales = torch.zeros(40, 48, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.full((512,), 127, dtype=torch.uint8)
    good = block8.Block8(values, scales, 40, 40)
    assert block8.Block8(values, scales, 40, 33).shape == (40, 33)                          # a pitch above the row's need
    for args, err in (((values, scales, 41, 40), ValueError), ((values, scales, 40, 49), ValueError), ((values, scales, 40, 0), ValueError),
                      ((values, scales, -1, 40), ValueError), ((values[:, :40], scales, 40, 40), ValueError), ((values[0], scales, 1, 40), ValueError),
                      ((values.view(torch.uint8)[:, :40].contiguous().view(torch.float8_e4m3fn), scales, 40, 40), ValueError),      # pitch not of 16 bytes
                      ((values.view(torch.uint8), scales, 40, 40), TypeError), ((values, scales.float(), 40, 40), TypeError),
                      ((values, scales[:511], 40, 40), ValueError), ((values, scales.repeat(2)[::2], 40, 40), ValueError),
                      ((values, scales.to("meta"), 40, 40), ValueError), ((values, scales, 40, 40, _block8(40, 41)), ValueError)):
        with pytest.raises(err, match="Block8"):
            block8.Block8(*args)
    assert block8.Block8(values, scales, 40, 40, good).transposed is good


def test_prepared_weights_of_another_pitch_are_refused():
    from hap_b200.linear8 import _check_prepared
    wide = block8.Block8(torch.zeros(40, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.full((512,), 127, dtype=torch.uint8), 40, 40)
    square = _block8(40, 40)
    _check_prepared(square, False)
    with pytest.raises(ValueError, match="64 bytes apart, 48"):
        _check_prepared(wide, False)
    with pytest.raises(ValueError, match="transposed form"):
        _check_prepared(square, True)
    with pytest.raises(ValueError, match="64 bytes apart, 48"):
        _check_prepared(block8.Block8(square.values, square.scales, 40, 40, wide), True)
    odd = _block8(40, 40)
    odd.transposed = _block8(40, 41)
    with pytest.raises(ValueError, match="not the transposed form"):
        _check_prepared(odd, True)


class _OnGpu(torch.Tensor):
    """A host tensor that passes for one on the GPU, for what happens before any launch."""
    is_cuda = True


def _operators(monkeypatch):
    """The four operators with their launches left out, as functions of one input and one parameter vector."""
    from hap_b200 import dropout, norm
    modules = [sys.modules[f"hap_b200.{m}"] for m in ("linear8", "dropout", "norm")]
    for m in modules:
        monkeypatch.setattr(m, "_launch", lambda *args: None)
    monkeypatch.setattr(modules[0], "_forward_workspace", lambda *args: 0)
    w, w8 = torch.ones(4, 8).as_subclass(_OnGpu), _block8(4, 8)
    linear8 = modules[0].linear8
    return {"linear8": lambda x, v: linear8(x, w, v[:4]), "linear8 of a prepared weight": lambda x, v: linear8(x, w8, v[:4]),
            "act_dropout8": lambda x, v: dropout.act_dropout8(x * v, "gelu", 0.0), "layer_norm8": lambda x, v: norm.layer_norm8(x, 8, v),
            "layer_norm_fork8": lambda x, v: norm.layer_norm_fork8(x, 8, v)}


@pytest.mark.parametrize("which", ["linear8", "linear8 of a prepared weight", "act_dropout8", "layer_norm8", "layer_norm_fork8"])
def test_tangents_are_refused(monkeypatch, which):
    """Forward-mode differentiation: a dual tensor has requires_grad False; a result without a tangent would read as a zero
    derivative."""
    from torch.autograd import forward_ad
    f = _operators(monkeypatch)[which]
    x, v = torch.ones(2, 8).as_subclass(_OnGpu), torch.ones(8).as_subclass(_OnGpu)
    f(x, v)
    with forward_ad.dual_level():
        f(x, v)                                                    # no tangent, nothing to refuse
        for args in ((forward_ad.make_dual(x, x), v), (x, forward_ad.make_dual(v, v))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                    f(*args)
    f(x, v)


def test_use_block8_leaves_norms_that_layer_norm_hands_to_torch():
    from hap_b200 import fxpass
    from hap_b200.norm import layer_norm, layer_norm8, layer_norm_fork, layer_norm_fork8
    root = torch.nn.Module()
    for name, dtype in (("p16", torch.float16), ("p64", torch.float64), ("pb16", torch.bfloat16), ("p32", torch.float32)):
        root.register_parameter(name, torch.nn.Parameter(torch.ones(8, dtype=dtype)))
    graph = torch.fx.Graph(root)
    x, n = graph.placeholder("x"), graph.placeholder("n")
    p = {name: graph.get_attr(name) for name, _ in root.named_parameters()}
    typed = graph.call_function(torch.relu, (x,))
    typed.meta["val"] = torch.empty(2, 8, dtype=torch.float16)
    stay = [graph.call_function(layer_norm, (x, (4, 8))), graph.call_function(layer_norm, (x, [4, 8], None, None)),
            graph.call_function(layer_norm_fork, (x,), {"normalized_shape": (4, 8)}), graph.call_function(layer_norm, (x, (1 << 20) + 1)),
            graph.call_function(layer_norm, (x, ())), graph.call_function(layer_norm, (x, (0,))), graph.call_function(layer_norm, (x, n)),
            graph.call_function(layer_norm, (x, (n,))), graph.call_function(layer_norm, (x, (8,), p["p16"])),
            graph.call_function(layer_norm, (x, (8,)), {"bias": p["p64"]}), graph.call_function(layer_norm, (x, (8,), p["p32"], p["pb16"])),
            graph.call_function(layer_norm, (typed, (8,))), graph.call_function(layer_norm_fork, (typed, 8))]
    move = [graph.call_function(layer_norm, (x, (8,))), graph.call_function(layer_norm, (x, 8, p["pb16"], p["pb16"])),
            graph.call_function(layer_norm, (x,), {"normalized_shape": [1 << 20], "weight": p["p32"], "eps": 1e-6}),
            graph.call_function(layer_norm_fork, (x, torch.Size([8]), p["p32"]))]
    graph.output(tuple(stay + move))
    before = [node.target for node in stay]
    assert fxpass.use_block8(graph, products=False) == {"act_dropout": 0, "layer_norm": 3, "layer_norm_fork": 1}
    assert [node.target for node in stay] == before
    assert [node.target for node in move] == [layer_norm8, layer_norm8, layer_norm8, layer_norm_fork8]


def test_every_bounded_wait_has_a_code_of_its_own():
    """hapx_gemm_status names the role that gave up: the quantiser and the product's own quantising warps are two."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(block8.__file__), "csrc")
    text = {name: open(os.path.join(csrc, name)).read() for name in ("hapx_block8.cu", "hapx_gemm8_sm100.cu", "hapx_gemm_sm100.cu")}
    codes = {name: re.findall(r"atomicCAS\(\w+\.error, 0u, (\d+)u\)", t) for name, t in text.items()}
    assert codes["hapx_block8.cu"] == ["4"] and sorted(codes["hapx_gemm8_sm100.cu"]) == ["1", "2", "3", "5"]
    message = text["hapx_gemm_sm100.cu"].split("gave up waiting on a barrier (role ")[1].split(";")[0]
    for code in sum(codes.values(), []):
        assert re.search(rf"\b{code} = ", message), f"role {code} is not named"
