"""The roofline that bench.py reports for a training step: a program on the 8-bit operators is held against their rate."""
import pytest

from bench import step_roofline

PEAKS = {"bf16_tflops": 1600.0, "bf16_tflops_sustained": 1400.0}


def test_bf16_step():
    r = step_roofline(7e12, 1e12, 100.0, PEAKS, "measured", False)
    assert r["kernel"].startswith("gemm2_bf16_kernel") and r["peak"] == 1400.0
    assert r["achieved"] == pytest.approx(210.0) and r["frac"] == pytest.approx(0.15)
    assert step_roofline(7e12, 1e12, 100.0, {"bf16_tflops": 1600.0}, "fallback", False)["peak"] == 1600.0


def test_block8_step_is_held_against_the_8_bit_rate():
    r = step_roofline(7e12, 1e12, 100.0, PEAKS, "measured", True)
    # 6 of 7 parts at 2800, one at 1400 TFLOP/s: no step can take less than 3 (6 / 2800 + 1 / 1400) s
    assert r["kernel"].startswith("gemm8_kernel") and "nominal ratio" in r["peak_kind"]
    assert r["frac"] == pytest.approx(3 * (6 / 2800 + 1 / 1400) / 0.1) and r["frac"] == pytest.approx(r["achieved"] / r["peak"])
    assert step_roofline(7e12, 0.0, 100.0, PEAKS, "measured", True)["peak"] == pytest.approx(2800.0)
    assert step_roofline(7e12, 7e12, 100.0, PEAKS, "measured", True)["peak"] == pytest.approx(1400.0)
