"""8-bit operators and norms without a GPU: what the library refuses before it touches a device, and the weight's codes."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as entry

    entry.build()
    from qwen3_moe_fused import _lib

    return _lib.load()


def test_argument_errors_return_before_any_launch(lib):
    assert lib.moe_fp8_quantize_rows(None, 9, 4, 128, None, None, None) == -1
    assert lib.moe_fp8_quantize_rows(None, 1, 4, 0, None, None, None) == -2
    assert lib.moe_fp8_quantize_rows(None, 1, -1, 128, None, None, None) == -2
    assert lib.moe_fp8_quantize_rows(None, 1, 4, 128, None, None, None) == -3
    assert lib.moe_fp8_quantize_rows(None, 1, 0, 128, None, None, None) == 0
    none8 = [None] * 8
    assert lib.moe_grouped_gemm_fp8(0, *none8, None, 3, None, 4, 8, 8, 2, 9, None) == -1
    assert lib.moe_grouped_gemm_fp8(0, *none8, None, 1, None, 4, 8, 8, 2, 1, None) == -1  # m_sizes in a floating type
    assert lib.moe_grouped_gemm_fp8(2, *none8, None, 3, None, 4, 8, 8, 2, 1, None) == -2
    assert lib.moe_grouped_gemm_fp8(0, *none8, None, 3, None, 4, 0, 8, 2, 1, None) == -2
    assert lib.moe_grouped_gemm_fp8(0, *none8, None, 3, None, 4, 8, 8, 70000, 1, None) == -2
    assert lib.moe_grouped_gemm_fp8(0, *none8, None, 3, None, 4, 8, 8, 2, 1, None) == -3
    assert lib.moe_combine_add_rms_norm(None, None, None, None, None, 1.0, 1e-6, None, None, None, 4, 2, 8, 1, None) == -2
    assert lib.moe_combine_add_rms_norm(None, None, None, None, None, 1.0, 1e-6, 64, None, None, 4, 1, 24577, 1, None) == -2
    assert lib.moe_combine_add_rms_norm(None, None, None, None, None, 1.0, 1e-6, 64, None, None, 4, 1, 8, 1, None) == -3
    assert lib.moe_combine_add_rms_norm_bwd(64, None, 64, 64, 64, None, None, None, 1.0, None, None, None, 64, 4, 1, 8, 1, None, 0,
                                            None) == -4  # the norm weight's gradient without a workspace
    assert lib.moe_combine_add_rms_norm_bwd_ws_bytes(0, 64) == 0


def test_wrappers_reject_cpu_tensors():
    from qwen3_moe_fused.kernels.norm import add_rms_norm
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8, quantize_fp8_rows
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    codes, s = quantize_fp8(torch.ones(2, 8, 16))
    with pytest.raises(AssertionError):
        moe_fused_linear_fp8(torch.ones(4, 16), codes, s, torch.tensor([2, 2]))
    with pytest.raises(AssertionError):
        quantize_fp8_rows(torch.ones(4, 16))
    with pytest.raises(AssertionError):
        add_rms_norm(torch.ones(4, 16), None, torch.ones(16))


def test_weight_codes():
    from qwen3_moe_fused.quantize.fp8 import dequantize_fp8, quantize_fp8

    w = torch.randn(2, 130, 257, generator=torch.Generator().manual_seed(0))
    codes, s = quantize_fp8(w)
    assert codes.dtype == torch.float8_e4m3fn and s.shape == (2, 2, 3)
    # each block's largest value is the largest code
    assert codes[0, :128, :128].float().abs().max() == 448 and codes[1, 128:, 256:].float().abs().max() == 448
    # half a step: 2^-4 of the value (the quotient is rounded once more, 2^-24) or 2^-10 of the scale
    full = s.repeat_interleave(128, 1)[:, :130].repeat_interleave(128, 2)[:, :, :257]
    assert bool(((dequantize_fp8(codes, s) - w).abs() <= w.abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + full * 2.0 ** -10).all())


def test_extents_past_an_int_are_refused(lib):
    big = (1 << 24) + 1
    none8 = [None] * 8
    for N, K in ((big, 8), (8, big), (2 ** 31 - 1, 8), (8, 2 ** 31 - 1)):
        assert lib.moe_grouped_gemm_fp8(0, *none8, None, 3, None, 4, N, K, 2, 1, None) == -2
        assert lib.moe_gate_up_silu_fp8(*[None] * 7, 3, *[None] * 4, 4, N, K, 2, 1, None) == -2
    assert lib.moe_fp8_quantize_rows(None, 1, 4, big, None, None, None) == -2
    assert lib.moe_fp8_quantize_rows(None, 1, 2 ** 31, 8, None, None, None) == -2
