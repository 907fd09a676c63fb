"""`MoeFusedLinear` forward on 8-bit weights with block scales: both directions are 8-bit products on the tensor cores.

The 8-bit weight is frozen and gets no gradient, like the 4-bit one (qwen3_moe_fused/quantize/layer.py:17-22).
"""
import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ..grouped_gemm.fp8 import grouped_gemm_fp8
from .fp8 import quantize_fp8_rows


class _FusedLinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, weight_scale, m_sizes):
        ctx.save_for_backward(weight, weight_scale, m_sizes)
        return _forward(input, weight, weight_scale, m_sizes)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        if not ctx.needs_input_grad[0]:
            return None, None, None, None
        weight, weight_scale, m_sizes = ctx.saved_tensors
        q, s = quantize_fp8_rows(grad_output.contiguous())
        return grouped_gemm_fp8(((q, s, weight, weight_scale),), m_sizes, grad_output.dtype, transposed=True), None, None, None


def _forward(input, weight, weight_scale, m_sizes):
    q, s = quantize_fp8_rows(input)
    return grouped_gemm_fp8(((q, s, weight, weight_scale),), m_sizes, input.dtype)


def moe_fused_linear_fp8(input: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, m_sizes: torch.Tensor) -> torch.Tensor:
    """
    Args:
        input: `(batch_size, in_features)`, rows sorted by expert; quantised in the call, see quantize/fp8.py.
        weight: `(num_experts, out_features, in_features)`, float8_e4m3fn.
        weight_scale: `(num_experts, ceil(out_features / 128), ceil(in_features / 128))`, float32.
        m_sizes: `(num_experts,)` integer row counts per expert; sums to `batch_size`.

    Returns:
        `(batch_size, out_features)` in the dtype of `input`, from fp32 sums rounded once.  The gradient of `input` is the
        product of the gradient, quantised like the input, with the weight; it can be taken once (no second derivative).
    """
    if _lib.has_tangent(input) or (torch.is_grad_enabled() and input.requires_grad):
        return _FusedLinearFp8.apply(input, weight, weight_scale, m_sizes)
    return _forward(input, weight, weight_scale, m_sizes)
