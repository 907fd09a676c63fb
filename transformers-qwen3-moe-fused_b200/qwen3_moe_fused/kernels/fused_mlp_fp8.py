"""Gated expert MLP on 8-bit weights (quantize/fp8.py): y = down(silu(gate x) * up x), and the gradient of x.

With Q for the quantisation of rows:
    e = Q(x) Wg^T    g = Q(x) Wu^T    h = silu(e) g    y = Q(h) Wd^T
    dh = Q(dy) Wd    de, dg from dh, e, g    dx = Q(de) Wg + Q(dg) Wu
Products, activation and gradients are fp32; what is rounded are the codes that Q makes, y, dx, and e and g where they are
kept for a backward pass (in the type of x, as an unquantised layer keeps them).  The weights are frozen.

The reference has no 8-bit weights; the MLP is that of qwen3_moe_fused/modular_qwen3_moe_fused.py:105-110.
"""
import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ..grouped_gemm.fp8 import grouped_gemm_fp8
from ..quantize.fp8 import FP8, check_weight, empty_scales, quantize_fp8_rows


def _codes(M: int, K: int, device):
    return torch.empty((M, K), device=device, dtype=FP8), empty_scales(M, K, device)


def _gate_up(x, gate, gate_scale, up, up_scale, m_sizes, keep: bool):
    """(hq, hs) and, with `keep`, (e, g) in the type of x."""
    q, s = quantize_fp8_rows(x)
    M, K = x.shape
    E, I = gate.shape[:2]
    check_weight(gate, gate_scale)
    check_weight(up, up_scale)
    assert gate.shape[2] == K and gate.device == up.device == m_sizes.device == x.device
    assert m_sizes.ndim == 1 and m_sizes.is_contiguous() and m_sizes.numel() == E and _lib.is_int_tensor(m_sizes)
    ms = _lib.as_index_tensor(m_sizes)
    hq, hs = _codes(M, I, x.device)
    e, g = (torch.empty((M, I), device=x.device, dtype=x.dtype) if keep else None for _ in range(2))
    lib = _lib.load()
    here, stream = _lib.launch_on(x.device)
    with here:
        status = lib.moe_gate_up_silu_fp8(
            _lib.ptr(q), _lib.ptr(s), _lib.ptr(gate), _lib.ptr(gate_scale), _lib.ptr(up), _lib.ptr(up_scale), _lib.ptr(ms),
            _lib.int_code(ms.dtype), _lib.ptr(hq), _lib.ptr(hs), _lib.ptr(e), _lib.ptr(g), M, I, K, E, _lib.float_code(x.dtype),
            stream)
    if status != _lib.ERR_UNSUPPORTED:
        _lib.check(status, "moe_gate_up_silu_fp8")
        return hq, hs, e, g
    # extents or types that the kernel does not cover: the products one by one
    e32 = grouped_gemm_fp8(((q, s, gate, gate_scale),), m_sizes, torch.float32)
    g32 = grouped_gemm_fp8(((q, s, up, up_scale),), m_sizes, torch.float32)
    with here:
        status = lib.moe_fp8_silu_quantize(_lib.ptr(e32), _lib.ptr(g32), M, I, _lib.ptr(hq), _lib.ptr(hs), _lib.ptr(e), _lib.ptr(g),
                                           _lib.float_code(x.dtype), stream)
    _lib.check(status, "moe_fp8_silu_quantize")
    return hq, hs, e, g


def _down_bwd(dy, down, down_scale, e, g, m_sizes):
    """Quantised gradients of e and g."""
    q, s = quantize_fp8_rows(dy)
    M, I = e.shape
    dh = grouped_gemm_fp8(((q, s, down, down_scale),), m_sizes, torch.float32, transposed=True)
    # (hooks on saved tensors may have given back another type, device or layout)
    assert e.dtype == g.dtype == dy.dtype and e.shape == g.shape == dh.shape and e.is_contiguous() and g.is_contiguous()
    assert e.device == g.device == dy.device
    (deq, des), (dgq, dgs) = _codes(M, I, dy.device), _codes(M, I, dy.device)
    here, stream = _lib.launch_on(dy.device)
    with here:
        status = _lib.load().moe_fp8_silu_bwd_quantize(_lib.ptr(dh), _lib.ptr(e), _lib.ptr(g), M, I, _lib.ptr(deq), _lib.ptr(des),
                                                       _lib.ptr(dgq), _lib.ptr(dgs), _lib.float_code(dy.dtype),
                                                       stream)
    _lib.check(status, "moe_fp8_silu_bwd_quantize")
    return deq, des, dgq, dgs


class MlpFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, gate_scale, up, up_scale, down, down_scale, m_sizes):
        hq, hs, e, g = _gate_up(x, gate, gate_scale, up, up_scale, m_sizes, True)
        ctx.save_for_backward(gate, gate_scale, up, up_scale, down, down_scale, m_sizes, e, g)
        return grouped_gemm_fp8(((hq, hs, down, down_scale),), m_sizes, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        none = (None,) * 7
        if not ctx.needs_input_grad[0]:
            return None, *none
        gate, gate_scale, up, up_scale, down, down_scale, m_sizes, e, g = ctx.saved_tensors
        deq, des, dgq, dgs = _down_bwd(dy.contiguous(), down, down_scale, e, g, m_sizes)
        return grouped_gemm_fp8(((deq, des, gate, gate_scale), (dgq, dgs, up, up_scale)), m_sizes, dy.dtype, transposed=True), *none


def moe_mlp_fp8(x: torch.Tensor, gate: torch.Tensor, gate_scale: torch.Tensor, up: torch.Tensor, up_scale: torch.Tensor,
                down: torch.Tensor, down_scale: torch.Tensor, m_sizes: torch.Tensor) -> torch.Tensor:
    """x (M, H), rows sorted by expert; gate, up (E, I, H) and down (E, H, I) float8_e4m3fn with their block scales (as in
    `moe_fused_linear_fp8`); m_sizes (E,) integers that sum to M.  Returns (M, H) in the type of x.  Differentiable in x,
    once."""
    assert gate.ndim == 3 and up.shape == gate.shape and down.shape == (gate.shape[0], gate.shape[2], gate.shape[1])
    if _lib.has_tangent(x) or (torch.is_grad_enabled() and x.requires_grad):
        return MlpFp8.apply(x, gate, gate_scale, up, up_scale, down, down_scale, m_sizes)
    hq, hs, _, _ = _gate_up(x, gate, gate_scale, up, up_scale, m_sizes, False)
    return grouped_gemm_fp8(((hq, hs, down, down_scale),), m_sizes, x.dtype)
