"""The residual stream around the sparse block: weighted combine or plain block output, scaled and added to the residual,
and the RMS norm in front of the next block, as one kernel per direction.

The reference leaves the addition and the norms to the decoder layer of transformers, one ATen call each, behind its own
combine (qwen3_moe_fused/modular_qwen3_moe_fused.py:112-115).
"""
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib


def _forward(y, inv_sort_idx, weights, residual, gamma, eps: float, scale: float, want_rstd: bool):
    H = y.shape[1]
    T, k = weights.shape if weights is not None else (y.shape[0], 1)
    total = torch.empty((T, H), device=y.device, dtype=y.dtype)
    normed = torch.empty_like(total)
    rstd = torch.empty(T, device=y.device, dtype=torch.float32) if want_rstd else None
    here, stream = _lib.launch_on(y.device)
    with here:
        status = _lib.load().moe_combine_add_rms_norm(
            _lib.ptr(y), _lib.ptr(inv_sort_idx), _lib.ptr(weights), _lib.ptr(residual), _lib.ptr(gamma), scale, eps,
            _lib.ptr(total), _lib.ptr(normed), _lib.ptr(rstd), T, k, H, _lib.float_code(y.dtype), stream)
    _lib.check(status, "moe_combine_add_rms_norm")
    return normed, total, rstd


class CombineAddRmsNorm(torch.autograd.Function):
    """(normed, sum); inv_sort_idx and weights None: y is added as it is.  Differentiable once."""

    @staticmethod
    def forward(ctx, y, inv_sort_idx, weights, residual, gamma, eps, scale):
        normed, total, rstd = _forward(y, inv_sort_idx, weights, residual, gamma, eps, scale, True)
        # the backward forms the sum again: `total` has been rounded, and may be infinite in fp16 where `normed` is not
        ctx.save_for_backward(y, inv_sort_idx, weights, residual, gamma, rstd)
        ctx.scale, ctx.y_shape, ctx.k = scale, y.shape, 1 if weights is None else weights.shape[1]
        ctx.set_materialize_grads(False)
        return normed, total

    @staticmethod
    @once_differentiable
    def backward(ctx, dnormed, dtotal):
        y, inv_sort_idx, weights, residual, gamma, rstd = ctx.saved_tensors
        rows, H = ctx.y_shape
        T, k = rstd.shape[0], ctx.k
        want_y, _, want_w, want_r, want_g = ctx.needs_input_grad[:5]
        if dnormed is None and dtotal is None:
            return (None,) * 7
        some = dtotal if dnormed is None else dnormed

        # (hooks on saved tensors may have given back another type, device or layout)
        def checked(t, shape, dtype=some.dtype):
            if t is not None and (t.shape != shape or t.dtype != dtype or t.device != some.device or not t.is_contiguous()):
                raise _lib.MoeB200Error("combine_add_rms_norm: a tensor of the backward pass has another type, device or layout "
                                        "than in the forward pass")
            return t

        dnormed = None if dnormed is None else checked(dnormed.contiguous(), (T, H))
        dtotal = None if dtotal is None else checked(dtotal.contiguous(), (T, H))
        checked(residual, (T, H)), checked(rstd, (T,), torch.float32), checked(gamma, (H,)), checked(y, (rows, H))
        checked(weights, (T, k)), checked(inv_sort_idx, (rows,), torch.int32)

        def out(want, *shape):
            return torch.empty(shape, device=some.device, dtype=some.dtype) if want else None

        dy, dw, dr, dg = out(want_y, rows, H), out(want_w, T, k), out(want_r, T, H), out(want_g, H)
        lib = _lib.load()
        nbytes = lib.moe_combine_add_rms_norm_bwd_ws_bytes(T, H) if want_g else 0
        here, stream = _lib.launch_on(some.device)
        with here:
            ws = torch.empty(nbytes, device=some.device, dtype=torch.uint8) if nbytes else None
            status = lib.moe_combine_add_rms_norm_bwd_inputs(
                _lib.ptr(dnormed), _lib.ptr(dtotal), _lib.ptr(residual), _lib.ptr(rstd), _lib.ptr(gamma), _lib.ptr(y),
                _lib.ptr(inv_sort_idx), _lib.ptr(weights), ctx.scale, _lib.ptr(dr), _lib.ptr(dy), _lib.ptr(dw), _lib.ptr(dg),
                T, k, H, _lib.float_code(some.dtype), _lib.ptr(ws), nbytes, stream)
        _lib.check(status, "moe_combine_add_rms_norm_bwd_inputs")
        return dy, None, dw, dr, dg, None, None


def _checked(rows: int, H: int, like: torch.Tensor, residual, weight):
    assert like.is_cuda
    assert weight.shape == (H,) and weight.dtype == like.dtype and weight.device == like.device
    if residual is not None:
        assert residual.dtype == like.dtype and residual.device == like.device
        assert residual.shape[-1:] == (H,) and residual.numel() == rows * H
        residual = residual.reshape(rows, H).contiguous()
    return residual, weight.contiguous()


def _run(y, inv_sort_idx, routing_weights, residual, weight, eps, scale):
    ts = (y, routing_weights, residual, weight)
    if _lib.has_tangent(*ts) or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)):
        return CombineAddRmsNorm.apply(y, inv_sort_idx, routing_weights, residual, weight, float(eps), float(scale))
    return _forward(y, inv_sort_idx, routing_weights, residual, weight, float(eps), float(scale), False)[:2]


def add_rms_norm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                 scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(normed, sum) with sum = residual + scale * x and normed = sum / sqrt(mean(sum^2) + eps) * weight over the last
    dimension (1 to 24576); `residual` None: zeros.  Both shaped like x.  x, residual and weight have one floating type; the
    arithmetic is fp32 and each output is rounded once.  Gradients for all three, once (no second derivative); x and residual are kept
    for them."""
    assert x.ndim >= 1 and x.shape[-1] >= 1
    H = x.shape[-1]
    rows = x.numel() // H
    residual, weight = _checked(rows, H, x, residual, weight)
    normed, total = _run(x.reshape(rows, H).contiguous(), None, None, residual, weight, eps, scale)
    return normed.view(x.shape), total.view(x.shape)


def combine_add_rms_norm(y: torch.Tensor, sort_idx: torch.Tensor, inv_sort_idx: torch.Tensor, routing_weights: torch.Tensor,
                         residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                         scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """`add_rms_norm` on the block's combined output, which is not written: with `routing_weights` (T, k) and the expert
    rows y (T * k, H) in sorted order, sum[t] = residual[t] + scale * sum_j routing_weights[t, j] * y[inv_sort_idx[t*k + j]].
    `sort_idx`, `inv_sort_idx`: as for `combine`, int32, each row once.  `residual`: T * H values; the outputs are shaped like it,
    (T, H) without one.  Gradients for y, routing_weights, residual and weight, once; all of them are kept for that."""
    assert y.ndim == 2 and routing_weights.ndim == 2 and y.shape[1] >= 1
    T, k = routing_weights.shape
    H = y.shape[1]
    assert k >= 1 and y.shape[0] == T * k
    for idx in (sort_idx, inv_sort_idx):
        assert idx.dtype == torch.int32 and idx.is_contiguous() and idx.numel() == T * k and idx.device == y.device
    assert routing_weights.dtype == y.dtype and routing_weights.device == y.device
    shape = (T, H) if residual is None else residual.shape
    residual, weight = _checked(T, H, y, residual, weight)
    normed, total = _run(y.contiguous(), inv_sort_idx.view(-1), routing_weights.contiguous(), residual, weight, eps, scale)
    return normed.view(shape), total.view(shape)
