"""8-bit weights with a scale for each block of 128 x 128, and 8-bit activations with one for each 128 values of a row.

Weights are what checkpoints in 8 bits hold: e4m3 codes shaped like the weight and an fp32 scale for each block,
weight = code * scale.  Any positive scales will do; `quantize_fp8` takes largest magnitude / 448.

Activations are quantised where they are used: the scale of a block is the smallest power of two with
max|x| <= 448 * scale (at least 2^-100), the code is x / scale rounded to the nearest e4m3 value, ties to even.  A power of two
takes no precision from e4m3, makes the division exact and the codes independent of the precision they are computed in.
A block with an infinity or a NaN gets the scale NaN.

The reference quantises to 4 bits only (qwen3_moe_fused/quantize/layer.py).
"""
from __future__ import annotations

import torch

from .. import _lib

BLOCK = 128
FP8 = torch.float8_e4m3fn


def blocks(n: int) -> int:
    return -(-n // BLOCK)


@torch.no_grad()
def quantize_fp8(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale) of a weight (E, out, in): e4m3 codes of the same shape, fp32 (E, ceil(out / 128), ceil(in / 128))."""
    assert weight.ndim == 3
    E, N, K = weight.shape
    nb, kb = blocks(N), blocks(K)
    codes = torch.empty((E, N, K), device=weight.device, dtype=FP8)
    scale = torch.empty((E, nb, kb), device=weight.device, dtype=torch.float32)
    for e in range(E):  # one expert at a time: the fp32 copy stays small
        w = weight[e].float()
        w = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N)).view(nb, BLOCK, kb, BLOCK)
        s = w.abs().amax(dim=(1, 3)) / 448
        s = torch.where(s > 0, s, torch.ones_like(s))
        scale[e] = s
        codes[e] = (w / s.view(nb, 1, kb, 1)).clamp(-448, 448).to(FP8).view(nb * BLOCK, kb * BLOCK)[:N, :K]
    return codes, scale


def dequantize_fp8(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that the codes of a weight stand for."""
    check_weight(codes, scale)
    _, N, K = codes.shape
    return (codes.float() * scale.repeat_interleave(BLOCK, 1)[:, :N].repeat_interleave(BLOCK, 2)[:, :, :K]).to(dtype)


def check_weight(codes: torch.Tensor, scale: torch.Tensor) -> None:
    assert codes.ndim == 3 and codes.dtype == FP8 and codes.is_contiguous()
    assert scale.dtype == torch.float32 and scale.device == codes.device and scale.is_contiguous()
    assert scale.shape == (codes.shape[0], blocks(codes.shape[1]), blocks(codes.shape[2]))


def empty_scales(M: int, K: int, device) -> torch.Tensor:
    """(ceil(K / 128), M) with rows padded to a multiple of 4, as the kernels lay them out."""
    return torch.empty((blocks(K), -(-M // 4) * 4), device=device, dtype=torch.float32)[:, :M]


@torch.no_grad()
def quantize_fp8_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes (M, K), scale (ceil(K / 128), M)) of activations x (M, K): x[m, k] is about codes[m, k] * scale[k // 128, m]."""
    assert x.is_cuda and x.ndim == 2 and x.is_contiguous() and x.shape[1] >= 1
    M, K = x.shape
    q = torch.empty((M, K), device=x.device, dtype=FP8)
    s = empty_scales(M, K, x.device)
    here, stream = _lib.launch_on(x.device)
    with here:
        status = _lib.load().moe_fp8_quantize_rows(_lib.ptr(x), _lib.float_code(x.dtype), M, K, _lib.ptr(q), _lib.ptr(s),
                                                   stream)
    _lib.check(status, "moe_fp8_quantize_rows")
    return q, s
