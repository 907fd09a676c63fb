"""The quantised SiLU-mul and its gradients of fp32 tensors: exponential and division of IEEE accuracy, over the whole range where the
sigmoid is a number that fp32 holds.

Tolerance: the exponential's rounding error (2 ulp), the sum's, the quotient's and two or three products' are 8 * 2^-24 together, and a
quotient below 2^-126 (e down to -88) is off by at most half of the smallest step, 2^-150, in place of 2^-24 of it.  Then one code:
half a step of e4m3, 2^-4 of the value or 2^-10 of the block's scale."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128


def decoded(q, s, n):
    return q.double() * s.double().t().repeat_interleave(BLOCK, 1)[:, :n]


def check(q, s, want, slack, what):
    n = want.shape[1]
    scale = s.double().t().repeat_interleave(BLOCK, 1)[:, :n]
    off = (decoded(q, s, n) - want).abs()
    bound = want.abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + scale * 2.0 ** -10 + slack
    assert bool((off <= bound).all()), f"{what}: {(off / bound).max().item():.2f} of the bound"


@pytest.mark.parametrize("I", [256, 200, 131])
def test_small_sigmoids(cuda, I):
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.quantize.fp8 import FP8, empty_scales

    gen = torch.Generator(device=cuda).manual_seed(I)
    M = 60
    lib, stream = _lib.load(), _lib.stream_ptr(cuda)
    e = -(torch.arange(M, device=cuda).float().view(M, 1) / (M - 1) * 8 + 80).expand(M, I).contiguous()  # -80 .. -88, a row each
    g = torch.randn(M, I, generator=gen, device=cuda) * 1e36
    dh = torch.randn(M, I, generator=gen, device=cuda)
    codes = lambda: (torch.empty(M, I, device=cuda, dtype=FP8), empty_scales(M, I, cuda))  # noqa: E731
    (hq, hs), (eq, es), (gq, gs) = codes(), codes(), codes()
    p = _lib.ptr
    _lib.check(lib.moe_fp8_silu_quantize(p(e), p(g), M, I, p(hq), p(hs), None, None, _lib.F32, stream), "moe_fp8_silu_quantize")
    _lib.check(lib.moe_fp8_silu_bwd_quantize(p(dh), p(e), p(g), M, I, p(eq), p(es), p(gq), p(gs), _lib.F32, stream),
               "moe_fp8_silu_bwd_quantize")
    e64, g64, dh64 = e.double(), g.double(), dh.double()
    sig = 1 / (1 + torch.exp(-e64))
    step = 2.0 ** -150
    check(hq, hs, e64 * sig * g64, step * 88 * g64.abs(), "h")
    assert bool((decoded(hq, hs, I)[-1].abs() > 0).any())  # e = -88: 5e-37 times 1e36
    check(eq, es, dh64 * g64 * sig * (1 + e64 * (1 - sig)), step * 88 * (dh64 * g64).abs(), "de")
    check(gq, gs, dh64 * e64 * sig, step * 88 * dh64.abs() + 2.0 ** -100, "dg")  # (below the smallest scale: zeros)
