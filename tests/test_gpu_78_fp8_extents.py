"""8-bit rows of the longest extent that is taken, 2^24, in every form of the quantising kernels: the ends of a row have the codes and
scales of a call on those columns alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LONGEST = 1 << 24


def ends(K):
    """Columns of the first blocks and of the last ones."""
    return (slice(0, 640), slice((K - 1) // 128 * 128 - 1280, K))


def values(shape, cuda, dtype, seed):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randn(*shape, generator=gen, device=cuda).to(dtype)


def same(q, s, cols, want_q, want_s):
    blocks = slice(cols.start // 128, (cols.stop + 127) // 128)
    assert torch.equal(q[:, cols].view(torch.uint8), want_q.view(torch.uint8)) and torch.equal(s[blocks], want_s)


@pytest.mark.parametrize("K,offset", [(LONGEST, 0), (LONGEST, 1), (LONGEST - 1, 0), (LONGEST - 255, 0)])
def test_quantised_rows(cuda, K, offset):
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_rows

    x = values((2 * K + offset,), cuda, torch.bfloat16, K)[offset:].view(2, K)
    q, s = quantize_fp8_rows(x)
    for cols in ends(K):
        same(q, s, cols, *quantize_fp8_rows(x[:, cols].contiguous()))


@pytest.mark.parametrize("K", [LONGEST, LONGEST - 3])
def test_activation_and_its_gradients(cuda, K):
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.quantize.fp8 import FP8, empty_scales

    lib, stream = _lib.load(), _lib.stream_ptr(cuda)
    codes = lambda M, n: (torch.empty(M, n, device=cuda, dtype=FP8), empty_scales(M, n, cuda))  # noqa: E731

    def forward(e, g):
        M, n = e.shape
        q, s = codes(M, n)
        _lib.check(lib.moe_fp8_silu_quantize(_lib.ptr(e), _lib.ptr(g), M, n, _lib.ptr(q), _lib.ptr(s), None, None, _lib.BF16, stream), "fwd")
        return ((q, s),)

    def backward(dh, e, g):
        M, n = e.shape
        (eq, es), (gq, gs) = codes(M, n), codes(M, n)
        _lib.check(lib.moe_fp8_silu_bwd_quantize(_lib.ptr(dh), _lib.ptr(e), _lib.ptr(g), M, n, _lib.ptr(eq), _lib.ptr(es), _lib.ptr(gq),
                                                 _lib.ptr(gs), _lib.BF16, stream), "bwd")
        return (eq, es), (gq, gs)

    f32, b16 = torch.float32, torch.bfloat16
    for call, dtypes in ((forward, (f32, f32)), (backward, (f32, b16, b16))):
        inputs = [values((1, K), cuda, dt, i) for i, dt in enumerate(dtypes)]
        got = call(*inputs)
        for cols in ends(K):
            for (q, s), (want_q, want_s) in zip(got, call(*(t[:, cols].contiguous() for t in inputs))):
                same(q, s, cols, want_q, want_s)
