"""The CTA-pair kernel of the 8-bit products, forced on groups of any size."""
import pytest
import torch

from . import test_gpu_73_fp8 as products

pytestmark = pytest.mark.gpu


@pytest.fixture
def pairs():
    from qwen3_moe_fused import _lib

    prev = _lib.set_gemm_path(_lib.PATH_TC)
    yield "pairs"
    _lib.set_gemm_path(prev)
    torch.cuda.synchronize()
    assert _lib.read_error_flag() == 0


@pytest.mark.parametrize("path", ["PATH_TC", "PATH_TC_SINGLE"])
def test_scales_of_any_alignment(cuda, path):
    """Scales that start between two 16-byte units: the tensor-core kernels take them, with the same bits."""
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_rows

    gen = products.gen_for(cuda, 21)
    M, K, N, E = 200, 384, 256, 2
    codes, ws = products.fp8_weight(E, N, K, gen, cuda)
    q, s = quantize_fp8_rows(torch.randn(M, K, generator=gen, device=cuda).to(torch.bfloat16))
    m_sizes = torch.tensor([130, 70], device=cuda, dtype=torch.int32)
    y = torch.empty(M, N, device=cuda, dtype=torch.bfloat16)
    prev = _lib.set_gemm_path(getattr(_lib, path))
    try:
        got = []
        for offset in (0, 1, 2, 3):
            base = torch.empty(s.shape[0] * s.stride(0) + offset, device=cuda)[offset:]
            scales = base.as_strided(s.shape, s.stride())
            scales.copy_(s)
            st = _lib.load().moe_grouped_gemm_fp8(0, q.data_ptr(), scales.data_ptr(), codes.data_ptr(), ws.data_ptr(), None, None, None,
                                                  None, m_sizes.data_ptr(), _lib.I32, y.data_ptr(), M, N, K, E, _lib.BF16,
                                                  _lib.stream_ptr(cuda))
            _lib.check(st, "moe_grouped_gemm_fp8")
            got.append(y.clone())
        assert all(torch.equal(g, got[0]) for g in got)
        torch.cuda.synchronize()
        assert _lib.read_error_flag() == 0
    finally:
        _lib.set_gemm_path(prev)


@pytest.mark.parametrize("K,N", [(2048, 1536), (128, 512), (384, 208)])
def test_the_same_bits_in_every_run(cuda, pairs, K, N):
    """Accumulators are handed back and overwritten a few hundred cycles after they are read: a reading that came late would show."""
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = products.gen_for(cuda, K)
    codes, s = products.fp8_weight(16, N, K, gen, cuda)
    sizes = torch.bincount((torch.rand(9001, generator=gen, device=cuda) ** 2 * 16).long(), minlength=16)
    x = torch.randn(9001, K, generator=gen, device=cuda).to(torch.bfloat16).requires_grad_()
    dy = torch.randn(9001, N, generator=gen, device=cuda).to(torch.bfloat16)

    def run():
        y = moe_fused_linear_fp8(x, codes, s, sizes)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    want = run()
    differ = torch.zeros((), device=cuda, dtype=torch.int64)
    for _ in range(200):
        for a, b in zip(run(), want):
            differ += (a != b).sum()
    assert differ.item() == 0
