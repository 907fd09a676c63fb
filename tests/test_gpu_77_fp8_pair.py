"""The CTA-pair kernel of the 8-bit products, forced on groups of any size: at the edges of its tiles (256 rows, 256 columns or 128
features, boxes of 16 rows), which the library's own choice gives to the kernel for few rows; and on every path what a NaN, an
infinity, rows behind the last group and skewed routing leave."""
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


SIZES = [[1], [0, 1, 15, 16, 17, 0], [31, 33, 2], [128, 129, 127], [255, 256, 257, 0, 1]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("K,N", [(256, 384), (16, 256), (720, 1008), (2048, 208), (128, 16), (1536, 144)])
def test_linear(cuda, pairs, dtype, sizes, K, N):
    products.test_linear_forward_and_gradient(cuda, pairs, dtype, sizes, K, N)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", [[1], [0, 1, 15, 16, 17, 0], [5, 128, 33, 257]], ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("H,I", [(256, 128), (400, 208), (2048, 768), (208, 1008), (128, 16)])
def test_mlp(cuda, pairs, dtype, sizes, H, I):
    products.test_mlp_forward_and_gradient(cuda, pairs, dtype, sizes, H, I)


def test_rows_next_to_nan_keep_their_bits(cuda, pairs):
    products.test_rows_next_to_nan_keep_their_bits(cuda, pairs)


def test_rows_behind_the_last_group_are_left(cuda, pairs):
    products.test_rows_behind_the_last_group_are_left(cuda, pairs)


# ------------------------------------------------------------------------------------------ the MLP on every path
@pytest.fixture(params=["PATH_AUTO", "PATH_SIMT", "PATH_TC", "PATH_TC_SINGLE"])
def each_path(request):
    from qwen3_moe_fused import _lib

    prev = _lib.set_gemm_path(getattr(_lib, request.param))
    yield request.param
    _lib.set_gemm_path(prev)
    torch.cuda.synchronize()
    assert _lib.read_error_flag() == 0


def mlp_weights(cuda, gen, E, H, I):
    unit = 2.0 / H ** 0.5
    return [products.fp8_weight(*shape, gen, cuda, unit) for shape in ((E, I, H), (E, I, H), (E, H, I))]


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("path", ["PATH_TC", "PATH_TC_SINGLE"])
def test_gate_up_leaves_rows_behind_the_last_group(cuda, path, keep):
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.quantize.fp8 import FP8, blocks, quantize_fp8_rows

    gen = products.gen_for(cuda, 41)
    M, H, I, rows = 100, 256, 208, 51
    (wg, gs), (wu, us), _ = mlp_weights(cuda, gen, 2, H, I)
    q, s = quantize_fp8_rows(torch.randn(M, H, generator=gen, device=cuda).to(torch.bfloat16))
    m_sizes = torch.tensor([30, rows - 30], device=cuda, dtype=torch.int32)
    hq = torch.full((M, I), 0x55, device=cuda, dtype=torch.uint8)
    hs = torch.full((blocks(I), M), 7.0, device=cuda)
    e, g = (torch.full((M, I), 7.0, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    p = _lib.ptr
    prev = _lib.set_gemm_path(getattr(_lib, path))
    try:
        st = _lib.load().moe_gate_up_silu_fp8(p(q), p(s), p(wg), p(gs), p(wu), p(us), p(m_sizes), _lib.I32, p(hq), p(hs),
                                              p(e) if keep else None, p(g) if keep else None, M, I, H, 2, _lib.BF16, _lib.stream_ptr(cuda))
        _lib.check(st, "moe_gate_up_silu_fp8")
        torch.cuda.synchronize()
        assert _lib.read_error_flag() == 0
    finally:
        _lib.set_gemm_path(prev)
    for t, old in ((hq, 0x55), (hs.t(), 7.0), (e, 7.0), (g, 7.0)):
        assert bool((t[rows:] == old).all())
    ys = [products.product(products.quantised(q.float() * s.t().repeat_interleave(128, 1)[:, :H])[0][:rows], products.decoded(*w), [30, rows - 30])
          for w in ((wg, gs), (wu, us))]
    h = ys[0][0] * torch.sigmoid(ys[0][0]) * ys[1][0]
    got = hq[:rows].view(FP8).double() * hs.t()[:rows].double().repeat_interleave(128, 1)[:, :I]
    # a code: half a step, 2^-4 of the value or 2^-10 of the block's scale, with 2^-9 for h's own sums where that moves it
    bound = h.abs() * 2.0 ** -4 * (1 + 2.0 ** -9) + hs.t()[:rows].double().repeat_interleave(128, 1)[:, :I] * 2.0 ** -9
    assert bool(((got - h).abs() <= bound).all())
    if keep:
        for t, (y, mag) in ((e, ys[0]), (g, ys[1])):
            assert bool(((t[:rows].double() - y).abs() <= 2.0 ** -8 * y.abs() + H * 2.0 ** -24 * mag + 2.0 ** -126).all())


def test_nan_and_infinity_stay_in_their_rows(cuda, each_path):
    """Through gate, up, their activation, the quantisation of h and down, and through the whole backward pass."""
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8

    gen = products.gen_for(cuda, 42)
    sizes, H, I = [40, 3, 300], 256, 208
    ws = [t for w in mlp_weights(cuda, gen, 3, H, I) for t in w]
    m_sizes = torch.tensor(sizes, device=cuda, dtype=torch.int32)
    x, dy = (torch.randn(sum(sizes), H, generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))

    def run(x, dy):
        x = x.clone().requires_grad_()
        y = moe_mlp_fp8(x, *ws, m_sizes)
        with torch.no_grad():
            assert torch.equal(moe_mlp_fp8(x, *ws, m_sizes).nan_to_num(9e9), y.nan_to_num(9e9))
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    y, dx = run(x, dy)
    assert torch.isfinite(y).all() and torch.isfinite(dx).all()
    odd = torch.tensor([float("nan"), float("inf"), float("-inf"), float("nan"), float("inf")], device=cuda, dtype=x.dtype)
    bad_x, bad_dy = [0, 39, 43, 100, 342], [1, 38, 42, 101, 341]
    x2, dy2 = x.clone(), dy.clone()
    x2[bad_x, 200], dy2[bad_dy, 3] = odd, odd
    y2, dx2 = run(x2, dy2)
    for got, want, bad in ((y2, y, bad_x), (dx2, dx, bad_x + bad_dy)):
        keep = [t for t in range(sum(sizes)) if t not in bad]
        assert torch.equal(got[keep], want[keep]) and bool(got[bad].isnan().all())


def test_skewed_routing_over_many_experts(cuda, each_path):
    """A few experts with most of the rows, many with a handful, some with one."""
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8

    gen = products.gen_for(cuda, 43)
    E, H, I, M, dtype = 128, 256, 128, 3001, torch.bfloat16
    ids = (torch.rand(M, generator=gen, device=cuda) ** 6 * E).long()
    m_sizes = torch.bincount(ids, minlength=E)[torch.randperm(E, generator=gen, device=cuda)]
    sizes = m_sizes.tolist()
    assert min(sizes) == 1 and max(sizes) > 1000
    ws = mlp_weights(cuda, gen, E, H, I)
    x = torch.randn(M, H, generator=gen, device=cuda).to(dtype).requires_grad_()
    dy = torch.randn(M, H, generator=gen, device=cuda).to(dtype)
    y = moe_mlp_fp8(x, *(t for w in ws for t in w), m_sizes)
    (dx,) = torch.autograd.grad(y, x, dy)
    for got, want in zip((y, dx), products.mlp_reference(x.detach(), ws, sizes, dy, dtype)):
        assert (got.double() - want).norm() / want.norm() <= torch.finfo(dtype).eps / 2 + 2.0 ** -8
