"""Expert products on 8-bit weights and the gated MLP on them, against their definitions in 64 bits.

Tolerances, d = eps / 2 of the output type.  Codes and scales: none.  A product: its terms are exact in fp32 and a sum of n
terms in fp32 is off by at most n 2^-24 of the sum of magnitudes (`mag`), in any order; then one rounding.  The MLP quantises
h, which is off by a few 2^-20 (sums, exponential): where that crosses the border between two codes, one value in 2^13 or fewer
(steps are 2^-3 to 2^-4 of a value), the result differs by a step, 2^-9.5 of the result's 2-norm together; kept projections that
round the other way, one in 2^10, move de and dg by 2 d each, which crosses a border for one value in 8 or fewer and adds as
much again.  2-norms are held to d + 2^-8."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK = 128


def gen_for(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def fp8_weight(E, N, K, gen, cuda, scale=0.05):
    """Codes over e4m3's whole range and scales that are no powers of two."""
    codes = (torch.randn(E, N, K, generator=gen, device=cuda) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(E, -(-N // BLOCK), -(-K // BLOCK), generator=gen, device=cuda) * scale / 100 + scale / 200
    return codes, s


def decoded(codes, s):
    N, K = codes.shape[1:]
    return codes.double() * s.double().repeat_interleave(BLOCK, 1)[:, :N].repeat_interleave(BLOCK, 2)[:, :, :K]


def quantised(x):
    """(values, scales (blocks, M)) in 64 bits."""
    x = x.double()
    M, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % BLOCK)).view(M, -1, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    s = torch.exp2(torch.ceil(torch.log2(top.clamp_min(2.0 ** -140) / 448)).clamp_min(-100))
    s = torch.where(top > 448 * s, 2 * s, s)
    s = torch.where((top <= 224 * s) & (s > 2.0 ** -100), s / 2, s)
    v = b / s
    step = torch.exp2(torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent.double() - 4)
    return ((v / step).round() * step * s).view(M, -1)[:, :K], s.squeeze(2).t()


def product(xq, w, sizes, transposed=False):
    """(values, sums of magnitudes) per expert."""
    out = [(r @ m, r.abs() @ m.abs()) for r, m in ((r, w[e] if transposed else w[e].t()) for e, r in enumerate(xq.split(sizes)))]
    return tuple(torch.cat(t) for t in zip(*out))


def close(got, want, mag, n, dtype, what):
    d = torch.finfo(dtype).eps / 2
    assert got.dtype == dtype and torch.isfinite(got).all(), what
    off = (got.double() - want).abs()
    bound = d * want.abs() + max(n, 64) * 2.0 ** -24 * mag + torch.finfo(dtype).tiny
    assert bool((off <= bound).all()), f"{what}: {(off / bound.clamp_min(1e-300)).max().item():.2f} of the bound"


@pytest.fixture(params=["auto", "simt"])
def path(request):
    from qwen3_moe_fused import _lib

    prev = _lib.set_gemm_path(_lib.PATH_AUTO if request.param == "auto" else _lib.PATH_SIMT)
    yield request.param
    _lib.set_gemm_path(prev)
    torch.cuda.synchronize()
    assert _lib.read_error_flag() == 0


# ------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 128), (3, 2048), (70, 1008), (5, 1), (9, 257), (2, 120), (1000, 768), (4, 136)])
def test_quantised_rows(cuda, dtype, M, K):
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_rows

    gen = gen_for(cuda, M + K)
    x = torch.randn(M, K, generator=gen, device=cuda) * torch.exp2(torch.randint(-12, 12, (M, 1), generator=gen, device=cuda))
    x[0, 0] = 0
    if K > 8:
        x[-1, : K // 2] = 0  # blocks of zeros, and a block that is partly zeros
        x[M // 2, 1], x[M // 2, 2], x[M // 2, 3] = 448.0, 449.0, -1e-6
    x = x.to(dtype)
    q, s = quantize_fp8_rows(x)
    values, scales = quantised(x)
    assert q.shape == (M, K) and s.shape == (-(-K // BLOCK), M)
    assert torch.equal(s.double(), scales)
    got = q.double() * s.double().t().repeat_interleave(BLOCK, 1)[:, :K]
    assert torch.equal(got, values)


@pytest.mark.parametrize("top,expect", [(448.0, 1.0), (448.5, 2.0), (224.0, 0.5), (224.5, 1.0), (1.75, 2.0 ** -8), (2.0, 2.0 ** -7),
                                        (2.0 ** -126, 2.0 ** -100), (1e-45, 2.0 ** -100), (3e38, 2.0 ** 120)])
def test_scale_at_its_borders(cuda, top, expect):
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_rows

    x = torch.zeros(2, 128, device=cuda)
    x[1, 77] = -top
    q, s = quantize_fp8_rows(x)
    assert s[0, 1].item() == expect and s[0, 0].item() == 2.0 ** -100
    assert q.float().abs().max().item() == (torch.tensor(x[1, 77].double().abs().item() / expect, dtype=torch.float64)
                                            .to(torch.float8_e4m3fn).float().item())


def test_infinity_and_nan_mark_their_block(cuda):
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_rows

    x = torch.ones(4, 300, device=cuda, dtype=torch.bfloat16)
    x[1, 5], x[2, 130], x[2, 299] = float("nan"), float("inf"), float("-inf")
    _, s = quantize_fp8_rows(x)
    want = torch.zeros(3, 4, dtype=torch.bool, device=cuda)
    want[0, 1] = want[1, 2] = want[2, 2] = True
    assert torch.equal(s.isnan(), want)


def test_weight_codes_stand_for_the_weight(cuda):
    from qwen3_moe_fused.quantize.fp8 import dequantize_fp8, quantize_fp8

    w = torch.randn(3, 200, 300, generator=gen_for(cuda, 1), device=cuda)
    w[1] = 0
    codes, s = quantize_fp8(w)
    assert codes.shape == w.shape and s.shape == (3, 2, 3)
    back = dequantize_fp8(codes, s)
    assert torch.equal(back[1], w[1])
    # half a step of e4m3: 2^-4 of a value, or half of the smallest step, 2^-10 of the block's scale
    s_all = s.repeat_interleave(BLOCK, 1)[:, :200].repeat_interleave(BLOCK, 2)[:, :, :300]
    assert bool(((back - w).abs() <= w.abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + s_all * 2.0 ** -10).all())


# ------------------------------------------------------------------------------------------ products
SIZES = [[300], [1], [0, 1, 15, 16, 17, 0], [255, 256, 257, 0, 1], [511, 513, 40], [64, 65, 31, 33, 128], [0, 0, 700, 0]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("K,N", [(256, 384), (2048, 208), (720, 1008), (128, 512), (130, 70), (16, 256), (1536, 200)])
def test_linear_forward_and_gradient(cuda, path, dtype, sizes, K, N):
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = gen_for(cuda, sum(sizes) + K + N)
    E, M = len(sizes), sum(sizes)
    codes, s = fp8_weight(E, N, K, gen, cuda)
    x = (torch.randn(M, K, generator=gen, device=cuda)).to(dtype).requires_grad_()
    dy = (torch.randn(M, N, generator=gen, device=cuda)).to(dtype)
    m_sizes = torch.tensor(sizes, device=cuda, dtype=torch.int64 if N == 384 else torch.int32)
    y = moe_fused_linear_fp8(x, codes, s, m_sizes)
    (dx,) = torch.autograd.grad(y, x, dy)
    w = decoded(codes, s)
    close(y.detach(), *product(quantised(x.detach())[0], w, sizes), K, dtype, "y")
    close(dx, *product(quantised(dy)[0], w, sizes, True), N, dtype, "dx")
    with torch.no_grad():
        assert torch.equal(moe_fused_linear_fp8(x, codes, s, m_sizes), y)


@pytest.mark.parametrize("skew", [False, True])
def test_many_experts(cuda, skew):
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = gen_for(cuda, 11)
    E, K, N, M = 128, 768, 512, 9001
    codes, s = fp8_weight(E, N, K, gen, cuda)
    ids = (torch.rand(M, generator=gen, device=cuda) ** (4 if skew else 1) * E).long()
    m_sizes = torch.bincount(ids, minlength=E)
    x = torch.randn(M, K, generator=gen, device=cuda).to(torch.bfloat16).requires_grad_()
    dy = torch.randn(M, N, generator=gen, device=cuda).to(torch.bfloat16)
    y = moe_fused_linear_fp8(x, codes, s, m_sizes)
    (dx,) = torch.autograd.grad(y, x, dy)
    w, sizes = decoded(codes, s), m_sizes.tolist()
    close(y.detach(), *product(quantised(x.detach())[0], w, sizes), K, torch.bfloat16, "y")
    close(dx, *product(quantised(dy)[0], w, sizes, True), N, torch.bfloat16, "dx")


def test_rows_next_to_nan_keep_their_bits(cuda, path):
    """A row with a NaN or an infinity is all NaN; every other row, in the same group and in the next, keeps its bits."""
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = gen_for(cuda, 12)
    sizes = [40, 3, 300]
    codes, s = fp8_weight(3, 256, 384, gen, cuda)
    x = torch.randn(sum(sizes), 384, generator=gen, device=cuda).to(torch.bfloat16)
    m_sizes = torch.tensor(sizes, device=cuda)
    y = moe_fused_linear_fp8(x, codes, s, m_sizes)
    bad = [0, 39, 43, 100, 342]
    x2 = x.clone()
    x2[bad, 200] = torch.tensor([float("nan"), float("inf"), float("-inf"), float("nan"), float("inf")], device=cuda, dtype=x.dtype)
    y2 = moe_fused_linear_fp8(x2, codes, s, m_sizes)
    keep = [t for t in range(sum(sizes)) if t not in bad]
    assert torch.equal(y2[keep], y[keep]) and bool(y2[bad].isnan().all())


def test_rows_behind_the_last_group_are_left(cuda, path):
    from qwen3_moe_fused import _lib

    gen = gen_for(cuda, 13)
    codes, s = fp8_weight(2, 256, 256, gen, cuda)
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8_rows
    x = torch.randn(100, 256, generator=gen, device=cuda).to(torch.bfloat16)
    q, sx = quantize_fp8_rows(x)
    y = torch.full((100, 256), 7.0, device=cuda, dtype=torch.bfloat16)
    m_sizes = torch.tensor([30, 21], device=cuda, dtype=torch.int32)
    for which in (0, 1):
        y.fill_(7.0)
        st = _lib.load().moe_grouped_gemm_fp8(which, q.data_ptr(), sx.data_ptr(), codes.data_ptr(), s.data_ptr(), None, None, None, None,
                                              m_sizes.data_ptr(), _lib.I32, y.data_ptr(), 100, 256, 256, 2, _lib.BF16,
                                              _lib.stream_ptr(cuda))
        _lib.check(st, "moe_grouped_gemm_fp8")
        assert bool((y[51:] == 7).all()) and bool((y[:51] != 7).any())


# ------------------------------------------------------------------------------------------ MLP
def mlp_reference(x, ws, sizes, dy, dtype):
    wg, wu, wd = (decoded(*w) for w in ws)
    xq = quantised(x)[0]
    e, g = product(xq, wg, sizes)[0], product(xq, wu, sizes)[0]
    y = product(quantised(e * torch.sigmoid(e) * g)[0], wd, sizes)[0]
    e, g = e.to(dtype).double(), g.to(dtype).double()
    dh = product(quantised(dy)[0], wd, sizes, True)[0]
    sig = torch.sigmoid(e)
    de, dg = dh * g * sig * (1 + e * (1 - sig)), dh * e * sig
    return y, product(quantised(de)[0], wg, sizes, True)[0] + product(quantised(dg)[0], wu, sizes, True)[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", [[300, 0, 20], [1], [0, 16, 257, 513], [5, 64, 700, 33]], ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("H,I", [(256, 128), (512, 384), (400, 208), (2048, 768), (70, 36), (208, 1008)])
def test_mlp_forward_and_gradient(cuda, path, dtype, sizes, H, I):
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8

    gen = gen_for(cuda, sum(sizes) + H + I)
    E, M = len(sizes), sum(sizes)
    unit = 2.0 / H ** 0.5
    ws = [fp8_weight(E, I, H, gen, cuda, unit), fp8_weight(E, I, H, gen, cuda, unit), fp8_weight(E, H, I, gen, cuda, unit)]
    x = torch.randn(M, H, generator=gen, device=cuda).to(dtype).requires_grad_()
    dy = torch.randn(M, H, generator=gen, device=cuda).to(dtype)
    m_sizes = torch.tensor(sizes, device=cuda, dtype=torch.int32)
    flat = [t for w in ws for t in w]
    y = moe_mlp_fp8(x, *flat, m_sizes)
    (dx,) = torch.autograd.grad(y, x, dy)
    want_y, want_dx = mlp_reference(x.detach(), ws, sizes, dy, dtype)
    for got, want, what in ((y, want_y, "y"), (dx, want_dx, "dx")):
        off = (got.double() - want).norm() / want.norm()
        assert off <= torch.finfo(dtype).eps / 2 + 2.0 ** -8, f"{what}: {off:.2e}"
    with torch.no_grad():
        assert torch.equal(moe_mlp_fp8(x, *flat, m_sizes), y)


def test_no_rows(cuda):
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = gen_for(cuda, 14)
    wg, wd = fp8_weight(3, 128, 256, gen, cuda), fp8_weight(3, 256, 128, gen, cuda)
    x = torch.empty(0, 256, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    m_sizes = torch.zeros(3, device=cuda, dtype=torch.int32)
    for y in (moe_fused_linear_fp8(x, *wg, m_sizes), moe_mlp_fp8(x, *wg, *wg, *wd, m_sizes)):
        (dx,) = torch.autograd.grad(y.sum(), x)
        assert y.shape[0] == 0 and dx.shape == x.shape


def test_graph_replay_and_other_stream(cuda):
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8

    gen = gen_for(cuda, 15)
    ws = [t for shape in ((4, 256, 512), (4, 256, 512), (4, 512, 256)) for t in fp8_weight(*shape, gen, cuda)]
    m_sizes = torch.tensor([100, 0, 30, 70], device=cuda, dtype=torch.int32)
    xa, xb = (torch.randn(200, 512, generator=gen, device=cuda).to(torch.bfloat16) for _ in range(2))
    with torch.no_grad():
        ya, yb = moe_mlp_fp8(xa, *ws, m_sizes), moe_mlp_fp8(xb, *ws, m_sizes)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ys = [moe_mlp_fp8(x, *ws, m_sizes) for x in (xa, xb)]
        ym = moe_mlp_fp8(xa, *ws, m_sizes)  # beside the other stream's
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(ys[0], ya) and torch.equal(ys[1], yb) and torch.equal(ym, ya)
        x, sz = xa.clone(), m_sizes.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = moe_mlp_fp8(x, *ws, sz)
        x.copy_(xb)
        graph.replay()
        assert torch.equal(y, yb)
        sz.copy_(torch.tensor([0, 150, 50, 0], device=cuda))  # another routing in the same graph
        graph.replay()
        assert torch.equal(y, moe_mlp_fp8(xb, *ws, sz))


def test_refusals(cuda):
    import torch.autograd.forward_ad as fw
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = gen_for(cuda, 16)
    codes, s = fp8_weight(2, 128, 256, gen, cuda)
    x = torch.ones(4, 256, device=cuda, dtype=torch.bfloat16)
    m = torch.tensor([1, 3], device=cuda)
    good = (x, codes, s, m)
    moe_fused_linear_fp8(*good)
    bad = [(x.t(), codes, s, m), (x[:, :128], codes, s, m), (x, codes.float(), s, m), (x, codes, s.double(), m), (x, codes, s[:, :, :1], m),
           (x, codes, s.cpu(), m), (x, codes, s, m[:1]), (x, codes, s, m.float()), (x, codes, s, m.cpu()), (x.cpu(), codes, s, m),
           (x, codes.transpose(1, 2), s.transpose(1, 2), m), (x.view(2, 2, 256), codes, s, m)]
    for args in bad:
        with pytest.raises(AssertionError):
            moe_fused_linear_fp8(*args)
    with pytest.raises(_lib.MoeB200Error):
        moe_fused_linear_fp8(x.double(), codes, s, m)
    down = fp8_weight(2, 256, 64, gen, cuda)
    with pytest.raises(AssertionError):
        moe_mlp_fp8(x, codes, s, codes, s, *down, m)
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(moe_fused_linear_fp8(xr, codes, s, m).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    with torch.no_grad(), fw.dual_level(), pytest.raises(NotImplementedError):
        moe_fused_linear_fp8(fw.make_dual(x, torch.ones_like(x)), codes, s, m)
