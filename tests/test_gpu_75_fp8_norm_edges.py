"""8-bit products and norms where offsets pass 32 bits, with many experts, in captured backward passes, and on gradients and saved
tensors that a kernel cannot read."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def fp8_weight(E, N, K, gen, cuda):
    codes = (torch.randn(E, N, K, generator=gen, device=cuda) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, torch.rand(E, -(-N // 128), -(-K // 128), generator=gen, device=cuda) * 1e-3 + 1e-4


def mlp_weights(E, H, I, gen, cuda):
    return [t for shape in ((E, I, H), (E, I, H), (E, H, I)) for t in fp8_weight(*shape, gen, cuda)]


def test_captured_backward(cuda):
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8
    from qwen3_moe_fused.kernels.norm import combine_add_rms_norm

    gen = torch.Generator(device=cuda).manual_seed(1)
    T, k, H, E = 70, 4, 256, 4
    ws = mlp_weights(E, H, 128, gen, cuda)
    m_sizes = torch.tensor([100, 0, 30, 150], device=cuda, dtype=torch.int32)
    inv = torch.randperm(T * k, generator=gen, device=cuda).int()
    idx = torch.argsort(inv).int()
    normal = lambda *s: torch.randn(*s, generator=gen, device=cuda).to(torch.bfloat16)  # noqa: E731
    gamma, dn = normal(H), normal(T, H)
    inputs = [[normal(T * k, H), normal(T, k), normal(T, H)] for _ in range(2)]

    def step(x, w, r):
        x, w, r, g = (t.detach().requires_grad_() for t in (x, w, r, gamma))
        n, s = combine_add_rms_norm(moe_mlp_fp8(x, *ws, m_sizes), idx, inv, w, r, g)
        return (n, s, *torch.autograd.grad((n, s), (x, w, r, g), (dn, dn)))

    want = [[t.detach().clone() for t in step(*i)] for i in inputs]
    static = [t.clone() for t in inputs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for i in (0, 1, 0):
        for a, b in zip(static, inputs[i]):
            a.copy_(b)
        graph.replay()
        for a, b in zip(got, want[i]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("E", [1024, 1025, 1500])
def test_more_experts_than_the_tensor_core_form_takes(cuda, E):
    """1025 and more go to the other kernel: the first 1024 experts' rows agree with a call on those alone."""
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = torch.Generator(device=cuda).manual_seed(2)
    K, N = 64, 48
    codes, s = fp8_weight(E, N, K, gen, cuda)
    sizes = torch.randint(0, 4, (E,), generator=gen, device=cuda, dtype=torch.int32)
    sizes[-1] = 3
    M, first = int(sizes.sum()), int(sizes[:1024].sum())
    x = torch.randn(M, K, generator=gen, device=cuda, requires_grad=True)
    y = moe_fused_linear_fp8(x, codes, s, sizes)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.isfinite(y).all() and torch.isfinite(dx).all() and (y[-3:] != 0).any(1).all()
    xf = x.detach()[:first].requires_grad_()
    yf = moe_fused_linear_fp8(xf, codes[:1024], s[:1024], sizes[:1024])
    (dxf,) = torch.autograd.grad(yf, xf, torch.ones_like(yf))
    # sums of K and N <= 64 products in another order: 64 steps of 2^-24 of the sum of magnitudes, of which there are no more
    # than terms times the largest term: weights <= 448 * 1.1e-3, activations rounded up by at most 1/16
    bound = 64 * 2.0 ** -24 * 64 * 448 * 1.1e-3 * 17 / 16
    for a, b, top in ((y.detach()[:first], yf.detach(), x.detach().abs().amax().item()), (dx[:first], dxf, 1.0)):
        assert (a - b).abs().max().item() <= 2 * bound * max(top, 1.0)


def test_product_past_32_bits(cuda):
    """Offsets of x, its codes, y and dx pass 2^32 (elements or bytes): the last rows have the bits of a short call."""
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = torch.Generator(device=cuda).manual_seed(3)
    M, K, N, tail = (1 << 20) + 75, 4096, 2176, 300
    w, s = fp8_weight(2, N, K, gen, cuda)
    x = torch.randn(tail, K, generator=gen, device=cuda).to(torch.bfloat16)
    d = torch.randn(tail, N, generator=gen, device=cuda).to(torch.bfloat16)
    long = lambda t: torch.cat([t.new_zeros(M - tail, t.shape[1]), t])  # noqa: E731

    def run(x, d, sizes):
        x.requires_grad_()
        y = moe_fused_linear_fp8(x, w, s, torch.tensor(sizes, device=cuda))
        return y.detach(), torch.autograd.grad(y, x, d)[0]

    y, dx = run(x, d, [tail - 100, 100])
    yl, dxl = run(long(x.detach()), long(d), [M - 100, 100])
    assert torch.equal(yl[-tail:], y) and torch.equal(dxl[-tail:], dx)
    assert not yl[:-tail].any() and not dxl[:-tail].any()
    del yl, dxl
    torch.cuda.empty_cache()


def test_norm_past_32_bits(cuda):
    from qwen3_moe_fused.kernels.norm import combine_add_rms_norm

    gen = torch.Generator(device=cuda).manual_seed(4)
    T, k, H, tail = (1 << 17) + 3, 8, 4096, 40
    y = torch.randn(T * k // 64, H, generator=gen, device=cuda).to(torch.bfloat16)
    y = torch.cat([y] * 64 + [y[: T * k - y.shape[0] * 64]])
    inv = torch.randperm(T * k, generator=gen, device=cuda).int()
    idx = torch.argsort(inv).int()
    w, r = (torch.randn(T, n, generator=gen, device=cuda).to(torch.bfloat16) for n in (k, H))
    g = torch.randn(H, generator=gen, device=cuda).to(torch.bfloat16)
    dn = torch.randn(T, H, generator=gen, device=cuda).to(torch.bfloat16)

    def run(y, idx, inv, w, r, dn):
        y, w, r = (t.detach().requires_grad_() for t in (y, w, r))
        n, s = combine_add_rms_norm(y, idx, inv, w, r, g)
        return n.detach(), s.detach(), *torch.autograd.grad((n, s), (y, w, r), (dn, dn))

    at = inv[-tail * k:].long()
    one = torch.arange(tail * k, device=cuda, dtype=torch.int32)
    n, s, dy, dw, dr = run(y[at], one, one, w[-tail:], r[-tail:], dn[-tail:])
    assert at.max().item() * H > 1 << 31 and T * k * H > 1 << 32
    nl, sl, dyl, dwl, drl = run(y, idx, inv, w, r, dn)
    assert torch.equal(nl[-tail:], n) and torch.equal(sl[-tail:], s) and torch.equal(dyl[at], dy)
    assert torch.equal(dwl[-tail:], dw) and torch.equal(drl[-tail:], dr)
    del nl, sl, dyl, dwl, drl, y
    torch.cuda.empty_cache()


def test_batched_gradients_are_refused(cuda):
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8
    from qwen3_moe_fused.kernels.norm import add_rms_norm
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    gen = torch.Generator(device=cuda).manual_seed(5)
    ws = mlp_weights(2, 256, 128, gen, cuda)
    m = torch.tensor([1, 3], device=cuda)
    x = torch.randn(4, 256, generator=gen, device=cuda, requires_grad=True)
    g = torch.ones(256, device=cuda)
    for out in (moe_fused_linear_fp8(x, *ws[:2], m), moe_mlp_fp8(x, *ws, m), add_rms_norm(x, None, g)[0]):
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out, x, torch.ones(2, *out.shape, device=cuda), is_grads_batched=True)
    for call in (lambda t: moe_fused_linear_fp8(t, *ws[:2], m), lambda t: add_rms_norm(t, None, g)[0]):
        with torch.no_grad(), pytest.raises((RuntimeError, AssertionError)):
            torch.func.vmap(call)(x.detach().expand(2, 4, 256))


def test_saved_tensors_on_another_device_are_refused(cuda):
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8
    from qwen3_moe_fused.kernels.norm import add_rms_norm

    gen = torch.Generator(device=cuda).manual_seed(6)
    ws = mlp_weights(2, 256, 128, gen, cuda)
    m = torch.tensor([1, 3], device=cuda)
    x = torch.randn(4, 256, generator=gen, device=cuda).to(torch.bfloat16).requires_grad_()
    g = torch.ones(256, device=cuda, dtype=torch.bfloat16)
    moved = lambda dtype: torch.autograd.graph.saved_tensors_hooks(  # noqa: E731
        lambda t: t, lambda t: t.cpu() if t.dtype == dtype else t)
    with moved(torch.bfloat16):
        y, (n, _) = moe_mlp_fp8(x, *ws, m), add_rms_norm(x, None, g)
    with pytest.raises(AssertionError):
        torch.autograd.grad(y, x, torch.ones_like(y))
    with pytest.raises(_lib.MoeB200Error):
        torch.autograd.grad(n, x, torch.ones_like(n))
    for dtype in (torch.float8_e4m3fn, torch.float32, torch.int64):
        with moved(dtype):
            y = moe_mlp_fp8(x, *ws, m)
        with pytest.raises(AssertionError):
            torch.autograd.grad(y, x, torch.ones_like(y))


def test_layer_without_tokens(cuda):
    from qwen3_moe_fused.moe_block import moe_layer_forward

    gen = torch.Generator(device=cuda).manual_seed(7)
    E, H, I = 4, 256, 128
    ws = mlp_weights(E, H, I, gen, cuda)
    g = torch.ones(H, device=cuda, dtype=torch.bfloat16)
    router = torch.randn(E, H, generator=gen, device=cuda).to(torch.bfloat16)
    for grad in (False, True):
        x = torch.zeros(2, 0, H, device=cuda, dtype=torch.bfloat16, requires_grad=grad)
        n, out, logits = moe_layer_forward(x, x, g, router, ws, 2, g)
        assert n.shape == out.shape == x.shape and logits.shape == (0, E)
        if grad:
            assert torch.autograd.grad(n.sum() + out.sum(), x)[0].shape == x.shape
