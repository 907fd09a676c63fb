"""moe_layer_forward: norm, block, residual and next norm as they follow one another, on 16-bit and on 8-bit experts."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(cuda, dtype, B, S, H, I, E, seed=0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    normal = lambda c, *s: (torch.randn(*s, device=cuda, generator=gen) * c).to(dtype)  # noqa: E731
    return {"hidden": normal(1, B, S, H), "residual": normal(1, B, S, H), "norm": (1 + normal(0.1, H)).to(dtype),
            "router": normal(H ** -0.5, E, H), "gate": normal(H ** -0.5, E, I, H), "up": normal(H ** -0.5, E, I, H),
            "down": normal(I ** -0.5, E, H, I), "next": (1 + normal(0.1, H)).to(dtype), "dn": normal(1, B, S, H), "ds": normal(1, B, S, H)}


def exact(d, selected, k, scale, eps):
    """The layer in 64 bits, with the experts that the kernels selected."""
    norm = lambda s, w: s * (s.square().mean(-1, keepdim=True) + eps).rsqrt() * w  # noqa: E731
    H = d["hidden"].shape[-1]
    stream = (d["hidden"] + d["residual"]).view(-1, H)
    n = norm(stream, d["norm"])
    w = torch.softmax(n @ d["router"].t(), 1).gather(1, selected)
    w = w / w.sum(1, keepdim=True)
    block = torch.zeros_like(stream)
    for j in range(k):
        e = selected[:, j]
        a, b = torch.einsum("tih,th->ti", d["gate"][e], n), torch.einsum("tih,th->ti", d["up"][e], n)
        block = block + w[:, j:j + 1] * torch.einsum("thi,ti->th", d["down"][e], torch.nn.functional.silu(a) * b)
    out = stream + scale * block
    return norm(out, d["next"]), out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_against_its_definition(cuda, dtype):
    from qwen3_moe_fused.moe_block import moe_layer_forward, route

    B, S, H, I, E, k, scale, eps = 2, 33, 256, 192, 8, 2, 0.75, 1e-6
    d = make(cuda, dtype, B, S, H, I, E)
    names = ("hidden", "residual", "norm", "router", "gate", "up", "down", "next")
    leaves = [d[m].requires_grad_() for m in names]
    args = (d["hidden"], d["residual"], d["norm"], d["router"], (d["gate"], d["up"], d["down"]), k, d["next"], True, eps, scale)
    normed, out, logits = moe_layer_forward(*args)
    grads = torch.autograd.grad((normed, out), leaves, (d["dn"], d["ds"]))
    _, selected = route(logits.detach(), k, True, dtype)
    d64 = {m: t.detach().double().requires_grad_(m in names) for m, t in d.items()}
    n64, o64 = exact(d64, selected, k, scale, eps)
    want = torch.autograd.grad((n64, o64), [d64[m] for m in names], (d64["dn"].view_as(n64), d64["ds"].view_as(o64)))
    # chains of at most twelve roundings one after the other (norm, logits, weights, three products, activation, combine and
    # back), each at most eps / 2 of what it applies to: 2-norm over 2-norm.  The router's gradient is what is left where the
    # renormalised weights cancel: its chain applies to terms up to four times its size here.
    bound = 12 * torch.finfo(dtype).eps / 2
    for name, got, ref in zip(("normed", "out", *names), (normed, out, *grads), (n64, o64, *want)):
        off = ((got.double().view_as(ref) - ref).norm() / ref.norm()).item()
        assert off <= bound * (4 if name == "router" else 1), f"{name}: {off:.2e}"
    with torch.no_grad():
        again = moe_layer_forward(*args)
    assert all(torch.equal(a, b) for a, b in zip(again, (normed, out, logits)))


@pytest.mark.parametrize("T", [1, 3, 300])
def test_layer_on_8_bit_experts(cuda, T):
    """The layer is its parts, bit for bit, with and without gradients, and replays in a graph."""
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8
    from qwen3_moe_fused.kernels.indexing import get_expert_counts_and_idx
    from qwen3_moe_fused.kernels.norm import add_rms_norm, combine_add_rms_norm
    from qwen3_moe_fused.kernels.routing import gather_rows
    from qwen3_moe_fused.moe_block import moe_layer_forward, route
    from qwen3_moe_fused.quantize.fp8 import quantize_fp8

    H, I, E, k = 256, 128, 8, 2
    d = make(cuda, torch.bfloat16, 1, T, H, I, E, seed=1)
    proj = [t for m in ("gate", "up", "down") for t in quantize_fp8(d[m])]
    args = (d["hidden"], d["residual"], d["norm"], d["router"], proj, k, d["next"])

    def parts():
        n, stream = add_rms_norm(d["hidden"], d["residual"], d["norm"])
        logits = torch.nn.functional.linear(n.view(T, H), d["router"])
        w, sel = route(logits, k, True, n.dtype)
        sizes, si, ii = get_expert_counts_and_idx(sel.view(T * k), E)
        y = moe_mlp_fp8(gather_rows(n.view(T, H), si, ii, k), *proj, sizes)
        return (*combine_add_rms_norm(y, si, ii, w, stream, d["next"]), logits)

    with torch.no_grad():
        want = parts()
        got = moe_layer_forward(*args)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            moe_layer_forward(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cap = moe_layer_forward(*args)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(cap, want))
    leaves = [d[m].requires_grad_() for m in ("hidden", "residual", "norm", "router", "next")]
    one = torch.autograd.grad(moe_layer_forward(*args)[:2], leaves, (d["dn"], d["ds"]))
    two = torch.autograd.grad(parts()[:2], leaves, (d["dn"], d["ds"]))
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(one, two))


def test_layer_refuses_other_projections(cuda):
    from qwen3_moe_fused.moe_block import moe_layer_forward

    d = make(cuda, torch.bfloat16, 1, 2, 64, 32, 4)
    with pytest.raises(AssertionError):
        moe_layer_forward(d["hidden"], None, d["norm"], d["router"], (d["gate"], d["up"]), 2, d["next"])
