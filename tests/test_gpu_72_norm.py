"""combine_add_rms_norm and add_rms_norm, forward and backward, against the formulas in 64 bits.

Tolerances.  With d = eps / 2 of the type (one rounding) the forward's outputs are off by d of the value and by fp32 sums of at
most 64 terms one after the other (2^-18 of the sum of magnitudes, `mag`).  The backward reads s as it was stored, each value
off by d |s| + 2^-18 mag: u = s r is off by Du = d |u| + 2^-18 r mag.  ds = .. - r u mean(a u) is off by at most
r (|Du| |mean(a u)| + |u| mean(|a| |Du|)), a row of it, with rms(u) <= 1, by 2 r ||a|| rms(Du) in the 2-norm, and what is computed
from ds by that times the other factor; dgamma by the sum of |dn| Du.  Each result is rounded once more."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SLACK = 2.0 ** -18
EPS = 1e-6


def make(cuda, T, H, k, dtype, seed=0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen, device=cuda).to(dtype)  # noqa: E731
    perm = torch.randperm(T * k, generator=gen, device=cuda)
    d = {"y": normal(T * k, H), "w": torch.rand(T, k, generator=gen, device=cuda).to(dtype), "residual": normal(T, H),
         "gamma": (1 + 0.1 * normal(H)).to(dtype), "dn": normal(T, H), "ds": normal(T, H),
         "inv": perm.to(torch.int32), "sort": torch.argsort(perm).to(torch.int32)}
    return d


def exact(d, scale, combine, dn=True, ds=True):
    """In 64 bits: outputs, gradients, and the magnitudes that the tolerances are made of."""
    y, r, g = d["y"].double(), d["residual"].double(), d["gamma"].double()
    T, H = r.shape
    rows = y[d["inv"].long()].view(T, -1, H) if combine else y.view(T, 1, H)
    w = d["w"].double() if combine else torch.ones(T, 1, device=y.device, dtype=torch.float64)
    s = r + scale * (w.unsqueeze(2) * rows).sum(1)
    mag = r.abs() + abs(scale) * (w.unsqueeze(2).abs() * rows.abs()).sum(1)
    rstd = (s.square().mean(1, keepdim=True) + EPS).rsqrt()
    u = s * rstd
    dn_ = d["dn"].double() if dn else torch.zeros_like(s)
    a = dn_ * g
    dsum = (d["ds"].double() if ds else 0) + rstd * (a - u * (a * u).mean(1, keepdim=True))
    dw = scale * (dsum.unsqueeze(1) * rows).sum(2)
    dy = scale * w.unsqueeze(2) * dsum.unsqueeze(1)
    return {"s": s, "mag": mag, "n": u * g, "rstd": rstd, "a": a, "dsum": dsum, "dgamma": (dn_ * u).sum(0),
            "dgamma_mag": (dn_ * u).abs().sum(0),
            "dgamma_mag_sum": (dn_.abs() * rstd * mag).sum(0), "rms_mag": (rstd * mag).square().mean(1, keepdim=True).sqrt(), "dw": dw, "dy": dy, "rows": rows, "w": w}


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert bool((off <= bound).all()), f"{what}: off by {(off - bound).max().item():.3e} more than the bound"


def check_forward(n, s, x, g, dtype):
    d = torch.finfo(dtype).eps / 2
    within(s, x["s"], d * x["s"].abs() + SLACK * x["mag"], "sum")
    # the sum's own error, and that of its root mean square, which is no larger
    rms = x["mag"].square().mean(1, keepdim=True).sqrt() * x["rstd"]
    within(n, x["n"], (d + 8 * SLACK) * x["n"].abs() + 2 * SLACK * x["rstd"] * x["mag"] * g.abs() * (1 + rms) +
           SLACK * x["n"].abs() * rms, "normed")


def check_backward(grads, x, T, scale, combine, dtype, inv):
    d = torch.finfo(dtype).eps / 2
    dr, dg, dy, dw = grads
    e_row = (2 * d + 2 * SLACK * x["rms_mag"] + 16 * SLACK) * x["rstd"] * x["a"].norm(dim=1, keepdim=True)  # of a row of ds, 2-norm
    e_row = e_row + SLACK * x["dsum"].norm(dim=1, keepdim=True)
    tiny = torch.finfo(dtype).tiny  # (half of the smallest step, and more, in fp16)

    def rows_within(got, want, bound, what):
        assert torch.isfinite(got).all(), what
        off = (got.double() - want).norm(dim=-1)
        limit = bound + d * want.norm(dim=-1) + tiny * want.shape[-1]
        assert bool((off <= limit).all()), f"{what}: {(off / limit.clamp_min(1e-300)).max().item():.2f} of the bound"

    if dr is not None:
        rows_within(dr, x["dsum"], e_row.squeeze(1), "dresidual")
    if dg is not None:
        within(dg, x["dgamma"], d * x["dgamma"].abs() + (d + 4 * SLACK) * x["dgamma_mag"] +
               SLACK * x["dgamma_mag_sum"], "dgamma")
    if dy is not None:
        got = dy[inv.long()].view(x["dy"].shape) if combine else dy.view(x["dy"].shape)
        rows_within(got, x["dy"], abs(scale) * x["w"].abs() * e_row, "dy")
    if dw is not None:
        y_norm = x["rows"].norm(dim=2)
        within(dw, x["dw"], d * x["dw"].abs() + abs(scale) * (e_row + SLACK * x["dsum"].norm(dim=1, keepdim=True)) * y_norm + tiny,
               "dweights")


SHAPES = [(1, 2048, 8), (3, 1001, 5), (257, 1024, 4), (70, 4096, 8), (9, 8192, 3), (5, 8200, 9), (2, 24576, 2), (4, 3, 1),
          (6, 1, 2), (700, 256, 17), (1200, 768, 8)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,k", SHAPES)
@pytest.mark.parametrize("scale", [1.0, -0.375])
def test_combine_add_rms_norm(cuda, dtype, T, H, k, scale):
    from qwen3_moe_fused.kernels.norm import combine_add_rms_norm

    d = make(cuda, T, H, k, dtype)
    x = exact(d, scale, True)
    with torch.no_grad():
        n, s = combine_add_rms_norm(d["y"], d["sort"], d["inv"], d["w"], d["residual"], d["gamma"], EPS, scale)
    check_forward(n, s, x, d["gamma"].double(), dtype)
    leaves = [d[m].requires_grad_() for m in ("residual", "gamma", "y", "w")]
    n2, s2 = combine_add_rms_norm(d["y"], d["sort"], d["inv"], d["w"], d["residual"], d["gamma"], EPS, scale)
    assert torch.equal(n2, n) and torch.equal(s2, s)
    grads = torch.autograd.grad((n2, s2), leaves, (d["dn"], d["ds"]), retain_graph=True)
    check_backward(grads, x, T, scale, True, dtype, d["inv"])
    again = torch.autograd.grad((n2, s2), leaves, (d["dn"], d["ds"]))
    assert all(torch.equal(p, q) for p, q in zip(grads, again))  # same bits in every run


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 2048), (3, 1001), (1025, 1024), (9, 8192), (5, 8200), (2, 24576), (4, 3)])
def test_add_rms_norm(cuda, dtype, T, H):
    from qwen3_moe_fused.kernels.norm import add_rms_norm

    d = make(cuda, T, H, 1, dtype, seed=1)
    x = exact(d, 0.5, False)
    leaves = [d[m].requires_grad_() for m in ("residual", "gamma", "y")]
    n, s = add_rms_norm(d["y"], d["residual"], d["gamma"], EPS, 0.5)
    check_forward(n.detach(), s.detach(), x, d["gamma"].detach().double(), dtype)
    grads = torch.autograd.grad((n, s), leaves, (d["dn"], d["ds"]))
    check_backward((*grads, None), x, T, 0.5, False, dtype, None)


@pytest.mark.parametrize("which", ["normed", "sum"])
@pytest.mark.parametrize("H", [2048, 1001])
@pytest.mark.parametrize("want", [("residual",), ("gamma",), ("y",), ("w",), ("y", "gamma")])
def test_one_output_or_one_gradient(cuda, which, H, want):
    """Only one output is used, and only some inputs want a gradient."""
    from qwen3_moe_fused.kernels.norm import combine_add_rms_norm

    T, k, dtype = 37, 3, torch.bfloat16
    d = make(cuda, T, H, k, dtype, seed=2)
    x = exact(d, 1.0, True, dn=which == "normed", ds=which == "sum")
    for m in want:
        d[m].requires_grad_()
    n, s = combine_add_rms_norm(d["y"], d["sort"], d["inv"], d["w"], d["residual"], d["gamma"], EPS)
    out, grad = (n, d["dn"]) if which == "normed" else (s, d["ds"])
    got = dict(zip(want, torch.autograd.grad(out, [d[m] for m in want], grad, allow_unused=True)))
    check_backward(tuple(got.get(m) for m in ("residual", "gamma", "y", "w")), x, T, 1.0, True, dtype, d["inv"])


def test_without_residual_and_without_tokens(cuda):
    from qwen3_moe_fused.kernels.norm import add_rms_norm, combine_add_rms_norm

    gen = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(2, 5, 2048, device=cuda, generator=gen, dtype=torch.float32)
    g = torch.randn(2048, device=cuda, generator=gen)
    n, s = add_rms_norm(x, None, g, EPS)
    assert torch.equal(s, x) and n.shape == x.shape
    want = x.double() * (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt() * g.double()
    within(n, want, 32 * 2.0 ** -24 * want.abs(), "norm alone")
    # no tokens: empty outputs, a gradient of zeros for the norm's weight
    e = torch.empty(0, 64, device=cuda, requires_grad=True)
    idx = torch.empty(0, device=cuda, dtype=torch.int32)
    gamma = torch.ones(64, device=cuda, requires_grad=True)
    n, s = combine_add_rms_norm(e, idx, idx, torch.empty(0, 8, device=cuda), torch.empty(0, 64, device=cuda), gamma)
    assert n.shape == s.shape == (0, 64)
    (dg,) = torch.autograd.grad(n.sum() + s.sum(), gamma)
    assert torch.equal(dg, torch.zeros_like(dg))
    # a row of zeros has a norm of zeros
    n, s = add_rms_norm(torch.zeros(1, 64, device=cuda), None, gamma.detach(), EPS)
    assert torch.equal(n, torch.zeros_like(n))


def test_nan_and_infinity_stay_in_their_row(cuda):
    from qwen3_moe_fused.kernels.norm import combine_add_rms_norm

    d = make(cuda, 12, 1024, 4, torch.bfloat16, seed=4)
    with torch.no_grad():
        n, s = combine_add_rms_norm(d["y"], d["sort"], d["inv"], d["w"], d["residual"], d["gamma"], EPS)
        y = d["y"].clone()
        y[d["inv"][5 * 4 + 1].item(), 17] = float("nan")
        y[d["inv"][7 * 4 + 3].item(), 0] = float("inf")
        n2, s2 = combine_add_rms_norm(y, d["sort"], d["inv"], d["w"], d["residual"], d["gamma"], EPS)
    keep = [t for t in range(12) if t not in (5, 7)]
    assert torch.equal(n2[keep], n[keep]) and torch.equal(s2[keep], s[keep])
    assert n2[5].isnan().all() and s2[5, 17].isnan() and s2[7, 0].isinf()


def test_against_differences(cuda):
    """Directional derivatives of the fp32 kernel itself, by central differences at two widths.  Rounding: each of the T H
    outputs is off by at most 2^-20 of its size (below 8 here) times its weight; truncation by what the two widths differ by."""
    from qwen3_moe_fused.kernels.norm import combine_add_rms_norm

    T, H, k = 3, 96, 2
    d = make(cuda, T, H, k, torch.float32, seed=5)
    names = ("residual", "gamma", "y", "w")

    def value(p):
        with torch.no_grad():
            n, s = combine_add_rms_norm(p["y"], d["sort"], d["inv"], p["w"], p["residual"], p["gamma"], EPS, 0.75)
        return (n.double() * d["dn"].double()).sum().item() + (s.double() * d["ds"].double()).sum().item()

    for name in names:
        p = {m: d[m].clone() for m in names}
        p[name].requires_grad_()
        n, s = combine_add_rms_norm(p["y"], d["sort"], d["inv"], p["w"], p["residual"], p["gamma"], EPS, 0.75)
        (grad,) = torch.autograd.grad((n, s), p[name], (d["dn"], d["ds"]))
        direction = torch.randn(p[name].shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(6))
        slopes = []
        for h in (2.0 ** -5, 2.0 ** -6):
            hi, lo = ({**d, name: (d[name].double() + q * h * direction.double()).float()} for q in (1, -1))
            slopes.append((value(hi) - value(lo)) / (2 * h))
        want = (grad.double() * direction.double()).sum().item()
        rounding = 2 * 8 * 2.0 ** -20 * (d["dn"].abs().sum() + d["ds"].abs().sum()).item() / (2 * 2.0 ** -6)
        assert abs(slopes[1] - want) <= 2 * abs(slopes[0] - slopes[1]) + rounding, (name, slopes, want)


def test_other_stream_graph_and_unaligned(cuda):
    from qwen3_moe_fused.kernels.norm import add_rms_norm

    gen = torch.Generator(device=cuda).manual_seed(7)
    flat = torch.randn(40 * 2048 + 1, device=cuda, generator=gen).to(torch.bfloat16)
    x, r = flat[1:].view(40, 2048), flat[:-1].view(40, 2048)  # x is not 16-byte aligned: the other form, the same formula
    g = torch.randn(2048, device=cuda, generator=gen).to(torch.bfloat16)
    with torch.no_grad():
        n, s = add_rms_norm(x, r, g, EPS)
        n_al, s_al = add_rms_norm(x.clone(), r, g, EPS)
        assert torch.equal(s, s_al)
        # (the mean of squares is summed in another order: a last bit of n may differ)
        within(n, n_al.double(), 2.0 ** -7 * n_al.double().abs(), "unaligned")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            n2, s2 = add_rms_norm(x, r, g, EPS)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(n2, n) and torch.equal(s2, s)
        xs = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n3, s3 = add_rms_norm(xs, r, g, EPS)
        xs.copy_(r)
        graph.replay()
        n4, s4 = add_rms_norm(r.clone(), r, g, EPS)
        assert torch.equal(n3, n4) and torch.equal(s3, s4)


def test_refusals(cuda):
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.kernels.norm import add_rms_norm, combine_add_rms_norm
    import torch.autograd.forward_ad as fw

    x, g = torch.ones(4, 64, device=cuda), torch.ones(64, device=cuda)
    for bad in (g.half(), g[:63], g.cpu()):
        with pytest.raises(AssertionError):
            add_rms_norm(x, None, bad)
    for bad in (x.half(), x[:3], x.cpu()):
        with pytest.raises(AssertionError):
            add_rms_norm(x, bad, g)
    with pytest.raises(_lib.MoeB200Error):
        add_rms_norm(torch.ones(1, 24577, device=cuda), None, torch.ones(24577, device=cuda))
    with pytest.raises(_lib.MoeB200Error):
        add_rms_norm(x.double(), None, g.double())
    idx = torch.arange(4, device=cuda, dtype=torch.int32)
    w = torch.ones(2, 2, device=cuda)
    for args in ((x, idx.long(), idx.long(), w), (x, idx[:3], idx[:3], w), (x[:3], idx, idx, w), (x, idx, idx, w.half())):
        with pytest.raises(AssertionError):
            combine_add_rms_norm(*args, None, g)
    # no second derivative, and no tangent dropped
    xr = x.clone().requires_grad_()
    n, _ = add_rms_norm(xr, None, g)
    (dx,) = torch.autograd.grad(n.sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    with torch.no_grad(), fw.dual_level(), pytest.raises(NotImplementedError):
        add_rms_norm(fw.make_dual(x, torch.ones_like(x)), None, g)
