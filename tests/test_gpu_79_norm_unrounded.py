"""The norms' backward pass starts from the sum before its rounding: gradients against the formulas in 64 bits, with one rounding each,
and finite where the sum is past fp16's range and the normed row is not.

Tolerances, d = eps / 2 of the type.  The sum s is off by fp32 sums of at most 64 terms, 2^-18 of the sum of magnitudes `mag`, so
u = s r by Du <= 2^-18 r mag; a row of ds = .. + r (a - u mean(a u)), with rms(u) <= 1, by 2 r ||a|| rms(Du) and 16 * 2^-18 r ||a|| for
its own sums and the reciprocal root in the 2-norm; what is computed from ds by that times the other factor; dgamma by the sum of
|dn| Du and 2^-16 of its own magnitudes.  Then one rounding, d of the result, and half of the smallest step where that is denormal."""
import pytest
import torch

from . import test_gpu_72_norm as norms

pytestmark = pytest.mark.gpu

SLACK, EPS = norms.SLACK, norms.EPS


def check(grads, x, scale, dtype, inv=None):
    d = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny
    dr, dg, dy, dw = grads
    e_row = (2 * SLACK * x["rms_mag"] + 16 * SLACK) * x["rstd"] * x["a"].norm(dim=1, keepdim=True)
    e_row = e_row + SLACK * x["dsum"].norm(dim=1, keepdim=True)

    def rows(got, want, bound, what):
        off = (got.double() - want).norm(dim=-1)
        limit = bound + d * want.norm(dim=-1) + tiny * want.shape[-1]
        assert torch.isfinite(got).all() and bool((off <= limit).all()), f"{what}: {(off / limit).max().item():.2f} of the bound"

    rows(dr, x["dsum"], e_row.squeeze(1), "dresidual")
    norms.within(dg, x["dgamma"], d * x["dgamma"].abs() + 4 * SLACK * x["dgamma_mag"] + SLACK * x["dgamma_mag_sum"], "dgamma")
    got = dy if inv is None else dy[inv.long()]
    rows(got.view(x["dy"].shape), x["dy"], abs(scale) * x["w"].abs() * e_row, "dy")
    if dw is not None:
        bound = abs(scale) * (e_row + SLACK * x["dsum"].norm(dim=1, keepdim=True)) * x["rows"].norm(dim=2)
        norms.within(dw, x["dw"], d * x["dw"].abs() + bound + tiny, "dweights")


# one vector of a row to a thread, two, four; rows in shared memory, three of them and two
SHAPES = [(301, 2048, 8), (33, 1024, 4), (70, 4096, 8), (9, 8192, 3), (40, 1001, 5), (5, 8200, 9), (2, 19200, 2), (2, 19201, 3), (2, 24576, 2),
          (3, 24575, 1), (6, 1, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,k", SHAPES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_gradients(cuda, dtype, T, H, k, with_residual):
    from qwen3_moe_fused.kernels.norm import add_rms_norm, combine_add_rms_norm

    scale = 0.625
    d = norms.make(cuda, T, H, k, dtype, seed=11)
    if not with_residual:
        d["residual"].zero_()
    r = d["residual"] if with_residual else None
    x = norms.exact(d, scale, True)
    leaves = [d[m].requires_grad_() for m in (("residual",) if with_residual else ()) + ("gamma", "y", "w")]
    out = combine_add_rms_norm(d["y"], d["sort"], d["inv"], d["w"], r, d["gamma"], EPS, scale)
    grads = torch.autograd.grad(out, leaves, (d["dn"], d["ds"]))
    if not with_residual:
        grads = (x["dsum"].to(dtype), *grads)
    check(grads, x, scale, dtype, d["inv"])
    plain = {m: d[m].detach() for m in ("residual", "gamma", "dn", "ds")} | {"y": d["y"].detach()[:T]}
    x = norms.exact(plain, scale, False)
    leaves = [plain[m].requires_grad_() for m in (("residual",) if with_residual else ()) + ("gamma", "y")]
    out = add_rms_norm(plain["y"], plain["residual"] if with_residual else None, plain["gamma"], EPS, scale)
    grads = torch.autograd.grad(out, leaves, (d["dn"], d["ds"]))
    if not with_residual:
        grads = (x["dsum"].to(dtype), *grads)
    check((*grads, None), x, scale, dtype)


@pytest.mark.parametrize("H,k", [(2048, 8), (1024, 2), (4096, 8), (1001, 3)])
def test_sums_past_the_range_of_the_type(cuda, H, k):
    """fp16 rows whose sum is past 65504 here and there: that output is infinite, the normed row and every gradient of it are not."""
    from qwen3_moe_fused.kernels.norm import add_rms_norm, combine_add_rms_norm

    T, dtype = 12, torch.float16
    d = norms.make(cuda, T, H, k, dtype, seed=12)
    d["y"] = (d["y"].float() * 2.0 ** 13).to(dtype)
    d["w"] = torch.full((T, k), 4.0, device=cuda, dtype=dtype)
    x = norms.exact(d, 1.0, True, ds=False)
    leaves = [d[m].requires_grad_() for m in ("residual", "gamma", "y", "w")]
    n, s = combine_add_rms_norm(d["y"], d["sort"], d["inv"], d["w"], d["residual"], d["gamma"], EPS)
    assert s.isinf().any() and torch.isfinite(n).all()
    check(torch.autograd.grad(n, leaves, d["dn"]), x, 1.0, dtype, d["inv"])
    plain = {m: d[m].detach() for m in ("residual", "gamma", "dn", "ds")} | {"y": d["y"].detach()[:T]}
    x = norms.exact(plain, 8.0, False, ds=False)
    leaves = [plain[m].requires_grad_() for m in ("residual", "gamma", "y")]
    n, s = add_rms_norm(plain["y"], plain["residual"], plain["gamma"], EPS, 8.0)
    assert s.isinf().any() and torch.isfinite(n).all()
    check((*torch.autograd.grad(n, leaves, d["dn"]), None), x, 8.0, dtype)


@pytest.mark.parametrize("H,k", [(2048, 8), (1024, 4), (1001, 5), (24576, 2)])
def test_c_form_on_the_stored_sum(cuda, H, k):
    """`moe_combine_add_rms_norm_bwd`, for callers that kept the sum alone: within the stored sum's rounding."""
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.kernels.norm import _forward

    T, scale, dtype = 35, 0.5, torch.bfloat16
    d = norms.make(cuda, T, H, k, dtype, seed=13)
    lib, stream = _lib.load(), _lib.stream_ptr(cuda)
    for combine in (True, False):
        y = d["y"] if combine else d["y"][:T]
        inv, w = (d["inv"], d["w"]) if combine else (None, None)
        x = norms.exact({**d, "y": y}, scale, combine)
        _, total, rstd = _forward(y, inv, w, d["residual"], d["gamma"], EPS, scale, True)
        dr, dy, dw, dg = torch.empty_like(total), torch.empty_like(y), torch.empty_like(d["w"]) if combine else None, torch.empty_like(d["gamma"])
        ws = torch.empty(lib.moe_combine_add_rms_norm_bwd_ws_bytes(T, H), device=cuda, dtype=torch.uint8)
        st = lib.moe_combine_add_rms_norm_bwd(*map(_lib.ptr, (d["dn"], d["ds"], total, rstd, d["gamma"], y if combine else None, inv, w)),
                                              scale, *map(_lib.ptr, (dr, dy, dw, dg)), T, k if combine else 1, H, _lib.BF16,
                                              _lib.ptr(ws), ws.numel(), stream)
        _lib.check(st, "moe_combine_add_rms_norm_bwd")
        norms.check_backward((dr, dg, dy, dw), x, T, scale, combine, dtype, d["inv"])


@pytest.mark.parametrize("H", [2048, 1001])
def test_c_forward_without_one_of_its_outputs(cuda, H):
    """sum, normed and rstd may each be NULL: the others keep their bits."""
    from qwen3_moe_fused import _lib
    from qwen3_moe_fused.kernels.norm import _forward

    T, k = 7, 8
    d = norms.make(cuda, T, H, k, torch.bfloat16, seed=14)
    lib, stream = _lib.load(), _lib.stream_ptr(cuda)
    for inv, w, kk, y in ((d["inv"], d["w"], k, d["y"]), (None, None, 1, d["y"][:T])):
        n, s, rstd = _forward(y, inv, w, d["residual"], d["gamma"], EPS, 0.5, True)
        for want in ((True, False, False), (False, True, False), (False, True, True), (True, True, False), (False, False, False)):
            outs = [torch.full_like(t, 7) for t in (s, n, rstd)]
            st = lib.moe_combine_add_rms_norm(*map(_lib.ptr, (y, inv, w, d["residual"], d["gamma"])), 0.5, EPS,
                                              *(_lib.ptr(t) if on else None for t, on in zip(outs, want)), T, kk, H, _lib.BF16, stream)
            _lib.check(st, "moe_combine_add_rms_norm")
            for got, full, on in zip(outs, (s, n, rstd), want):
                assert torch.equal(got, full) if on else bool((got == 7).all())
