"""Operators of a sparse layer whose experts are held in 8 bits: what is measured when their kernels change.

  linear   moe_fused_linear_fp8: one expert projection on e4m3 weights with a scale for each 128 x 128 block; the tokens are
           quantised in the call, in blocks of 128 of a row.  "train": the gradient of the tokens too (the weights are frozen)
  mlp      moe_mlp_fp8: gate, up, SiLU-mul and down on such weights; "train": the gradient of the tokens too
  combine_norm  combine_add_rms_norm: weighted sum of a token's expert rows, scaled and added to the residual stream, and the
           RMS norm in front of the next block; "train": the gradients of rows, routing weights, residual and norm weight too
  add_norm add_rms_norm: the same for a block whose output is one row for each token

Sizes: hidden 2048, expert width 768 (gate and up together 1536), 128 experts, 8 per token are those of bench.py and of the
tests; (1024, 512, 32, 4) is a generic smaller layer.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
#             hidden, expert width, experts, experts per token
GEOMETRY = {"large": (2048, 768, 128, 8), "small": (1024, 512, 32, 4)}
BLOCK = 128
E4M3 = torch.float8_e4m3fn
EPS = 1e-6


def listed():
    return [
        # serving: the down projection for one token; gate and up (stacked) for a batch of 48 sequences, one new token each
        {"name": "linear_decode_1", "kind": "linear", "rows": 8, "in": 768, "out": 2048, "experts": 128, "routing": "softmax",
         "train": False, "dtype": "bf16"},
        {"name": "linear_decode_48", "kind": "linear", "rows": 384, "in": 2048, "out": 1536, "experts": 128,
         "routing": "softmax", "train": False, "dtype": "bf16"},
        # fine-tuning around frozen 8-bit weights: gate and up (stacked) on 8192 tokens; down with skewed routing and experts
        # that get nothing; a small odd batch in fp16
        {"name": "linear_gate_up_65536", "kind": "linear", "rows": 65536, "in": 2048, "out": 1536, "experts": 128,
         "routing": "softmax", "train": True, "dtype": "bf16"},
        {"name": "linear_down_zipf_65536", "kind": "linear", "rows": 65536, "in": 768, "out": 2048, "experts": 128,
         "routing": "zipf", "train": True, "dtype": "bf16"},
        {"name": "linear_f16_5003", "kind": "linear", "rows": 5003, "in": 2048, "out": 768, "experts": 128,
         "routing": "random", "train": True, "dtype": "f16"},
        # the whole expert MLP: a decoding step of 48 sequences, a prefill of 4 prompts of 2048 tokens, a training batch
        {"name": "mlp_decode_48", "kind": "mlp", "tokens": 48, "geometry": "large", "routing": "softmax", "train": False,
         "dtype": "bf16"},
        {"name": "mlp_prefill_8192", "kind": "mlp", "tokens": 8192, "geometry": "large", "routing": "softmax", "train": False,
         "dtype": "bf16"},
        {"name": "mlp_train_4095", "kind": "mlp", "tokens": 4095, "geometry": "large", "routing": "softmax", "train": True,
         "dtype": "bf16"},
        # after the block: one new token; a batch of 8 prompts of 2048 tokens; a training batch of odd size
        {"name": "combine_norm_1", "kind": "combine_norm", "tokens": 1, "hidden": 2048, "k": 8, "scale": 1.0, "train": False,
         "dtype": "bf16"},
        {"name": "combine_norm_16384", "kind": "combine_norm", "tokens": 16384, "hidden": 2048, "k": 8, "scale": 1.0,
         "train": False, "dtype": "bf16"},
        {"name": "combine_norm_train_8191", "kind": "combine_norm", "tokens": 8191, "hidden": 2048, "k": 8, "scale": 0.5,
         "train": True, "dtype": "bf16"},
        # before the block: residual and norm behind the attention of a training batch
        {"name": "add_norm_train_16001", "kind": "add_norm", "tokens": 16001, "hidden": 2048, "scale": 1.0, "train": True,
         "dtype": "f16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "mlp", "mlp", "combine_norm", "add_norm"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    train = rng.random() < 0.5
    if kind == "linear":
        # (1008 -> 720: neither side a whole number of blocks)
        k_in, n_out, experts = rng.choice([(2048, 1536, 128), (2048, 768, 128), (768, 2048, 128), (1024, 512, 32), (1008, 720, 32)])
        return {"kind": kind, "rows": _log_int(rng, 1, 65536), "in": k_in, "out": n_out, "experts": experts,
                "routing": rng.choice(["softmax", "random", "zipf"]), "train": train, "dtype": dtype}
    if kind == "mlp":
        return {"kind": kind, "tokens": _log_int(rng, 1, 8192 if not train else 4096), "geometry": rng.choice(["large", "large", "small"]),
                "routing": rng.choice(["softmax", "zipf"]), "train": train, "dtype": dtype}
    case = {"kind": kind, "tokens": _log_int(rng, 1, 16384 if not train else 8192), "hidden": rng.choice([2048, 2048, 1024, 1536, 1001]),
            "scale": rng.choice([1.0, 0.5, 0.22]), "train": train, "dtype": dtype}
    if kind == "combine_norm":
        case["k"] = rng.choice([8, 8, 4, 2, 5])
    return case


# ------------------------------------------------------------------------------------------ inputs
def _sizes(rows, experts, routing, k, gen, dev):
    """Rows of each expert: top-k of N(0,1) logits, ids drawn evenly, or Zipf(1.2) over experts in random order with three of
    them left without rows."""
    if routing == "softmax":
        logits = torch.randn(-(-rows // k), experts, generator=gen, device=dev)
        ids = logits.topk(k, dim=1).indices.reshape(-1)[:rows]
    elif routing == "random":
        ids = torch.randint(experts, (rows,), generator=gen, device=dev)
    else:
        pmf = (torch.arange(experts, device=dev, dtype=torch.float64) + 1) ** -1.2
        pmf[[5, experts // 2, experts - 1]] = 0
        cdf = (pmf / pmf.sum()).cumsum(0)
        ids = torch.searchsorted(cdf, torch.rand(rows, generator=gen, device=dev, dtype=torch.float64)).clamp_max(experts - 2)
        ids = torch.randperm(experts, generator=gen, device=dev)[ids]
    return torch.bincount(ids, minlength=experts).to(torch.int32)


def _fp8_weight(e, n, k, gen, dev):
    """N(0, 0.02) weights as a checkpoint holds them: e4m3 values and one fp32 scale (largest magnitude / 448) for each block."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(e, nb * BLOCK, kb * BLOCK, device=dev, dtype=torch.bfloat16)
    w[:, :n, :k] = torch.randn(e, n, k, generator=gen, device=dev, dtype=torch.bfloat16).mul_(0.02)
    blocks = w.view(e, nb, BLOCK, kb, BLOCK)
    scale = blocks.abs().amax(dim=(2, 4)).float() / 448
    data = (blocks / scale.view(e, nb, 1, kb, 1)).to(E4M3).view(e, nb * BLOCK, kb * BLOCK)
    return data[:, :n, :k].contiguous(), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, kind = DTYPES[case["dtype"]], case["kind"]

    def normal(*shape, scale=1.0):
        t = torch.randn(*shape, generator=gen, device=dev, dtype=dt)
        return t if scale == 1.0 else t.mul_(scale)

    state = {"kind": kind, "train": case["train"]}
    if kind in ("linear", "mlp"):
        if kind == "linear":
            rows, k_in, n_out, experts = case["rows"], case["in"], case["out"], case["experts"]
            state["weights"] = _fp8_weight(experts, n_out, k_in, gen, dev)
            per_token = 8
        else:
            k_in, width, experts, per_token = GEOMETRY[case["geometry"]]
            rows, n_out = case["tokens"] * per_token, k_in
            state["weights"] = (*_fp8_weight(experts, width, k_in, gen, dev), *_fp8_weight(experts, width, k_in, gen, dev),
                                *_fp8_weight(experts, k_in, width, gen, dev))
        state["m_sizes"] = _sizes(rows, experts, case["routing"], per_token, gen, dev)
        state["sizes"] = state["m_sizes"].tolist()  # what the plain form cuts the rows by; the calls take m_sizes
        state["x"] = normal(rows, k_in).requires_grad_(case["train"])
        if case["train"]:
            state["dy"] = normal(rows, n_out)
        return state
    tokens, hidden = case["tokens"], case["hidden"]
    state["scale"] = case["scale"]
    state["residual"] = normal(tokens, hidden, scale=2.0).requires_grad_(case["train"])
    state["gamma"] = (1 + normal(hidden, scale=0.1)).requires_grad_(case["train"])
    if kind == "combine_norm":
        k = case["k"]
        logits, experts = torch.randn(tokens, 128, generator=gen, device=dev).topk(k, dim=1)
        state["weights"] = torch.softmax(logits, dim=1).to(dt).requires_grad_(case["train"])
        state["sort_idx"] = torch.argsort(experts.reshape(-1), stable=True).to(torch.int32)
        state["inv"] = torch.argsort(state["sort_idx"]).to(torch.int32)
        state["y"] = normal(tokens * k, hidden).requires_grad_(case["train"])
    else:
        state["y"] = normal(tokens, hidden).requires_grad_(case["train"])
    if case["train"]:
        state["dn"], state["ds"] = normal(tokens, hidden), normal(tokens, hidden)
    return state


# ------------------------------------------------------------------------------------------ plain forms
def _quantised_rows(x):
    """The values that e4m3 codes with one power of two for each 128 of a row stand for, in 32 bits."""
    rows, n = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -n % BLOCK)).view(rows, -1, BLOCK)
    mantissa, exponent = torch.frexp(blocks.abs().amax(dim=2, keepdim=True))  # mantissa in [0.5, 1)
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp_min(-100)
    scale = torch.ldexp(torch.ones_like(mantissa), exponent)
    return ((blocks / scale).to(E4M3).float() * scale).view(rows, -1)[:, :n]


def _decoded(data, scale):
    n, k = data.shape[1:]
    return data.float() * scale.repeat_interleave(BLOCK, 1)[:, :n].repeat_interleave(BLOCK, 2)[:, :, :k]


def _grouped(x, w, sizes, transposed=False):
    """Rows of expert e times its weight (or the weight's transpose)."""
    parts = [r @ (w[e] if transposed else w[e].T) for e, r in enumerate(x.split(sizes))]
    return torch.cat(parts)


def _plain_mlp(state):
    wg, wu, wd = (_decoded(*state["weights"][2 * i:2 * i + 2]) for i in range(3))
    x, sizes = state["x"].detach(), state["sizes"]
    xq = _quantised_rows(x)
    e, g = _grouped(xq, wg, sizes), _grouped(xq, wu, sizes)
    y = _grouped(_quantised_rows(e * torch.sigmoid(e) * g), wd, sizes).to(x.dtype)
    if not state["train"]:
        return (y,)
    e, g = e.to(x.dtype).float(), g.to(x.dtype).float()  # kept for the backward pass in the tokens' type
    dh = _grouped(_quantised_rows(state["dy"]), wd, sizes, True)
    sig = torch.sigmoid(e)
    de, dg = dh * g * sig * (1 + e * (1 - sig)), dh * e * sig
    dx = _grouped(_quantised_rows(de), wg, sizes, True) + _grouped(_quantised_rows(dg), wu, sizes, True)
    return y, dx.to(x.dtype)


def _plain_norm(state):
    y, residual, gamma, scale = (state[n] for n in ("y", "residual", "gamma", "scale"))
    dt = y.dtype
    y, r, gm = y.detach().float(), residual.detach().float(), gamma.detach().float()
    combine = state["kind"] == "combine_norm"
    if combine:
        w = state["weights"].detach().float()
        tokens, k = w.shape
        y = y[state["inv"].long()].view(tokens, k, -1)
        block = (w.unsqueeze(2) * y).sum(1)
    else:
        block = y
    s = r + scale * block
    rstd = torch.rsqrt(s.square().mean(1, keepdim=True) + EPS)
    n = s * rstd * gm
    if not state["train"]:
        return n.to(dt), s.to(dt)
    dn, ds = state["dn"].float(), state["ds"].float()
    hat, a = s * rstd, dn * gm
    ds = ds + rstd * (a - hat * (a * hat).mean(1, keepdim=True))
    dgamma = (dn * hat).sum(0)
    grads = [ds, dgamma]
    if combine:
        dy = torch.empty_like(y).view(tokens * k, -1)
        dy[state["inv"].long()] = (scale * w.unsqueeze(2) * ds.unsqueeze(1)).view(tokens * k, -1)
        grads += [dy, scale * (ds.unsqueeze(1) * y).sum(2)]
    else:
        grads += [scale * ds]
    return tuple(t.to(dt) for t in (n, s, *grads))


# ------------------------------------------------------------------------------------------ one pass
@functools.lru_cache(None)
def _calls():
    pkg = os.path.join(os.getcwd(), "transformers-qwen3-moe-fused_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from qwen3_moe_fused.kernels.fused_mlp_fp8 import moe_mlp_fp8
    from qwen3_moe_fused.kernels.norm import add_rms_norm, combine_add_rms_norm
    from qwen3_moe_fused.quantize.linear8bit import moe_fused_linear_fp8

    return moe_fused_linear_fp8, moe_mlp_fp8, add_rms_norm, combine_add_rms_norm


def run(state):
    kind, train = state["kind"], state["train"]
    if not own:
        with torch.no_grad():
            if kind == "mlp":
                return _plain_mlp(state)
            if kind != "linear":
                return _plain_norm(state)
            w, x = _decoded(*state["weights"]), state["x"]
            y = _grouped(_quantised_rows(x), w, state["sizes"]).to(x.dtype)
            if not train:
                return (y,)
            return y, _grouped(_quantised_rows(state["dy"]), w, state["sizes"], True).to(x.dtype)
    moe_fused_linear_fp8, moe_mlp_fp8, add_rms_norm, combine_add_rms_norm = _calls()
    with torch.set_grad_enabled(train):
        if kind in ("linear", "mlp"):
            if kind == "linear":
                y = moe_fused_linear_fp8(state["x"], *state["weights"], state["m_sizes"])
            else:
                y = moe_mlp_fp8(state["x"], *state["weights"], state["m_sizes"])
            if not train:
                return (y,)
            return y.detach(), *torch.autograd.grad(y, state["x"], state["dy"])
        if kind == "combine_norm":
            out = combine_add_rms_norm(state["y"], state["sort_idx"], state["inv"], state["weights"], state["residual"],
                                       state["gamma"], EPS, state["scale"])
            leaves = [state["residual"], state["gamma"], state["y"], state["weights"]]
        else:
            out = add_rms_norm(state["y"], state["residual"], state["gamma"], EPS, state["scale"])
            leaves = [state["residual"], state["gamma"], state["y"]]
        if not train:
            return out
        return *(t.detach() for t in out), *torch.autograd.grad(out, leaves, (state["dn"], state["ds"]))


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def _used(experts, rows):
    return experts * (1.0 - (1.0 - 1.0 / experts) ** rows)  # experts that get a row


def work(case):
    kind, train = case["kind"], case["train"]
    both = 2 if train else 1
    block_bytes = 1 + 4 / BLOCK ** 2  # of a weight, with its share of the scale
    if kind == "linear":
        m, k, n, e = case["rows"], case["in"], case["out"], case["experts"]
        return {"bytes": _used(e, m) * k * n * block_bytes + 2.0 * m * (k + n) * both, "flops": 2.0 * m * k * n * both}
    if kind == "mlp":
        h, i, e, k = GEOMETRY[case["geometry"]]
        m = case["tokens"] * k
        return {"bytes": _used(e, m) * 3 * h * i * block_bytes + 2.0 * m * 2 * h * both, "flops": 6.0 * m * h * i * both}
    t, h, k = case["tokens"], case["hidden"], case.get("k", 1)
    rows = t * h * (k + 3) + h  # expert rows and residual read, norm and sum written
    if not train:
        return {"bytes": 2.0 * rows, "flops": 2.0 * t * h * (k + 3)}
    # two gradients read; gradients of the residual and of the expert rows written
    return {"bytes": 2.0 * (rows + t * h * (3 + k) + h), "flops": 2.0 * t * h * (3 * k + 10)}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(x):
    """Nearest e4m3 value (ties to the even code) of x over the block's power of two: three bits behind the leading one, steps
    of 2^-9 below 2^-6."""
    x = x.double()
    out = torch.empty_like(x)
    for a in range(0, x.shape[1], BLOCK):
        b = x[:, a:a + BLOCK]
        top = b.abs().max(dim=1, keepdim=True).values
        scale = torch.full_like(top, 2.0 ** -100)
        nz = top > 0
        scale[nz] = torch.exp2(torch.ceil(torch.log2(top[nz] / 448)).clamp_min(-100))
        scale = torch.where(top > 448 * scale, scale * 2, scale)  # (the logarithm may be off by its last bit)
        scale = torch.where(top <= 224 * scale, scale / 2, scale).clamp_min(2.0 ** -100)
        v = b / scale
        step = torch.exp2(torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent.double() - 4)
        out[:, a:a + BLOCK] = torch.round(v / step) * step * scale
    return out


def _exact_product(x, weight, sizes, back=False):
    data, scale = weight
    out = torch.empty(x.shape[0], data.shape[2 if back else 1], dtype=torch.float64, device=x.device)
    row = 0
    for e, m in enumerate(sizes):
        if m == 0:
            continue
        w = data[e].double()
        for i in range(scale.shape[1]):
            for j in range(scale.shape[2]):
                w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale[e, i, j].double()
        torch.mm(x[row:row + m], w if back else w.t(), out=out[row:row + m])
        row += m
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind, train = st["kind"], st["train"]
    with torch.no_grad():
        if kind in ("linear", "mlp"):
            sizes = [int(v) for v in st["m_sizes"].cpu()]
            xq = _exact_rows(st["x"])
            if kind == "linear":
                y = _exact_product(xq, st["weights"], sizes)
                return (y, _exact_product(_exact_rows(st["dy"]), st["weights"], sizes, True)) if train else (y,)
            gate, up, down = st["weights"][0:2], st["weights"][2:4], st["weights"][4:6]
            e, g = _exact_product(xq, gate, sizes), _exact_product(xq, up, sizes)
            y = _exact_product(_exact_rows(e / (1 + torch.exp(-e)) * g), down, sizes)
            if not train:
                return (y,)
            e, g = e.to(st["x"].dtype).double(), g.to(st["x"].dtype).double()  # as the operator keeps them
            dh = _exact_product(_exact_rows(st["dy"]), down, sizes, True)
            z = torch.exp(-e)
            de = dh * g * (1 / (1 + z) + e * z / (1 + z) ** 2)
            dg = dh * e / (1 + z)
            return y, _exact_product(_exact_rows(de), gate, sizes, True) + _exact_product(_exact_rows(dg), up, sizes, True)
        scale, gm = st["scale"], st["gamma"].double()
        s = st["residual"].double()
        y = st["y"].double()
        if kind == "combine_norm":
            inv = st["inv"].long()
            w = st["weights"].double()
            tokens, k = w.shape
            for j in range(k):
                s = s + scale * w[:, j:j + 1] * y[inv[j::k]]
        else:
            s = s + scale * y
        h = s.shape[1]
        root = torch.sqrt((s * s).sum(1) / h + EPS)[:, None]
        n = gm * s / root
        if not train:
            return n, s
        dn = st["dn"].double()
        # d/ds of gamma s / root: gamma dn / root - s <gamma dn, s> / (h root^3)
        ds = st["ds"].double() + gm * dn / root - s * (gm * dn * s).sum(1, keepdim=True) / (h * root ** 3)
        dgamma = (dn * s / root).sum(0)
        if kind == "add_norm":
            return n, s, ds, dgamma, scale * ds
        dy, dw = torch.empty_like(y), torch.empty_like(w)
        for j in range(k):
            dy[inv[j::k]] = scale * w[:, j:j + 1] * ds
            dw[:, j] = scale * (ds * y[inv[j::k]]).sum(1)
        return n, s, ds, dgamma, dy, dw
