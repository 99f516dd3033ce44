"""Cases, inputs, plain forms and exact values of the 4-bit expert operators and of the norm around an expert block.

Operators (``wisp_b200.mx4``, ``wisp_b200.norm``):

* ``quant``   ``mx4_quantize`` then ``mx4_dequantize``: blocks of 32 values along the last axis share a power-of-two
  scale 2^(floor(log2 amax) - 2) (E8M0 byte), the values are E2M1 codes, two a byte, rounded to nearest even;
* ``matmul``  ``mx4_matmul``: rows of a quantised matrix times the quantised weights of the group they belong to;
* ``moe``     ``mx4_moe``: router product, softmax top-k, gate-up, SiLU, down and the weighted sum for a few tokens;
* ``norm``    ``block_norm``: residual + scale * gate * rmsnorm(y), and its rmsnorm for the block that follows.

Sizes are those of the Qwen3-30B-A3B and Mixtral-8x7B expert layers this package serves, or generic odd ones.
"""
import math

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decoded token's activations
        {"name": "quant one token", "op": "quant", "rows": 1, "cols": 2048, "dtype": "bf16"},
        # a ragged prefill chunk's activations, as a router in fp16 leaves them
        {"name": "quant chunk", "op": "quant", "rows": 1021, "cols": 4096, "dtype": "fp16"},
        # bf16 expert weights on their way to 4-bit masters: the gate-up rows of 32 experts
        {"name": "quant experts", "op": "quant", "rows": 32 * 1536, "cols": 2048, "dtype": "bf16"},
        # a dense projection for a decode batch
        {"name": "matmul decode", "op": "matmul", "groups": 1, "rows": 16, "n": 4096, "k": 4096},
        # gate-up of a Qwen3-30B-A3B layer over 2,048 tokens at top-8: about 128 rows an expert, every expert ragged
        {"name": "matmul experts", "op": "matmul", "groups": 128, "rows": 2048 * 8, "n": 1536, "k": 2048},
        # gate-up of a Mixtral-8x7B layer over 2,048 tokens at top-2
        {"name": "matmul wide experts", "op": "matmul", "groups": 8, "rows": 2048 * 2, "n": 28672, "k": 4096},
        # Qwen3-30B-A3B, one sequence decoding
        {"name": "moe one token", "op": "moe", "tokens": 1, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 768},
        # Qwen3-30B-A3B, a decode batch
        {"name": "moe batch", "op": "moe", "tokens": 16, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 768},
        # Mixtral-8x7B, a decode batch
        {"name": "moe wide experts", "op": "moe", "tokens": 8, "experts": 8, "top_k": 2, "hidden": 4096, "inter": 14336},
        # after one decoded token's expert block
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 2048, "dtype": "bf16", "residual": "bf16",
         "post": False, "gate": "none"},
        # after a prefill chunk's expert block: both norms and a gate for each channel
        {"name": "norm chunk", "op": "norm", "rows": 2048, "cols": 4096, "dtype": "bf16", "residual": "bf16",
         "post": True, "gate": "channel"},
        # several chunks, an odd width, a residual kept in fp32 and a gate for each token
        {"name": "norm odd", "op": "norm", "rows": 8191, "cols": 2050, "dtype": "bf16", "residual": "fp32",
         "post": True, "gate": "token"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("quant", "matmul", "moe", "norm"))
    if op == "quant":
        cols = 32 * _log(rng, 4, 256)
        return {"op": op, "rows": _log(rng, 1, max(1, 80_000_000 // cols)), "cols": cols,
                "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    if op == "matmul":
        k, n, groups = 32 * _log(rng, 8, 128), _log(rng, 64, 8192), _log(rng, 1, 128)
        return {"op": op, "groups": groups, "rows": _log(rng, 1, 8192), "n": min(n, 400_000_000 // (k * groups)), "k": k}
    if op == "moe":
        experts, hidden, inter = _log(rng, 4, 160), 32 * _log(rng, 16, 128), 32 * _log(rng, 8, 128)
        return {"op": op, "tokens": _log(rng, 1, 64), "experts": experts, "top_k": rng.randint(1, min(8, experts)),
                "hidden": hidden, "inter": max(32, min(inter, 600_000_000 // (3 * hidden * experts) // 32 * 32))}
    cols = _log(rng, 64, 8192)
    return {"op": op, "rows": _log(rng, 1, max(1, 30_000_000 // cols)), "cols": cols,
            "dtype": rng.choice(("bf16", "fp16", "fp32")), "residual": rng.choice(("same", "fp32")),
            "post": rng.random() < 0.5, "gate": rng.choice(("none", "channel", "token", "full"))}


def _dtype(case, key="dtype"):
    name = case[key] if case[key] != "same" else case["dtype"]
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[name]


# ---- plain forms --------------------------------------------------------------------------------------------------

def _quantize(x):
    """(codes [..., K / 2], scale bytes [..., K / 32]) of x [..., K]."""
    v = x.float().unflatten(-1, (-1, 32))
    amax = v.abs().amax(-1)
    shared = (torch.frexp(amax).exponent - 3).clamp(-127, 127)
    a = (v.double() * torch.exp2(-shared.double()).unsqueeze(-1)).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + 8 * torch.signbit(v).to(torch.uint8)).flatten(-2)
    scales = torch.where(amax > 0, shared + 127, 0).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _dequantize(codes, scales, dtype):
    """Values of (codes, scale bytes) in `dtype`, each the exact product of its E2M1 value and its block's scale."""
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=codes.device)
    block = torch.exp2(scales.to(torch.float64) - 127).to(dtype)
    return (table[both.int()].unflatten(-1, (-1, 32)) * block.unsqueeze(-1)).flatten(-2)


def _plain_matmul(s):
    offsets, rows = s["offsets"].long(), s["a"].shape[0]
    at = torch.arange(rows, device=offsets.device)
    group = torch.searchsorted(offsets, at, right=True) - 1
    padded = torch.zeros(offsets.numel() - 1, s["most"], 2 * s["a"].shape[1], device=at.device)
    padded[group, at - offsets[group]] = _dequantize(s["a"], s["a_scales"], torch.float32)
    out = padded @ _dequantize(s["w"], s["w_scales"], torch.float32).transpose(1, 2)
    return out[group, at - offsets[group]].to(torch.bfloat16)


def _plain_moe(s):
    x = s["x"].float()
    logits = s["x"].double() @ s["gate"].double().t()
    best = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, ids = best.values[:, :s["top_k"]], best.indices[:, :s["top_k"]]
    share = torch.softmax(top, -1).float()
    weight = torch.zeros_like(logits, dtype=torch.float32).scatter_(1, ids, share)  # [T, E]
    hit = ids.unique()  # the experts that a token is routed to: [U]
    h = x @ _dequantize(s["w13"][hit], s["s13"][hit], torch.float32).transpose(1, 2)  # [U, T, 2I]
    g, u = h.chunk(2, -1)
    y = (g / (1 + torch.exp(-g)) * u) @ _dequantize(s["w2"][hit], s["s2"][hit], torch.float32).transpose(1, 2)
    return (y * weight[:, hit].t().unsqueeze(-1)).sum(0).to(torch.bfloat16)


def _plain_norm(s):
    z = s["y"].float()
    if s["post"] is not None:
        z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + s["eps"]) * s["post"].float()
    if s["gate"] is not None:
        z = z * s["gate"].float()
    r = s["residual"].float() + s["scale"] * z
    n = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + s["eps"]) * s["pre"].float()
    return n.to(s["y"].dtype), r.to(s["residual"].dtype)


# ---- inputs -------------------------------------------------------------------------------------------------------

def _weights(g, experts, rows, cols):
    """Quantised N(0, 0.02) weights of `experts` matrices, a few matrices at a time."""
    codes = torch.empty(experts, rows, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(experts, rows, cols // 32, dtype=torch.uint8, device="cuda")
    step = max(1, 60_000_000 // (rows * cols))
    for e in range(0, experts, step):
        w = torch.randn(min(step, experts - e), rows, cols, generator=g, device="cuda") * 0.02
        codes[e:e + step], scales[e:e + step] = _quantize(w)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"op": case["op"]}
    if case["op"] == "quant":
        # activations: a few channels far larger than the rest, as in trained models
        x = normal(case["rows"], case["cols"]) * torch.exp(normal(case["cols"]))
        s["x"] = x.to(_dtype(case))
    elif case["op"] == "matmul":
        k, n, groups, rows = case["k"], case["n"], case["groups"], case["rows"]
        s["a"], s["a_scales"] = _quantize(normal(rows, k))
        s["w"], s["w_scales"] = _weights(g, groups, n, k)
        ids = torch.randint(0, groups, (rows,), generator=g, device="cuda")
        counts = torch.bincount(ids, minlength=groups)
        s["offsets"] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
        s["most"] = int(counts.max())
    elif case["op"] == "moe":
        t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inter"]
        s["x"] = normal(t, h).to(torch.bfloat16)
        s["gate"] = (normal(e, h) / math.sqrt(h)).to(torch.bfloat16)
        s["w13"], s["s13"] = _weights(g, e, 2 * i, h)
        s["w2"], s["s2"] = _weights(g, e, h, i)
        s["top_k"] = case["top_k"]
    else:
        rows, cols, dtype = case["rows"], case["cols"], _dtype(case)
        s["y"] = (normal(rows, cols) * 0.3).to(dtype)
        s["residual"] = (normal(rows, cols) * 2).to(_dtype(case, "residual"))
        s["pre"] = (1 + 0.1 * normal(cols)).to(dtype)
        s["post"] = (1 + 0.1 * normal(cols)).to(dtype) if case["post"] else None
        shape = {"none": None, "channel": (cols,), "token": (rows, 1), "full": (rows, cols)}[case["gate"]]
        s["gate"] = None if shape is None else torch.tanh(normal(*shape)).to(dtype)
        s["scale"], s["eps"] = 0.25, 1e-6
    return s


def run(s):
    if not own:
        if s["op"] == "quant":
            return _dequantize(*_quantize(s["x"]), s["x"].dtype)
        return {"matmul": _plain_matmul, "moe": _plain_moe, "norm": _plain_norm}[s["op"]](s)
    from wisp_b200 import mx4, norm
    if s["op"] == "quant":
        return mx4.mx4_dequantize(mx4.mx4_quantize(s["x"]), s["x"].dtype)
    if s["op"] == "matmul":
        return mx4.mx4_matmul(mx4.Mx4Tensor(s["a"], s["a_scales"]), mx4.Mx4Tensor(s["w"], s["w_scales"]), s["offsets"])
    if s["op"] == "moe":
        return mx4.mx4_moe(s["x"], mx4.Mx4Tensor(s["w13"], s["s13"]), mx4.Mx4Tensor(s["w2"], s["s2"]), s["top_k"],
                           router=s["gate"])
    return norm.block_norm(s["y"], s["residual"], s["pre"], post_weight=s["post"], gate=s["gate"], scale=s["scale"],
                           eps=s["eps"])


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    mx4 = 0.5 + 1 / 32  # bytes of a value
    if case["op"] == "quant":
        count, size = case["rows"] * case["cols"], _dtype(case).itemsize
        return {"bytes": count * (2 * size + 2 * mx4), "flops": 0}
    if case["op"] == "matmul":
        k, n, rows = case["k"], case["n"], case["rows"]
        hit = case["groups"] * (1 - (1 - 1 / case["groups"]) ** rows)  # groups that a row falls in, on average
        return {"bytes": mx4 * k * (rows + hit * n) + 2 * rows * n, "flops": 2.0 * rows * n * k}
    if case["op"] == "moe":
        t, e, h, i, k = (case[x] for x in ("tokens", "experts", "hidden", "inter", "top_k"))
        hit = e * (1 - (1 - k / e) ** t)  # experts that a token is routed to, on average
        return {"bytes": hit * 3 * h * i * mx4 + 2 * e * h + 4 * t * h, "flops": 2.0 * t * (k * 3 * h * i + e * h)}
    count, size, more = case["rows"] * case["cols"], _dtype(case).itemsize, _dtype(case, "residual").itemsize
    gate = {"none": 0, "channel": case["cols"], "token": case["rows"], "full": count}[case["gate"]]
    return {"bytes": count * 2 * (size + more) + gate * size + (1 + case["post"]) * case["cols"] * size, "flops": 12 * count}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _values64(codes, scales):
    """fp64 values of E2M1 codes with E8M0 scales, from the formats' bit fields."""
    out = torch.empty(*codes.shape, 2, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes >> (4 * half)).int() & 15
        exponent, mantissa = (c >> 1) & 3, (c & 1).double()
        size = torch.where(exponent == 0, mantissa * 0.5, (1 + mantissa / 2) * torch.exp2(exponent.double() - 1))
        out[..., half] = torch.where(c >= 8, -size, size)
    out = out.reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    return out * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _exact_quant(s):
    x = s["x"].double()
    blocks = x.reshape(x.shape[0], -1, 32)
    top = blocks.abs().max(-1, keepdim=True).values
    unit = torch.exp2(torch.floor(torch.log2(top.clamp_min(1e-300))) - 2)
    unit = torch.where(unit * 4 > top, unit / 2, unit)  # log2 next to a power of two
    unit = torch.where(unit * 8 <= top, unit * 2, unit)
    v = blocks.abs() / unit
    # spacing of E2M1: 0.5 below 2, 1 below 4, 2 above; torch.round takes ties to even multiples of it
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0)).double()
    v = (torch.round(v / step) * step).clamp_max(6.0)
    return torch.where(top > 0, torch.sign(blocks) * v * unit, 0.0).reshape(x.shape)


def _exact_matmul(s):
    a, ends = _values64(s["a"], s["a_scales"]), s["offsets"].tolist()
    return torch.cat([a[p:q] @ _values64(s["w"][i], s["w_scales"][i]).T
                      for i, (p, q) in enumerate(zip(ends[:-1], ends[1:]))])


def _exact_moe(s):
    x = s["x"].double()
    scores = torch.exp(x @ s["gate"].double().T)
    chosen = torch.argsort(scores, dim=1, descending=True, stable=True)[:, :s["top_k"]].tolist()
    out = torch.zeros_like(x)
    for e in range(s["gate"].shape[0]):
        tokens = [t for t, ids in enumerate(chosen) if e in ids]
        if not tokens:
            continue
        h = x[tokens] @ _values64(s["w13"][e], s["s13"][e]).T
        inter = h.shape[1] // 2
        y = (torch.sigmoid(h[:, :inter]) * h[:, :inter] * h[:, inter:]) @ _values64(s["w2"][e], s["s2"][e]).T
        for row, t in enumerate(tokens):
            out[t] += y[row] * scores[t, e] / scores[t, chosen[t]].sum()
    return out


def _exact_norm(s):
    def rms(v, w):
        return v / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + s["eps"]) * w.double()

    z = s["y"].double()
    z = z if s["post"] is None else rms(z, s["post"])
    r = s["residual"].double() + s["scale"] * (z if s["gate"] is None else z * s["gate"].double())
    return rms(r, s["pre"]), r


def exact(case, seed):
    s = prepare(case, seed)
    return {"quant": _exact_quant, "matmul": _exact_matmul, "moe": _exact_moe, "norm": _exact_norm}[case["op"]](s)
