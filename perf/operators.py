"""The MXFP4 operators' workloads: inputs, plain forms, values in 64 bits and the work each cannot do without.

Four operators: ``quantize`` (rows to 4-bit codes with one power-of-two scale per 32, and back to the values
they stand for), ``linear`` (the grouped product by expert on quantised operands), ``swiglu`` (the gate and up
products with silu(gate) * up) and ``experts`` (quantise, dispatch, both products, weighted combine).
Expert weights are held as a checkpoint holds them, as codes [G, N, K'/2] (low nibble first) and scales
[G, N, K'/32] (biased exponents), K' being K filled up to whole blocks; activations come in the layer's dtype and are quantised within the call.
"""
import importlib
import math

import torch

own = False

BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # one token's hidden state at decode, XL hidden size: launch latency
        {"name": "quantize-token", "op": "quantize", "rows": 1, "k": 1536, "dtype": "bf16"},
        # the hidden states of a 16K-token prefill
        {"name": "quantize-prefill", "op": "quantize", "rows": 16384, "k": 1536, "dtype": "bf16"},
        # the gate and up weights of an L-scale layer (64 x 896 rows) from fp32 masters
        {"name": "quantize-weights", "op": "quantize", "rows": 57344, "k": 1280, "dtype": "f32"},
        # down product of a 64-token decode step, XL: every expert's weight for about 8 rows
        {"name": "linear-decode", "op": "linear", "rows": 512, "groups": 64, "n": 1536, "k": 512, "skew": 0.0, "dead": 0},
        # down product of the L-scale layer: an odd row count, K not a multiple of 128, experts without rows
        {"name": "linear-odd", "op": "linear", "rows": 8191, "groups": 64, "n": 1280, "k": 448, "skew": 0.5, "dead": 3},
        # down product of a 16K-token prefill, XL, Zipf-loaded experts, four of them without rows
        {"name": "linear-prefill", "op": "linear", "rows": 131072, "groups": 64, "n": 1536, "k": 512, "skew": 1.2, "dead": 4},
        # gate and up of a single token at decode: 8 rows in 8 experts
        {"name": "swiglu-token", "op": "swiglu", "rows": 8, "groups": 64, "n": 512, "k": 1536, "skew": 0.0, "dead": 0},
        # gate and up of a 16K-token prefill, XL
        {"name": "swiglu-prefill", "op": "swiglu", "rows": 131072, "groups": 64, "n": 512, "k": 1536, "skew": 0.0, "dead": 0},
        # the experts of one token at decode, XL 64x8
        {"name": "experts-token", "op": "experts", "tokens": 1, "hidden": 1536, "inter": 512, "experts": 64, "top_k": 8, "skew": 0.0, "dead": 0},
        # a batch of 64 sequences at decode, XL 64x8
        {"name": "experts-decode", "op": "experts", "tokens": 64, "hidden": 1536, "inter": 512, "experts": 64, "top_k": 8, "skew": 0.0, "dead": 0},
        # a ragged chunk through 128 L-scale experts, Zipf-loaded
        {"name": "experts-chunk", "op": "experts", "tokens": 1001, "hidden": 1280, "inter": 448, "experts": 128, "top_k": 8, "skew": 1.2, "dead": 5},
        # a 16K-token prefill, XL 64x8
        {"name": "experts-prefill", "op": "experts", "tokens": 16384, "hidden": 1536, "inter": 512, "experts": 64, "top_k": 8, "skew": 0.0, "dead": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _by8(rng, lo, hi):
    return 8 * _log(rng, lo // 8, hi // 8)


def draw(rng):
    op = rng.choice(["quantize", "linear", "swiglu", "experts"])
    if op == "quantize":
        k = _by8(rng, 32, 4096)
        return {"op": op, "rows": _log(rng, 1, min(131072, 70_000_000 // k)), "k": k, "dtype": rng.choice(["bf16", "f32"])}
    skew = rng.choice([0.0, 0.5, 1.2])
    if op == "experts":
        experts = _log(rng, 2, 128)
        top_k = rng.randint(1, min(8, experts))
        return {"op": op, "tokens": _log(rng, 1, 16384), "hidden": _by8(rng, 64, 1536), "inter": _by8(rng, 32, 512),
                "experts": experts, "top_k": top_k, "skew": skew, "dead": rng.randint(0, min(4, experts - top_k))}
    groups = _log(rng, 1, 128)
    return {"op": op, "rows": _log(rng, 1, 131072 if groups >= 32 else 16384), "groups": groups,
            "n": _by8(rng, 32, 1536 if op == "linear" else 512), "k": _by8(rng, 64, 512 if op == "linear" else 1536),
            "skew": skew, "dead": rng.randint(0, min(4, groups - 1))}


# ------------------------------------------------------------------ inputs --
def _load(count, skew, dead, gen):
    """log of each expert's share of the rows: rank^-skew over a random order, nothing for the dead ones."""
    rank = torch.randperm(count, generator=gen, device="cuda").double()
    share = -skew * torch.log(rank + 1.0)
    return torch.where(rank >= count - dead, -math.inf, share)


def _activations(rows, k, dtype, gen):
    """N(0, 1) with a few channels ten times as large, as hidden states have them."""
    x = torch.randn((rows, k), generator=gen, device="cuda")
    wide = torch.rand((k,), generator=gen, device="cuda") < 0.005
    return torch.where(wide, 10.0 * x, x).to(dtype)


def _weights(groups, n, k, gen):
    """A checkpoint's MXFP4 weight of N(0, 0.02) values: codes [G, N, K'/2] and scales [G, N, K'/32]."""
    w = torch.randn((groups, n, k), generator=gen, device="cuda") * 0.02
    q, s = _to_mxfp4(w)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    code = torch.searchsorted(grid, q.abs()).to(torch.uint8)
    code += 8 * torch.signbit(q).to(torch.uint8)
    code = code.reshape(groups, n, -1, 2)
    return code[..., 0] + 16 * code[..., 1], (s + 127).to(torch.uint8)


def _pack(codes, scales, k, swiglu):
    """The weight as the framework's products take it, laid out once when a program loads it."""
    return importlib.import_module("hrm-moe_b200.ops").pack_mxfp4_weight((codes, scales), k, swiglu=swiglu)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantize":
        s["x"] = _activations(case["rows"], case["k"], DTYPES[case["dtype"]], gen)
        return s
    if case["op"] == "experts":
        t, d, i, e, k = (case[n] for n in ("tokens", "hidden", "inter", "experts", "top_k"))
        s["x"] = _activations(t, d, torch.bfloat16, gen)
        score = _load(e, case["skew"], case["dead"], gen) - torch.log(
            torch.empty((t, e), device="cuda", dtype=torch.float64).exponential_(generator=gen))
        top, idx = score.topk(k, dim=-1)
        s["selected"] = idx.to(torch.int32)
        s["routing"] = torch.softmax(top.float(), dim=-1).to(torch.bfloat16)
        s["most"] = int(torch.bincount(idx.reshape(-1), minlength=e).max())
        s["gate_up"] = _weights(e, 2 * i, d, gen)
        s["down"] = _weights(e, d, i, gen)
        if own:  # a serving program lays its weights out when it loads them
            s["gate_up_packed"] = _pack(*s["gate_up"], d, True)
            s["down_packed"] = _pack(*s["down"], i, False)
        return s
    swiglu = case["op"] == "swiglu"
    m, g, n, k = (case[c] for c in ("rows", "groups", "n", "k"))
    s["x"] = _activations(m, k, torch.bfloat16, gen)
    if swiglu and m < g:  # one row each in some of the experts, as a single token's are
        counts = torch.zeros(g, dtype=torch.int64, device="cuda")
        counts[torch.randperm(g, generator=gen, device="cuda")[:m]] = 1
    else:
        share = torch.softmax(_load(g, case["skew"], case["dead"], gen), dim=0)
        counts = torch.bincount(torch.multinomial(share, m, replacement=True, generator=gen), minlength=g)
    s["counts"] = counts.to(torch.int32)
    s["most"] = int(counts.max())
    s["weight"] = _weights(g, 2 * n if swiglu else n, k, gen)
    if own:
        s["packed"] = _pack(*s["weight"], k, swiglu)
    return s


# ------------------------------------------------------------- plain forms --
def _blocks(x):
    """[..., K] in fp32 as blocks of 32, the last one filled with zeros."""
    x = x.float()
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))


def _to_mxfp4(x):
    """e2m1 values [..., K'] and scale exponents [..., K'/32]: the block's largest power of two becomes e2m1's (4)."""
    b = _blocks(x)
    top = b.abs().amax(-1)
    exponent = (torch.frexp(top).exponent - 3).clamp(min=-127)  # frexp's mantissa is in [0.5, 1)
    exponent = torch.where(top == 0, -127, exponent)
    y = torch.ldexp(b, -exponent[..., None]).clamp(-6.0, 6.0)
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return (torch.round(y / step) * step).flatten(-2), exponent


def _values(x):
    """x rounded to MXFP4, in fp32 (exact: at most two significant bits each)."""
    q, e = _to_mxfp4(x)
    return torch.ldexp(q.unflatten(-1, (-1, BLOCK)), e[..., None]).flatten(-2)


def _weight_values(codes, scales):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()
    q = torch.where(code >= 8, -grid[code & 7], grid[code & 7])
    return torch.ldexp(q.unflatten(-1, (-1, BLOCK)), scales.int()[..., None] - 127).flatten(-2)


def _grouped(x, weight, group, place, most):
    """Row r of x times its group's weight: rows laid out [G, most, K] at (group, place), one batched product."""
    padded = x.new_zeros((weight.shape[0], most, x.shape[-1]))
    padded[group, place] = x
    return torch.bmm(padded, weight.transpose(1, 2))[group, place]


def _swiglu(gate_up):
    gate, up = gate_up.chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _plain_experts(s):
    t, k = s["selected"].shape
    flat = s["selected"].reshape(-1).long()
    counts = torch.bincount(flat, minlength=s["experts"])
    order = torch.argsort(flat, stable=True)
    group = flat[order]
    place = torch.arange(t * k, device=flat.device) - (torch.cumsum(counts, 0) - counts)[group]
    x = _values(s["x"])[order // k]
    h = _swiglu(_grouped(x, _weight_values(*s["gate_up"]), group, place, s["most"]))
    out = _grouped(_values(h), _weight_values(*s["down"]), group, place, s["most"])
    back = torch.empty_like(out)
    back[order] = out * s["routing"].float().reshape(-1)[order, None]
    return back.reshape(t, k, -1).sum(1).to(s["x"].dtype)


def run(s):
    if own:
        ops = importlib.import_module("hrm-moe_b200.ops")
        if s["op"] == "quantize":
            return ops.quantize_mxfp4(s["x"]).dequantize(torch.bfloat16)
        if s["op"] == "linear":
            return ops.grouped_linear_mxfp4(s["x"], s["packed"], s["counts"])
        if s["op"] == "swiglu":
            return ops.grouped_swiglu_mxfp4(s["x"], s["packed"], s["counts"])
        return ops.experts_forward_mxfp4(s["x"], s["selected"], s["routing"], s["gate_up_packed"], s["down_packed"])
    if s["op"] == "quantize":
        return _values(s["x"])[:, :s["k"]].to(torch.bfloat16)
    if s["op"] == "experts":
        return _plain_experts(s)
    counts = s["counts"].long()
    group = torch.repeat_interleave(torch.arange(s["groups"], device=counts.device), counts, output_size=s["rows"])
    place = torch.arange(s["rows"], device=counts.device) - (torch.cumsum(counts, 0) - counts)[group]
    out = _grouped(_values(s["x"]), _weight_values(*s["weight"]), group, place, s["most"])
    return (_swiglu(out) if s["op"] == "swiglu" else out).to(s["x"].dtype)


# ------------------------------------------------------- values in 64 bits --
def _nearest(x):
    """MXFP4 values of a float64 [R, K], by the definition: each element goes to the nearer of its two neighbours
    on the 4-bit grid, and from the middle to the one whose code is even."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    rows, k = x.shape
    b = torch.cat((x, x.new_zeros((rows, -k % BLOCK))), dim=1).reshape(-1, BLOCK)
    top = b.abs().max(dim=1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    e = e + (torch.exp2(e + 1) <= top).double() - (torch.exp2(e) > torch.where(top > 0, top, 1.0)).double()
    scale = torch.exp2(torch.clamp(torch.where(top > 0, e - 2, -127.0), min=-127.0))
    y = b.abs() / scale
    hi = torch.searchsorted(grid, y).clamp(max=7)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - y, y - grid[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (torch.sign(b) * grid[pick] * scale).reshape(rows, -1)[:, :k]


def _checkpoint(codes, scales, k):
    """One expert's weight [N, K] in float64."""
    n = codes.shape[0]
    code = torch.empty((n, 2 * codes.shape[1]), dtype=torch.int64, device=codes.device)
    code[:, 0::2], code[:, 1::2] = codes % 16, codes // 16
    mantissa, exponent, sign = code % 2, code // 2 % 4, 1.0 - 2.0 * (code // 8).double()
    q = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.exp2(exponent.double() - 1))
    return (sign * q * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, dim=1))[:, :k]


def _silu_up(z):
    n = z.shape[1] // 2
    return z[:, :n] * torch.special.expit(z[:, :n]) * z[:, n:]


def exact(case, seed):
    s = prepare(case, seed)
    x = _nearest(s["x"].double())
    if case["op"] == "quantize":
        return x
    if case["op"] == "experts":
        y = torch.zeros_like(x)
        for e in range(case["experts"]):
            token, slot = torch.nonzero(s["selected"] == e, as_tuple=True)
            if not len(token):
                continue
            w1 = _checkpoint(s["gate_up"][0][e], s["gate_up"][1][e], case["hidden"])
            w2 = _checkpoint(s["down"][0][e], s["down"][1][e], case["inter"])
            h = _nearest(_silu_up(x[token] @ w1.T))
            y[token] += s["routing"][token, slot].double()[:, None] * (h @ w2.T)
        return y
    out, start = [], 0
    for g, c in enumerate(s["counts"].tolist()):
        z = x[start:start + c] @ _checkpoint(s["weight"][0][g], s["weight"][1][g], case["k"]).T
        out.append(_silu_up(z) if case["op"] == "swiglu" else z)
        start += c
    return torch.cat(out)


# -------------------------------------------------------------------- work --
def work(case):
    mx = 17 / 32  # bytes per value: half a byte of code and a 32nd of a scale
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 2 * n, "flops": 2 * n}
    if case["op"] == "experts":
        t, d, i, k = (case[c] for c in ("tokens", "hidden", "inter", "top_k"))
        used = min(case["experts"] - case["dead"], t * k)
        return {"bytes": 4 * t * d + 6 * t * k + used * 3 * i * d * mx, "flops": 6 * t * k * d * i}
    m, n, k = case["rows"], case["n"], case["k"]
    wide = 2 * n if case["op"] == "swiglu" else n
    used = min(case["groups"] - case["dead"], m)
    return {"bytes": 2 * m * k + 2 * m * n + used * wide * k * mx, "flops": 2 * m * wide * k}
