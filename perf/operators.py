"""Measured calls of the operators on 4-bit microscaled floating point: quantisation, dense products, and products grouped by expert.

The format: a row is cut into blocks of 32 values; a block has one scale, a power of two held as its biased
exponent in 8 bits (255: the block is no number), and 32 values of one sign, two exponent and one mantissa bit
(0, 0.5, 1, 1.5, 2, 3, 4, 6).  With m the largest magnitude of a block the scale is 2^max(floor(log2 m) - 2, -127), and a
value becomes the nearest there is (a tie goes to the even code, larger ones to 6).  A block that holds an infinity or a
NaN is no number as a whole.  Products are those of the rows' and the weights' quantised values, summed in 32 bits.

Sizes are those of the Llama-3-8B and Llama-3.2-1B shapes and of the expert layers that ``bench.py`` measures.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# width, width of the dense feed-forward, experts, chosen experts, width of an expert
SIZES = {"1b": dict(d=2048, f=8192, experts=32, top=4, ef=1024),
         "8b": dict(d=4096, f=14336, experts=64, top=6, ef=1408)}


# ------------------------------------------------------------------------------------- cases
def listed() -> list:
    return [
        # a decoded token's row on its way into a product: nothing but latency
        dict(name="quantize_1b_row", kind="quantize", rows=1, k=2048, dtype="bfloat16"),
        # a float32 weight matrix at load time
        dict(name="quantize_8b_weight", kind="quantize", rows=14336, k=4096, dtype="float32"),
        # one user of a small model: the output projection of a decoded token
        dict(name="linear_1b_1", kind="linear", m=1, n=2048, k=2048, dtype="bfloat16"),
        # eight users: the down projection, a stream of weights
        dict(name="linear_8b_8", kind="linear", m=8, n=4096, k=14336, dtype="bfloat16"),
        # a prompt through the down projection: arithmetic
        dict(name="linear_8b_2048", kind="linear", m=2048, n=4096, k=14336, dtype="bfloat16"),
        # gate and up projections with SwiGLU, eight users
        dict(name="glu_8b_8", kind="glu", m=8, n=14336, k=4096, dtype="bfloat16", limit=0.0),
        # the same for a prompt of odd length of the small model
        dict(name="glu_1b_707", kind="glu", m=707, n=8192, k=2048, dtype="bfloat16", limit=0.0),
        # sixteen decoded tokens through routed gated experts, some of which get nothing
        dict(name="experts_up_8b_16", kind="up", size="8b", unit="gated", tokens=16, limit=0.0),
        # a prompt through the same: some 190 rows an expert
        dict(name="experts_up_8b_2048", kind="up", size="8b", unit="gated", tokens=2048, limit=0.0),
        # a short prompt through ungated experts whose weights multiply what enters
        dict(name="experts_up_1b_707", kind="up", size="1b", unit="relu_squared", tokens=707, limit=0.0),
        # the experts' second product and the sum over a token's experts: decoded tokens, a prompt
        dict(name="experts_down_1b_16", kind="down", size="1b", tokens=16),
        dict(name="experts_down_8b_2048", kind="down", size="8b", tokens=2048),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["quantize", "linear", "linear", "glu", "glu", "up", "up", "down"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "quantize":
        rows = _log(rng, 1, 14336)
        return dict(kind=kind, rows=rows, k=min(_log(rng, 32, 14336), 14336 * 4096 // rows), dtype=dtype)
    if kind == "linear":
        return dict(kind=kind, m=_log(rng, 1, 2048), n=_log(rng, 256, 4096), k=_log(rng, 256, 14336), dtype=dtype)
    if kind == "glu":
        return dict(kind=kind, m=_log(rng, 1, 2048), n=_log(rng, 256, 7168), k=_log(rng, 256, 4096), dtype=dtype,
                    limit=rng.choice([0.0, 7.0]))
    size = rng.choice(["1b", "8b"])
    if kind == "up":
        return dict(kind=kind, size=size, unit=rng.choice(["gated", "relu_squared"]), tokens=_log(rng, 1, 2048),
                    limit=rng.choice([0.0, 7.0]))
    return dict(kind=kind, size=size, tokens=_log(rng, 1, 2048))


def _dtype(case):
    return torch.float32 if case.get("dtype") == "float32" else torch.bfloat16


# ------------------------------------------------------------------------------------- inputs
class _Inputs:
    """Tensors in the order in which they are asked for, from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 29)

    def __call__(self, *shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=self.gen)


def _raw(case, seed) -> dict:
    """A case's inputs before anything is quantised: rows as a norm leaves them (unit variance, some channels
    larger), weights N(0, 0.02^2), a routing in which some experts are liked better."""
    draw_, kind = _Inputs(seed), case["kind"]
    if kind == "quantize":
        x = draw_(case["rows"], case["k"], dtype=torch.float32)
        x *= torch.exp(draw_(case["k"], dtype=torch.float32))
        x[::7, : case["k"] // 2] = 0.0
        return {"x": x.to(_dtype(case))}
    if kind in ("linear", "glu"):
        rows = (case["n"], case["k"]) if kind == "linear" else (2, case["n"], case["k"])
        return {"a": draw_(case["m"], case["k"], dtype=_dtype(case)), "w": draw_(*rows, std=0.02)}
    s = SIZES[case["size"]]
    t, e, top = case["tokens"], s["experts"], s["top"]
    liked = draw_(t, e, dtype=torch.float32) + 0.5 * draw_(e, dtype=torch.float32)
    best = liked.topk(top, dim=1)
    idx = best.indices.reshape(-1)
    by_expert = torch.sort(idx, stable=True)
    offsets = torch.searchsorted(by_expert.values, torch.arange(e + 1, device=DEV))
    out = {"idx": idx.int(), "order": by_expert.indices.int(), "offsets": offsets.int(),
           "weight": torch.softmax(best.values, dim=1).reshape(-1).contiguous()}
    if kind == "up":
        mats = (2,) if case["unit"] == "gated" else ()
        out.update(a=draw_(t, s["d"]), w=draw_(e, *mats, s["ef"], s["d"], std=0.02))
    else:
        out.update(a=draw_(t * top, s["ef"]), w=draw_(e, s["d"], s["ef"], std=0.02))
    return out


_OPS = []


def _ops():
    if not _OPS:
        from mini_llm_stack_b200.ops.kernels import Runtime
        _OPS.append(Runtime(DEV, torch.bfloat16).ops)
    return _OPS[0]


def prepare(case, seed) -> dict:
    """The inputs, the weights as 4-bit values in the form that the products read, and memory for the outputs."""
    s = dict(_raw(case, seed), case=case)
    kind, bf16, f32 = case["kind"], torch.bfloat16, torch.float32
    if kind == "quantize":
        s["out"] = torch.empty_like(s["x"])
        if own:
            s["ops"] = _ops()
        return s
    w = s.pop("w")
    if own:
        s["ops"] = _ops()
        s["w"] = s["ops"].prepare_weight_mx4(w, gate_up=kind == "glu" or case.get("unit") == "gated")
    else:
        s["w"] = (*_quantized(w), w.shape[-1])
    del w
    if kind in ("linear", "glu"):
        s["out"] = torch.empty((case["m"], case["n"]), dtype=bf16, device=DEV)
        return s
    z = SIZES[case["size"]]
    s["top"], s["most"] = z["top"], int(s["offsets"].diff().max())
    slots = case["tokens"] * z["top"]
    if kind == "up":
        s["out"] = torch.empty((slots, z["ef"]), dtype=bf16, device=DEV)
    else:
        s["per_slot"] = torch.empty((slots, z["d"]), dtype=f32, device=DEV)
        s["out"] = torch.empty((case["tokens"], z["d"]), dtype=bf16, device=DEV)
    return s


# ------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        return _values(*_quantized(s["x"]), s["x"].shape[-1]).to(s["x"].dtype)
    a = _rounded(s["a"])
    if kind == "linear":
        return (a @ _values(*s["w"]).T).to(torch.bfloat16)
    if kind == "glu":
        gate, up = (a @ _values(*s["w"]).transpose(1, 2)).unbind(0)
        return _unit(gate, up, case["limit"]).to(torch.bfloat16)
    slots = s["order"].numel()
    # every expert's rows side by side, as many places each as the expert with the most has
    starts = s["offsets"][:-1].long()
    expert = s["idx"][s["order"].long()].long()
    place = expert * s["most"] + torch.arange(slots, device=DEV) - starts[expert]
    rows = a[s["order"].long() // s["top"]] if kind == "up" else a
    padded = a.new_zeros((starts.numel() * s["most"], a.shape[1])).index_copy_(0, place, rows)
    padded = padded.view(starts.numel(), s["most"], -1)
    w = _values(*s["w"])
    if kind == "down":
        sums = torch.bmm(padded, w.transpose(1, 2)).flatten(0, 1)[place]
        sums = sums * s["weight"][s["order"].long(), None]
        per_slot = torch.empty_like(sums).index_copy_(0, s["order"].long(), sums)
        return per_slot.view(case["tokens"], s["top"], -1).sum(1).to(torch.bfloat16)
    sums = torch.matmul(padded, w.flatten(1, -2).transpose(1, 2)).flatten(0, 1)[place]
    if case["unit"] == "relu_squared":
        return (sums * s["weight"][s["order"].long(), None]).relu().square().to(torch.bfloat16)
    gate, up = sums.chunk(2, dim=1)
    return _unit(gate, up, case["limit"]).to(torch.bfloat16)


def _run_own(s):
    ops, case = s["ops"], s["case"]
    kind = case["kind"]
    if kind == "quantize":
        ops.mx4_values(ops.quantize_mx4(s["x"]), s["out"])
    elif kind == "linear":
        ops.linear_mx4(s["a"], s["w"], s["out"])
    elif kind == "glu":
        ops.linear_glu_mx4(s["a"], s["w"], s["out"], limit=case["limit"])
    elif kind == "up" and case["unit"] == "gated":
        ops.expert_glu_mx4(s["a"], s["w"], s["out"], s, s["top"], False, limit=case["limit"])
    elif kind == "up":
        ops.expert_relu_squared_mx4(s["a"], s["w"], s["out"], s, s["top"], True)
    else:
        ops.expert_down_mx4(s["a"], s["w"], s["per_slot"], s, s["top"], True)
        ops.expert_combine(s["per_slot"], s["top"], None, s["out"])
    return s["out"]


def _unit(gate, up, limit):
    if limit > 0:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit) + 1
    return gate / (1 + torch.exp(-gate)) * up


def _quantized(x):
    """(codes, two to a byte with the even place in the low bits; scales) of the last axis, blocks filled up with zeros."""
    k = x.shape[-1]
    blocks = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    most = blocks.abs().amax(-1)
    # most = fraction * 2^e with a fraction of at least 1/2
    e = (torch.frexp(most).exponent - 3).clamp(min=-127)
    e = torch.where(most > 0, e, -127)
    # (a block's largest value is below 8 behind its scale; two steps, as 2^127 is the largest power there is)
    v = torch.ldexp(torch.ldexp(blocks.abs(), (-e[..., None]).clamp(max=100)), (-e[..., None] - 100).clamp(min=0))
    code = ((v > 0.25).byte() + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0))
    code = code + 8 * (blocks < 0).byte()
    fine = torch.isfinite(most)
    scales = torch.where(fine, e + 127, 255).byte()
    code = torch.where(fine[..., None], code, 0).flatten(-2)
    return code[..., ::2] | code[..., 1::2] << 4, scales


def _values(codes, scales, k):
    """What codes and scales stand for, in 32 bits."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=DEV)
    v = grid[torch.stack((codes & 15, codes >> 4), -1).int()].flatten(-2).unflatten(-1, (-1, BLOCK))
    e = scales.int() - 127
    scale = torch.where(scales == 255, math.nan, torch.ldexp(torch.ldexp(torch.ones_like(e).float(), e // 2), e - e // 2))
    return (v * scale[..., None]).flatten(-2)[..., :k]


def _rounded(x):
    return _values(*_quantized(x), x.shape[-1])


# ------------------------------------------------------------------------------------- work
def work(case) -> dict:
    """Rows and weights read once (weights as 4-bit values with their scales), outputs written once."""
    kind, four = case["kind"], 0.5 + 1 / BLOCK
    wide = 4 if case.get("dtype") == "float32" else 2
    if kind == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 * wide + four), "flops": 2 * n}
    if kind in ("linear", "glu"):
        m, n, k = case["m"], case["n"], case["k"]
        weights = n * k * (2 if kind == "glu" else 1)
        return {"bytes": m * k * wide + weights * four + m * n * 2, "flops": 2 * m * weights}
    s, t = SIZES[case["size"]], case["tokens"]
    slots = t * s["top"]
    asked = s["experts"] * (1 - (1 - s["top"] / s["experts"]) ** t)           # experts that get a row, on average
    matrix = s["d"] * s["ef"] * (2 if case.get("unit") == "gated" else 1)
    rows = t * s["d"] + slots * s["ef"]                                       # read and written, or the other way round
    return {"bytes": asked * matrix * four + rows * 2, "flops": 2 * slots * matrix}


# ------------------------------------------------------------------------------------- exact
def _nearest(x):
    """The format's nearest values in 64 bits, from its definition: a step of a quarter of the scale's power below 2, a half of
    it up to 4, a whole one above."""
    x = x.double()
    k = x.shape[-1]
    short = -k % BLOCK
    if short:
        x = torch.cat((x, x.new_zeros((*x.shape[:-1], short))), -1)
    x = x.view(*x.shape[:-1], -1, BLOCK)
    top = x.abs().max(-1, keepdim=True).values
    whole = torch.floor(torch.log2(top.clamp(min=2.0 ** -149)))
    # (the logarithm of a value just below a power of two may round up to it)
    whole = torch.where(2.0 ** whole > top.clamp(min=2.0 ** -149), whole - 1, whole)
    scale = 2.0 ** (whole - 2).clamp(min=-127)
    v = x / scale
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0)).double()
    v = (torch.round(v / step) * step).clamp(-6, 6) * scale
    v = torch.where(torch.isfinite(top), v, math.nan)
    return v.flatten(-2)[..., :k]


def exact(case, seed):
    r, kind = _raw(case, seed), case["kind"]
    if kind == "quantize":
        return _nearest(r["x"])
    a = _nearest(r["a"])

    def unit(gate, up):
        limit = case["limit"]
        if limit > 0:
            gate, up = torch.clamp(gate, max=limit), torch.clamp(up, -limit, limit) + 1.0
        return gate * torch.sigmoid(gate) * up

    if kind == "linear":
        return a @ _nearest(r["w"]).T
    if kind == "glu":
        return unit(a @ _nearest(r["w"][0]).T, a @ _nearest(r["w"][1]).T)
    s = SIZES[case["size"]]
    offsets, order, weight = r["offsets"].tolist(), r["order"].long(), r["weight"].double()
    if kind == "up":
        out = a.new_empty((order.numel(), s["ef"]))
    else:
        out = a.new_empty((order.numel(), s["d"]))
    for e in range(s["experts"]):
        lo, hi = offsets[e], offsets[e + 1]
        if lo == hi:
            continue
        slot = order[lo:hi]
        if kind == "down":
            out[slot] = a[lo:hi] @ _nearest(r["w"][e]).T * weight[slot, None]
        elif case["unit"] == "gated":
            x = a[slot // s["top"]]
            out[lo:hi] = unit(x @ _nearest(r["w"][e, 0]).T, x @ _nearest(r["w"][e, 1]).T)
        else:
            x = a[slot // s["top"]] @ _nearest(r["w"][e]).T * weight[slot, None]
            out[lo:hi] = torch.clamp(x, min=0.0) ** 2
    return out.view(case["tokens"], s["top"], -1).sum(1) if kind == "down" else out
