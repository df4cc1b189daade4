"""The 8-bit floating point path of a transformer's feed-forward and expert layers, operator by operator.

Values are e4m3 (torch.float8_e4m3fn) with one f32 scale for each block of 128 consecutive values of a row
(activations) or for each block of 128 x 128 values (weights); a value stands for q * scale. Each case names one
operator:

  quantize   rows of activations, or a weight matrix, into that form
  rms_norm   residual addition, root-mean-square norm and the 8-bit form of its result in one call
  silu_mul   silu(gate) * up, in the 8-bit form
  mul_mat    activations times a weight matrix, both in the 8-bit form
  grouped    the same product for rows that are grouped by expert, each group against its own weight matrix

`run` computes them from elementary torch operations, or with `own` set by the calls of feml_b200.ops.
"""
import math

import torch

own = False

BLOCK = 128
TOP = 448.0  # the largest e4m3 value
FLOOR = 2.0 ** -100  # least block maximum that a scale is made of: it and its reciprocal stay normal numbers
EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the attention's output of one token, before its output projection: nothing but latency
        {"name": "quantize 1x4096", "op": "quantize", "rows": 1, "k": 4096, "block_rows": 1, "type": "bf16"},
        # an f32 weight matrix brought into the 8-bit form when a model is loaded
        {"name": "quantize weight 11008x4096", "op": "quantize", "rows": 11008, "k": 4096, "block_rows": 128, "type": "f32"},
        # one token between two layers
        {"name": "rms_norm 1x4096", "op": "rms_norm", "rows": 1, "k": 4096, "residual": True, "type": "bf16"},
        # a long prompt between two layers
        {"name": "rms_norm 8192x4096", "op": "rms_norm", "rows": 8192, "k": 4096, "residual": True, "type": "bf16"},
        # eight sequences that decode together, with the f32 activations of this framework's own products
        {"name": "silu_mul 8x14336", "op": "silu_mul", "rows": 8, "k": 14336, "type": "f32"},
        # a prompt in the middle of a feed-forward layer
        {"name": "silu_mul 4096x11008", "op": "silu_mul", "rows": 4096, "k": 11008, "type": "bf16"},
        # one token: a matrix is read once
        {"name": "mul_mat 4096x4096 n1", "op": "mul_mat", "n": 1, "k": 4096, "m": 4096, "type": "f32"},
        # a batch of decoding sequences against a wide down-projection
        {"name": "mul_mat 14336x4096 n64", "op": "mul_mat", "n": 64, "k": 14336, "m": 4096, "type": "f32"},
        # a long prompt against an up-projection
        {"name": "mul_mat 4096x14336 n8192", "op": "mul_mat", "n": 8192, "k": 4096, "m": 14336, "type": "bf16"},
        # eight decoding tokens over eight experts: nearly every expert's matrix is read for a row or two
        {"name": "grouped 8 experts n8", "op": "grouped", "experts": 8, "n": 8, "selected": 2, "k": 4096, "m": 14336,
         "gather": True, "skew": 0.0, "dropped": 0.0, "type": "f32"},
        # a prompt over the same experts
        {"name": "grouped 8 experts n512", "op": "grouped", "experts": 8, "n": 512, "selected": 2, "k": 4096, "m": 14336,
         "gather": True, "skew": 0.0, "dropped": 0.0, "type": "bf16"},
        # the down-projection of many small experts with unequal shares, an eighth of the slots on other machines
        {"name": "grouped 64 experts n3001", "op": "grouped", "experts": 64, "n": 3001, "selected": 6, "k": 1408, "m": 2048,
         "gather": False, "skew": 1.0, "dropped": 0.125, "type": "bf16"},
    ]


def _size(rng, lo, hi, step=1):
    """A size between lo and hi, even over its logarithm, a multiple of `step`."""
    return max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))) // step * step)


def draw(rng):
    op = rng.choice(["quantize", "rms_norm", "silu_mul", "mul_mat", "grouped"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op in ("quantize", "rms_norm", "silu_mul"):
        # whole vectors in most cases, as hidden sizes are; any length in the others
        k = _size(rng, 64, 16384, rng.choice([64, 64, 8, 1]))
        rows = _size(rng, 1, max(1, min(16384, 11008 * 4096 // k)))
        if op == "quantize":
            return {"op": op, "rows": rows, "k": k, "block_rows": rng.choice([1, 128]), "type": kind}
        if op == "rms_norm":
            return {"op": op, "rows": rows, "k": k, "residual": rng.random() < 0.75, "type": kind}
        return {"op": op, "rows": rows, "k": k, "type": kind}
    if op == "mul_mat":
        k, m = _size(rng, 256, 16384, 16), _size(rng, 64, 16384, rng.choice([64, 1]))
        return {"op": op, "n": _size(rng, 1, max(1, min(8192, 8192 * 4096 * 14336 // (k * m)))), "k": k, "m": m, "type": kind}
    experts = _size(rng, 4, 128)
    k, m = _size(rng, 256, 8192, 16), _size(rng, 128, 16384, rng.choice([64, 1]))
    while experts * k * m > 8 * 4096 * 14336:
        k, m = max(256, k // 32 * 16), max(128, m // 2)
    selected = rng.randint(1, min(8, experts))
    n = _size(rng, 1, max(1, min(4096, 10 ** 9 // (experts * (k + m)))))  # the plain form pads every group to the largest
    return {"op": op, "experts": experts, "n": n, "selected": selected, "k": k, "m": m,
            "gather": rng.random() < 0.5, "skew": rng.choice([0.0, 0.5, 1.0]), "dropped": rng.choice([0.0, 0.0, 0.125, 0.5]),
            "type": kind}


def work(case):
    size = TYPES[case["type"]].itemsize
    op = case["op"]
    if op in ("quantize", "rms_norm", "silu_mul"):
        n = case["rows"] * case["k"]
        blocks = -(-case["rows"] // case.get("block_rows", 1)) * -(-case["k"] // BLOCK)
        reads = {"quantize": 1, "rms_norm": 3 if case.get("residual") else 1, "silu_mul": 2}[op]  # rms_norm: x, residual, their sum
        extra = case["k"] * size if op == "rms_norm" else 0
        return {"bytes": n * (reads * size + 1) + 4 * blocks + extra, "flops": n * {"quantize": 3, "rms_norm": 7, "silu_mul": 8}[op]}
    k, m, kb = case["k"], case["m"], -(-case["k"] // BLOCK)
    weight = k * m + 4 * kb * -(-m // BLOCK)
    if op == "mul_mat":
        return {"bytes": weight + case["n"] * (k + 4 * kb + m * size), "flops": 2 * case["n"] * k * m}
    slots = case["n"] * case["selected"]
    routed = max(1, round(slots * (1 - case["dropped"])))
    read = min(case["experts"], routed) if case["skew"] else case["experts"] * (1 - (1 - 1 / case["experts"]) ** routed)
    source = min(case["n"], routed) if case["gather"] else routed
    return {"bytes": read * weight + source * (k + 4 * kb) + routed * (m * size + 4), "flops": 2 * routed * k * m}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _to_blocks(x, rows):
    """An f32 matrix [..., r, k] in the 8-bit form with blocks of `rows` x 128."""
    r, k = x.shape[-2:]
    pad = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -r % rows))
    blocks = pad.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, rows))
    top = blocks.abs().amax((-3, -1), keepdim=True).clamp_min(FLOOR)
    q = (blocks * (TOP / top)).flatten(-4, -3).flatten(-2, -1)[..., :r, :k]
    return q.to(torch.float8_e4m3fn), (top / TOP).squeeze(-1).squeeze(-2).contiguous()


def _activations(g, rows, k, scale=1.0):
    """Rows of unequal size with a few channels that stand out, as hidden states have."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(k, generator=g, device="cuda")) * scale
    x[:, torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] *= 12.0
    return x * torch.exp(0.2 * torch.randn(rows, 1, generator=g, device="cuda"))


def _ids(g, case):
    """The experts of each token, [n, selected] without repetition; -1 where the expert is on another machine."""
    n, e, skew = case["n"], case["experts"], case["skew"]
    share = torch.arange(1, e + 1, device="cuda", dtype=torch.float32).pow(-skew).log()
    share = share[torch.randperm(e, generator=g, device="cuda")]
    noise = -torch.log(-torch.log(torch.rand(n, e, generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
    ids = (share + noise).topk(case["selected"], dim=1).indices
    return torch.where(torch.rand(ids.shape, generator=g, device="cuda") < case["dropped"], -1, ids)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, kind = case["op"], TYPES[case["type"]]
    s = {"op": op}
    if op in ("quantize", "rms_norm", "silu_mul"):
        rows, k, br = case["rows"], case["k"], case.get("block_rows", 1)
        if op == "silu_mul":
            # the two halves of one product's output
            both = _activations(g, rows, 2 * k).to(kind)
            s["gate"], s["up"] = both[:, :k], both[:, k:]
        elif br > 1:
            s["x"] = (torch.randn(rows, k, generator=g, device="cuda") * 0.02).to(kind)
        else:
            s["x"] = _activations(g, rows, k).to(kind)
        if op == "quantize":
            s["block_rows"] = br
        if op == "rms_norm":
            s["weight"] = (1 + 0.1 * torch.randn(k, generator=g, device="cuda")).to(kind)
            s["residual"] = _activations(g, rows, k, 3.0).to(kind) if case["residual"] else None
            s["sum"] = torch.empty(rows, k, dtype=kind, device="cuda") if case["residual"] else None
        s["out"] = torch.empty(rows, k, dtype=torch.float8_e4m3fn, device="cuda")
        s["scale"] = torch.empty(-(-rows // br), -(-k // BLOCK), device="cuda")
        return s
    k, m = case["k"], case["m"]
    if op == "mul_mat":
        s["w"], s["w_scale"] = _to_blocks(torch.randn(m, k, generator=g, device="cuda") * 0.02, BLOCK)
        s["x"], s["x_scale"] = _to_blocks(_activations(g, case["n"], k), 1)
        s["out"] = torch.empty(case["n"], m, dtype=kind, device="cuda")
        return s
    e = case["experts"]
    s["w"] = torch.empty(e, m, k, dtype=torch.float8_e4m3fn, device="cuda")
    s["w_scale"] = torch.empty(e, -(-m // BLOCK), -(-k // BLOCK), device="cuda")
    for i in range(e):
        s["w"][i], s["w_scale"][i] = _to_blocks(torch.randn(m, k, generator=g, device="cuda") * 0.02, BLOCK)
    ids = _ids(g, case).flatten()
    order = torch.argsort(torch.where(ids < 0, e, ids), stable=True)  # slots by expert, the dropped ones last
    counts = torch.bincount(ids[ids >= 0], minlength=e)
    s["counts"] = counts.to(torch.int32)
    s["offsets"] = (counts.cumsum(0) - counts).to(torch.int32)
    s["rows"] = order.to(torch.int32) if case["gather"] else None
    s["selected"] = case["selected"] if case["gather"] else 1
    s["x"], s["x_scale"] = _to_blocks(_activations(g, case["n"] if case["gather"] else ids.numel(), k), 1)
    s["most"] = max(1, int(counts.max()))
    # rows behind the last group keep what the buffer holds
    s["out"] = torch.zeros(ids.numel(), m, dtype=kind, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def _values(q, scale, rows):
    """The f32 values that the 8-bit form stands for."""
    r, k = q.shape[-2:]
    each = scale.repeat_interleave(rows, -2)[..., :r, :].repeat_interleave(BLOCK, -1)[..., :k]
    return q.float() * each


def _plain(s):
    op = s["op"]
    if op == "quantize":
        return _to_blocks(s["x"].float(), s["block_rows"])
    if op == "rms_norm":
        x, h = s["x"], None
        if s["residual"] is not None:
            x = h = (x.float() + s["residual"].float()).to(x.dtype)
        x = x.float()
        y = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
        return (*_to_blocks(y, 1), h)
    if op == "silu_mul":
        gate = s["gate"].float()
        return _to_blocks(gate / (1 + torch.exp(-gate)) * s["up"].float(), 1)
    if op == "mul_mat":
        return (_values(s["x"], s["x_scale"], 1) @ _values(s["w"], s["w_scale"], BLOCK).T).to(s["out"].dtype)
    # every group padded to the largest, one batched product, and its rows put where they belong
    slots, most = s["out"].shape[0], s["most"]
    j = torch.arange(most, device="cuda")
    at = s["offsets"][:, None] + j
    inside = j < s["counts"][:, None]
    source = at.clamp_max(slots - 1)
    if s["rows"] is not None:
        source = s["rows"][source] // s["selected"]
    y = torch.bmm(_values(s["x"], s["x_scale"], 1)[source], _values(s["w"], s["w_scale"], BLOCK).transpose(1, 2))
    out = torch.zeros(slots + 1, y.shape[-1], dtype=s["out"].dtype, device="cuda")
    out.index_copy_(0, torch.where(inside, at, slots).flatten(), y.flatten(0, 1).to(out.dtype))
    return out[:slots]


def run(state):
    if not own:
        return _plain(state)
    from feml_b200 import ops
    s, op = state, state["op"]
    if op == "quantize":
        return ops.quantize_f8(s["x"], block_rows=s["block_rows"], out=s["out"], scale=s["scale"])
    if op == "rms_norm":
        return ops.rms_norm_f8(s["x"], s["weight"], EPS, residual=s["residual"], residual_out=s["sum"], out=s["out"],
                               scale=s["scale"])
    if op == "silu_mul":
        return ops.silu_mul_f8(s["gate"], s["up"], out=s["out"], scale=s["scale"])
    if op == "mul_mat":
        return ops.mul_mat_f8(s["w"], s["w_scale"], s["x"], s["x_scale"], out=s["out"])
    return ops.mul_mat_f8_grouped(s["w"], s["w_scale"], s["x"], s["x_scale"], s["counts"], s["offsets"], rows=s["rows"],
                                  n_selected=s["selected"], out=s["out"])


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits; a value in 8 bits is given as it is before its rounding
# ---------------------------------------------------------------------------------------------------------------
def _exact_blocks(y, rows):
    r, k = y.shape
    scale = torch.zeros(-(-r // rows), -(-k // BLOCK), dtype=torch.float64, device=y.device)
    q = torch.empty_like(y)
    for b in range(scale.shape[1]):
        part = y[:, b * BLOCK:(b + 1) * BLOCK]
        top = part.abs().amax(1)
        if rows > 1:
            top = torch.stack([t.amax() for t in top.split(rows)])
        scale[:, b] = torch.clamp(top, min=FLOOR) / TOP
        q[:, b * BLOCK:(b + 1) * BLOCK] = part / scale[:, b].repeat_interleave(rows)[:r, None]
    return q, scale


def _exact_product(w, w_scale, x, x_scale):
    """sum over blocks b of x_scale[n, b] w_scale[m / 128, b] (sum over k in b of x[n, k] w[m, k])"""
    k, m = w.shape[1], w.shape[0]
    of = torch.arange(k, device=w.device) // BLOCK
    a = x.double() * x_scale.double()[:, of]
    b = w.double() * w_scale.double()[torch.arange(m, device=w.device) // BLOCK][:, of]
    return a @ b.t()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_blocks(s["x"].double(), case["block_rows"])
    if op == "rms_norm":
        x, h = s["x"].double(), None
        if case["residual"]:
            h = x + s["residual"].double()
            x = h.to(s["x"].dtype).double()  # the norm is that of the sum as it is stored
        inv = 1 / torch.sqrt((x * x).sum(1) / case["k"] + EPS)
        return (*_exact_blocks(x * inv[:, None] * s["weight"].double(), 1), h)
    if op == "silu_mul":
        gate = s["gate"].double()
        return _exact_blocks(gate * torch.sigmoid(gate) * s["up"].double(), 1)
    if op == "mul_mat":
        return _exact_product(s["w"], s["w_scale"], s["x"], s["x_scale"])
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for e, count in enumerate(s["counts"].tolist()):
        if count:
            take = torch.arange(at, at + count, device="cuda")
            if s["rows"] is not None:
                take = torch.div(s["rows"][take].long(), case["selected"], rounding_mode="floor")
            out[at:at + count] = _exact_product(s["w"][e], s["w_scale"][e], s["x"][take], s["x_scale"][take])
        at += count
    return out
