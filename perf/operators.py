"""Microscaled products: weights held in 4 bits, the rows that meet them in 8, and the operators that make such rows.

A block of 32 neighbouring values shares one scale, a power of two (8 bits of exponent): the smallest with which the
block's largest magnitude stays within the format's largest value.  Each value is then rounded to the format's nearest
(ties to even).  4 bits: sign, two bits of exponent, one of mantissa (largest 6).  8 bits: sign, four of exponent, three of
mantissa (largest 448).

  quantise   a weight matrix [n, k] to 4 bits, and the values that it stands for then
  norm       v = stream + pending sum of the sublayer before; rows of rmsnorm(v) * w in 8 bits; v is the new stream
  product    rows x [t, k] (taken to 8 bits) times a 4-bit weight [n, k], sums in 32 bits
  gated      silu(x gate^T) * (x up^T) with gate and up in 4 bits, its result taken to 8 bits for the product behind it

Sizes are the layers' of the dense models that this engine serves (widths 1,024 to 4,096, feed-forwards of up to 12,288) and
odd ones between.  Weights have a standard deviation of 1 / sqrt(inputs); activations one of 1, with a few channels
many times larger, as normed layers and gated feed-forwards show them.
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 32
EPS = 1e-6
#: mantissa bits, least exponent, largest value as m * 2^e with m in [0.5, 1)
E2M1 = (1, 0, 0.75, 3)
E4M3 = (3, -6, 0.875, 9)


def listed():
    return [
        # a feed-forward's matrix when a model is loaded
        dict(name="quantise_matrix", op="quantise", n=12288, k=4096, dtype="bfloat16"),
        # a matrix in 32 bits with sides that fill no tile
        dict(name="quantise_odd", op="quantise", n=1003, k=1358, dtype="float32"),
        # one token being decoded: latency
        dict(name="norm_token", op="norm", t=1, k=4096, pending="float32"),
        # a prompt
        dict(name="norm_prompt", op="norm", t=4096, k=4096, pending="float32"),
        # a narrow odd stream, the pending sum in 16 bits
        dict(name="norm_odd", op="norm", t=333, k=1450, pending="bfloat16"),
        # one token through the query, key and value projections
        dict(name="product_token", op="product", t=1, n=6144, k=4096, out="float32"),
        # a few chats through the projection behind the feed-forward
        dict(name="product_chats", op="product", t=16, n=4096, k=12288, out="float32"),
        # ragged sizes between decoding and prompts
        dict(name="product_odd", op="product", t=197, n=2501, k=1358, out="bfloat16"),
        # a prompt's portion through the attention's output projection
        dict(name="product_portion", op="product", t=700, n=4096, k=4096, out="float32"),
        # a long prompt through a feed-forward's first matrix
        dict(name="product_prompt", op="product", t=4096, n=24576, k=4096, out="bfloat16"),
        # decoding a few chats
        dict(name="gated_chats", op="gated", t=8, n=12288, k=4096),
        # a prompt
        dict(name="gated_prompt", op="gated", t=2045, n=12288, k=4096),
    ]


def _between(rng, low, high):
    """A whole number spread evenly over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["quantise", "norm", "norm", "product", "product", "product", "gated", "gated"])
    # half of the sides are whole blocks, as layers have them, half are whatever comes
    side = lambda low, high: _between(rng, low, high) if rng.random() < 0.5 else BLOCK * _between(rng, low // BLOCK, high // BLOCK)
    if op == "quantise":
        return dict(op=op, n=side(64, 12288), k=side(64, 4096), dtype=rng.choice(["bfloat16", "float32"]))
    if op == "norm":
        return dict(op=op, t=_between(rng, 1, 4096), k=side(64, 4096), pending=rng.choice(["float32", "bfloat16", "none"]))
    if op == "product":
        return dict(op=op, t=_between(rng, 1, 4096), n=side(64, 8192), k=side(64, 8192), out=rng.choice(["float32", "bfloat16"]))
    return dict(op=op, t=_between(rng, 1, 2048), n=side(64, 12288), k=side(64, 4096))


# ---- inputs ------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)

    def activations(t, k):
        loud = torch.where(torch.rand((k,), generator=g, device=DEVICE) < 0.01, 12.0, 1.0)
        return normal(t, k) * loud

    op, k = case["op"], case["k"]
    if op == "quantise":
        return {"w": (normal(case["n"], k) / math.sqrt(k)).to(getattr(torch, case["dtype"]))}
    if op == "norm":
        got = {"h": activations(case["t"], k) * 3, "weight": 1 + 0.1 * normal(k), "pending": None}
        if case["pending"] != "none":
            got["pending"] = normal(case["t"], k).to(getattr(torch, case["pending"]))
        return got
    rows = 2 * case["n"] if op == "gated" else case["n"]
    return {"x": activations(case["t"], k).to(torch.bfloat16), "w": (normal(rows, k) / math.sqrt(k)).to(torch.bfloat16)}


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case["op"] == "norm":
        state["sum"] = torch.empty_like(state["h"])          # where the new stream goes
    if case["op"] in ("product", "gated"):
        w = state.pop("w")                                   # a program keeps the 4-bit weight only
        if own:
            from litellmengine_b200.csrc import ops
            state["w"] = ops.mx_weight(w, gated=case["op"] == "gated")
        else:
            state["w"] = _held(w.float(), E2M1)
    return state


# ---- the plain form ----------------------------------------------------------------------------------------------
def _power(e):
    """2^e in 32 bits for whole e of normal numbers."""
    return ((e.clamp(-126, 127) + 127) << 23).view(torch.float32)


def _held(x, fmt):
    """The values that float32 x [rows, k] stands for in a microscaled format."""
    bits, least, top_m, top_e = fmt
    rows, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % BLOCK)).view(rows, -1, BLOCK)
    m, e = torch.frexp(b.abs().amax(dim=-1, keepdim=True))
    scale = e - top_e + (m > top_m).to(torch.int32)          # frexp: the magnitude is m * 2^e, m in [0.5, 1)
    q = b * _power(-scale)
    step = _power((torch.frexp(q)[1] - 1).clamp(min=least) - bits)
    return (torch.round(q / step) * step * _power(scale)).view(rows, -1)[:, :k]


def _plain(state):
    case, bf16 = state["case"], torch.bfloat16
    if case["op"] == "quantise":
        return _held(state["w"].float(), E2M1).to(bf16)
    if case["op"] == "norm":
        v = state["h"] if state["pending"] is None else state["h"] + state["pending"].float()
        n = v / torch.sqrt(v.square().mean(dim=-1, keepdim=True) + EPS) * state["weight"]
        return v, _held(n, E4M3).to(bf16)
    y = _held(state["x"].float(), E4M3) @ state["w"].t()
    if case["op"] == "product":
        return y.to(getattr(torch, case["out"]))
    gate, up = y[:, :case["n"]], y[:, case["n"]:]
    return _held(gate / (1 + torch.exp(-gate)) * up, E4M3).to(bf16)


# ---- the framework's calls ---------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    from litellmengine_b200.csrc import ops
    case, bf16 = state["case"], torch.bfloat16
    if case["op"] == "quantise":
        return ops.mx_weight(state["w"]).values(bf16)
    if case["op"] == "norm":
        rows = ops.rmsnorm_mx(state["h"], state["weight"], EPS, delta=state["pending"], sum_out=state["sum"])
        return state["sum"], rows.values(bf16)
    if case["op"] == "product":
        return ops.linear_mx(state["x"], state["w"], getattr(torch, case["out"]))
    return ops.linear_silu_mul_mx(state["x"], state["w"]).values(bf16)


def work(case):
    op, k = case["op"], case["k"]
    held = 17 / 32                                           # bytes of a value in 4 bits with its share of the scale
    if op == "quantise":
        n = case["n"] * k
        return {"bytes": n * (2 if case["dtype"] == "bfloat16" else 4) + n * 2, "flops": 3 * n}
    t = case["t"]
    if op == "norm":
        pending = {"float32": 4, "bfloat16": 2, "none": 0}[case["pending"]]
        return {"bytes": t * k * (4 + pending + 4 + 2) + 4 * k, "flops": 8 * t * k}
    n = case["n"]
    if op == "product":
        return {"bytes": t * k * 2 + n * k * held + t * n * (4 if case["out"] == "float32" else 2), "flops": 2 * t * n * k}
    return {"bytes": t * k * 2 + 2 * n * k * held + t * n * 2, "flops": 4 * t * n * k}


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------
def _grid(bits, least, most, top):
    """Every magnitude of a format, in order: a place's parity is its last mantissa bit."""
    values = [m * 2.0 ** (least - bits) for m in range(2 ** bits)]
    for e in range(least, most + 1):
        values += [(1 + m / 2 ** bits) * 2.0 ** e for m in range(2 ** bits)]
    return torch.tensor([v for v in values if v <= top], dtype=torch.float64, device=DEVICE)


def _nearest(x, which):
    """x (64 bits) block by block to the nearest values of a format under the block's scale."""
    grid, top = (_grid(1, 0, 2, 6.0), 6.0) if which == 4 else (_grid(3, -6, 8, 448.0), 448.0)
    out = torch.empty_like(x)
    middle = (grid[1:] + grid[:-1]) / 2
    for at in range(0, x.shape[1], BLOCK):
        b = x[:, at:at + BLOCK]
        most = b.abs().amax(dim=1, keepdim=True)
        need = torch.where(most > 0, most / top, 1.0)
        scale = torch.exp2(torch.ceil(torch.log2(need)).clamp(min=-127))
        scale = torch.where(scale / 2 >= need, scale / 2, torch.where(scale < need, scale * 2, scale))
        q = (b.abs() / scale).contiguous()
        low = torch.searchsorted(middle, q)                  # the place just below, where q lies in a middle
        tie = (low < len(middle)) & (middle[low.clamp(max=len(middle) - 1)] == q) & (low % 2 == 1)
        out[:, at:at + BLOCK] = torch.sign(b) * grid[low + tie.to(low.dtype)] * scale
    return out


def exact(case, seed):
    raw = _inputs(case, seed)
    double = lambda t: t.to(torch.float64)
    if case["op"] == "quantise":
        return _nearest(double(raw["w"]), 4)
    if case["op"] == "norm":
        v = double(raw["h"])
        if raw["pending"] is not None:
            v = v + double(raw["pending"])
        mean = (v * v).sum(dim=1, keepdim=True) / case["k"]
        return v, _nearest(v * torch.rsqrt(mean + EPS) * double(raw["weight"]), 8)
    y = torch.mm(_nearest(double(raw["x"]), 8), _nearest(double(raw["w"]), 4).t())
    if case["op"] == "product":
        return y
    gate, up = torch.split(y, case["n"], dim=1)
    return _nearest(gate * torch.sigmoid(gate) * up, 8)
