"""Products with matrices in 8 bits, a scale for each block of 128: weights, dense layers, and routed experts whose rows are ragged.

A number keeps 8 bits: sign, four bits of exponent, three of mantissa (e4m3, largest 448).  A weight has one float32 scale for
each block of 128 x 128 values, a row of activations one for each 128 neighbouring values: the block's largest magnitude / 448,
at least 2^-126, rounded to float32.  A code is the format's value nearest to x * 448 / largest, ties to even.

  quantise      a weight matrix [n, k], and the values that it stands for then
  product       rows x [t, k] (taken to 8 bits) times a weight [n, k], sums in 32 bits
  feed_forward  silu(x gate^T) * (x up^T), taken to 8 bits, times down: the gated layer of a dense model
  experts       the same for the experts that a router chose for each token, their results weighted and added up

Sizes are the layers' of the models that this engine serves (widths 1,024 to 4,096, feed-forwards of up to 12,288, 8 to 128
experts) and odd ones between.  Weights have a standard deviation of 1 / sqrt(inputs); activations one of 1, with a few channels
many times larger, as normed layers show them.  Some experts are chosen several times as often as others.
"""
import math

import torch

own = False

DEVICE = "cuda"
BLOCK = 128
TOP = 448.0
LEAST = 2.0 ** -126


def listed():
    return [
        # a feed-forward's matrix when a model is loaded
        dict(name="quantise_matrix", op="quantise", n=12288, k=4096, dtype="bfloat16"),
        # a matrix in 32 bits with sides that fill no block
        dict(name="quantise_odd", op="quantise", n=1003, k=1358, dtype="float32"),
        # one token being decoded, through the query, key and value projections: latency
        dict(name="product_token", op="product", t=1, n=6144, k=4096, out="float32"),
        # a few chats through the projection behind the feed-forward
        dict(name="product_chats", op="product", t=24, n=4096, k=12288, out="float32"),
        # ragged sizes between decoding and prompts
        dict(name="product_odd", op="product", t=197, n=2501, k=1358, out="bfloat16"),
        # a long prompt through a feed-forward's first matrix
        dict(name="product_prompt", op="product", t=4096, n=24576, k=4096, out="bfloat16"),
        # decoding a few chats
        dict(name="feed_forward_chats", op="feed_forward", t=8, ff=12288, k=4096),
        # a prompt
        dict(name="feed_forward_prompt", op="feed_forward", t=2045, ff=12288, k=4096),
        # one token being decoded: eight experts of 64
        dict(name="experts_token", op="experts", t=1, experts=64, top=8, ff=1024, k=2048),
        # four dozen chats being decoded: most experts, a few rows each
        dict(name="experts_chats", op="experts", t=48, experts=64, top=8, ff=1024, k=2048),
        # few experts with odd sides, a short prompt
        dict(name="experts_odd", op="experts", t=301, experts=8, top=2, ff=1450, k=1358),
        # a long prompt
        dict(name="experts_prompt", op="experts", t=4096, experts=64, top=8, ff=1024, k=2048),
    ]


def _between(rng, low, high):
    """A whole number spread evenly over the logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "product", "feed_forward", "feed_forward", "experts", "experts", "experts"])
    # half of the sides are whole blocks, as most layers have them, half are whatever comes
    side = lambda low, high: _between(rng, low, high) if rng.random() < 0.5 else BLOCK * _between(rng, max(1, low // BLOCK), high // BLOCK)
    if op == "quantise":
        return dict(op=op, n=side(64, 12288), k=side(64, 4096), dtype=rng.choice(["bfloat16", "float32"]))
    if op == "product":
        return dict(op=op, t=_between(rng, 1, 4096), n=side(64, 8192), k=side(64, 8192), out=rng.choice(["float32", "bfloat16"]))
    if op == "feed_forward":
        return dict(op=op, t=_between(rng, 1, 2048), ff=side(64, 12288), k=side(64, 4096))
    experts = rng.choice([8, 16, 24, 64, 128])
    k = side(256, 4096)
    ff = min(side(64, 2048), 64 * 1024 * 2048 // (experts * k))              # no more weights than the largest listed case
    top = rng.randint(1, 8)
    return dict(op=op, t=_between(rng, 1, max(1, min(4096, 4096 * 8 * 1024 * 2048 // (top * ff * k)))), experts=experts, top=top, ff=ff, k=k)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)
    matrix = lambda *shape: (normal(*shape) / math.sqrt(shape[-1])).to(torch.bfloat16)

    def activations(t, k):
        loud = torch.where(torch.rand((k,), generator=g, device=DEVICE) < 0.01, 12.0, 1.0)
        return (normal(t, k) * loud).to(torch.bfloat16)

    op, k = case["op"], case["k"]
    if op == "quantise":
        return {"w": (normal(case["n"], k) / math.sqrt(k)).to(getattr(torch, case["dtype"]))}
    if op == "product":
        return {"x": activations(case["t"], k), "w": matrix(case["n"], k)}
    if op == "feed_forward":
        return {"x": activations(case["t"], k), "gate_up": matrix(2 * case["ff"], k), "down": matrix(k, case["ff"])}
    experts, ff = case["experts"], case["ff"]
    got = {"x": activations(case["t"], k), "gate_up": matrix(experts, 2 * ff, k), "down": matrix(experts, k, ff)}
    score, ids = torch.topk(normal(case["t"], experts) + 0.5 * normal(experts), case["top"], dim=1)
    return dict(got, ids=ids.to(torch.int32), weights=torch.softmax(score, dim=1))


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    for name in ("w", "gate_up", "down"):                    # a program keeps the matrices in 8 bits only
        if name in state and case["op"] != "quantise":
            if own:
                from litellmengine_b200.csrc import ops
                state[name] = ops.f8_weight(state[name], gated=name == "gate_up")
            else:
                state[name] = _held(state[name].float(), BLOCK)
    if case["op"] == "experts":
        state["most"] = int(torch.bincount(state["ids"].view(-1).long()).max())      # rows that the plain form has room for
    return state


# ---- the plain form ----------------------------------------------------------------------------------------------
def _held(x, tall):
    """The values that x [..., rows, k] stands for in 8 bits, a scale for each block of `tall` rows and 128 values."""
    rows, k = x.shape[-2:]
    b = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -rows % tall)).unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, tall))
    most = b.abs().amax(dim=(-3, -1), keepdim=True)
    q = b * TOP / most.clamp(min=TOP * LEAST)
    step = torch.ldexp(torch.ones_like(q), (torch.frexp(q)[1] - 1).clamp(min=-6) - 3)
    scale = (most / TOP).clamp(min=LEAST).float()
    return ((torch.round(q / step) * step).float() * scale).flatten(-4, -3).flatten(-2, -1)[..., :rows, :k]


def _gated(y):
    gate, up = y.chunk(2, dim=-1)
    return gate / (1 + torch.exp(-gate)) * up


def _plain(state):
    case, bf16 = state["case"], torch.bfloat16
    if case["op"] == "quantise":
        # what is itself in 32 bits needs more for the values next to a border
        return _held(state["w"].double() if state["w"].dtype == torch.float32 else state["w"].float(), BLOCK).to(bf16)
    x = _held(state["x"].float(), 1)
    if case["op"] == "product":
        return (x @ state["w"].t()).to(getattr(torch, case["out"]))
    if case["op"] == "feed_forward":
        return (_held(_gated(x @ state["gate_up"].t()), 1) @ state["down"].t()).to(bf16)
    t, top, experts, k = case["t"], case["top"], case["experts"], case["k"]
    ids = state["ids"].view(-1).long()
    token = torch.arange(t, device=DEVICE).repeat_interleave(top)
    if t * top < experts:                                    # few rows: each with its own expert's matrices
        a = _held(_gated(torch.bmm(x[token, None], state["gate_up"][ids].transpose(1, 2))), 1)
        y = torch.bmm(a, state["down"][ids].transpose(1, 2))[:, 0]
    else:                                                    # every expert with room for the most rows that one has
        order = torch.argsort(ids, stable=True)
        first = torch.searchsorted(ids[order].contiguous(), torch.arange(experts, device=DEVICE))
        place = torch.empty_like(order)
        place[order] = torch.arange(t * top, device=DEVICE) - first[ids[order]]
        rows = torch.zeros((experts, state["most"], k), device=DEVICE)
        rows[ids, place] = x[token]
        a = _held(_gated(torch.bmm(rows, state["gate_up"].transpose(1, 2))), 1)
        y = torch.bmm(a, state["down"].transpose(1, 2))[ids, place]
    return (y.view(t, top, k) * state["weights"][..., None]).sum(dim=1).to(bf16)


# ---- the framework's calls ---------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    from litellmengine_b200.csrc import ops
    case, bf16 = state["case"], torch.bfloat16
    if case["op"] == "quantise":
        return ops.f8_weight(state["w"]).values(bf16)
    if case["op"] == "product":
        return ops.linear_f8(state["x"], state["w"], getattr(torch, case["out"]))
    if case["op"] == "feed_forward":
        return ops.linear_f8(ops.linear_silu_mul_f8(state["x"], state["gate_up"]), state["down"], bf16)
    return ops.moe_f8(state["x"], state["gate_up"], state["down"], state["ids"], state["weights"], out_dtype=bf16)


def work(case):
    op, k = case["op"], case["k"]
    if op == "quantise":
        n = case["n"] * k
        return {"bytes": n * (2 if case["dtype"] == "bfloat16" else 4) + n * 2, "flops": 3 * n}
    t = case["t"]
    if op == "product":
        n = case["n"]
        return {"bytes": t * k * 2 + n * k + t * n * (4 if case["out"] == "float32" else 2), "flops": 2 * t * n * k}
    ff, io = case["ff"], t * k * 4
    if op == "feed_forward":
        return {"bytes": io + 3 * ff * k, "flops": 6 * t * ff * k}
    # experts that this many picks reach, were all as likely
    reached = case["experts"] * (1 - (1 - case["top"] / case["experts"]) ** t)
    return {"bytes": io + reached * 3 * ff * k + t * case["top"] * 8, "flops": 6 * t * case["top"] * ff * k}


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------
def _nearest(x, tall):
    """x (64 bits, two dimensions) block by block: the nearest of the format's magnitudes, listed in order so that a place's parity is its last
    mantissa bit."""
    grid = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)]
    grid = torch.tensor([v for v in grid if v <= TOP], dtype=torch.float64, device=DEVICE)
    middle = (grid[1:] + grid[:-1]) / 2
    rows, k = x.shape
    out = torch.empty_like(x)
    for at in range(0, k, BLOCK):
        part = x[:, at:at + BLOCK]
        most = part.abs().amax(dim=1)
        if tall > 1:
            most = torch.cat([m.amax().expand(len(m)) for m in most.split(tall)])
        most = most[:, None]
        scale = torch.where(most / TOP > LEAST, most / TOP, LEAST)
        q = (part.abs() * TOP / torch.where(most / TOP > LEAST, most, TOP * LEAST)).contiguous()
        low = torch.searchsorted(middle, q)                  # the place just below, where q lies in a middle
        tie = (low < len(middle)) & (middle[low.clamp(max=len(middle) - 1)] == q) & (low % 2 == 1)
        out[:, at:at + BLOCK] = torch.sign(part) * grid[low + tie.to(low.dtype)] * scale.to(torch.float32).to(torch.float64)
    return out


def exact(case, seed):
    raw = _inputs(case, seed)
    double = lambda t: t.to(torch.float64)

    def layer(x, gate_up, down):
        y = torch.mm(x, _nearest(double(gate_up), BLOCK).t())
        gate, up = y[:, :case["ff"]], y[:, case["ff"]:]
        return torch.mm(_nearest(gate * torch.sigmoid(gate) * up, 1), _nearest(double(down), BLOCK).t())

    if case["op"] == "quantise":
        return _nearest(double(raw["w"]), BLOCK)
    x = _nearest(double(raw["x"]), 1)
    if case["op"] == "product":
        return torch.mm(x, _nearest(double(raw["w"]), BLOCK).t())
    if case["op"] == "feed_forward":
        return layer(x, raw["gate_up"], raw["down"])
    out = torch.zeros((case["t"], case["k"]), dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        token, choice = torch.nonzero(raw["ids"] == e, as_tuple=True)
        if len(token):
            out[token] += layer(x[token], raw["gate_up"][e], raw["down"][e]) * double(raw["weights"])[token, choice, None]
    return out
