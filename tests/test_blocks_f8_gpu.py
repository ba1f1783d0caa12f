"""Rows, weights and products of 8 bits against their definition in 64 bits: a float32 scale for each block of 128 (128 x 128 of a weight), the block's
largest magnitude / 448; codes to the nearest of x * 448 / largest (ties to even).  Routed experts on top of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64, F32, BF16 = torch.float64, torch.float32, torch.bfloat16
LEAST = 2.0 ** -126


def ops():
    from litellmengine_b200.csrc import ops as o
    return o


def blocks(x, tall):
    rows, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % 128, 0, -rows % tall))
    return b.view(b.shape[0] // tall, tall, -1, 128)


def flat(b, rows, k):
    return b.reshape(b.shape[0] * b.shape[1], -1)[:rows, :k]


def held(x, tall):
    """The values that x stands for, as float32 (a code times a scale, rounded); NaN where a block holds something that is not finite."""
    b = blocks(x.to(F64), tall)
    most = b.abs().amax(dim=(1, 3), keepdim=True)
    scale = (most / 448).clamp(min=LEAST).to(F32)
    q = b * 448 / most.clamp(min=448 * LEAST)
    step = torch.exp2(torch.floor(torch.log2(torch.where(q == 0, 1.0, q.abs()))).clamp(min=-6) - 3)
    got = (torch.round(q / step) * step).to(F32) * scale          # torch.round: ties to even
    got = torch.where(b.isfinite().all(dim=3, keepdim=True).all(dim=1, keepdim=True), got, float("nan"))
    return flat(got, *x.shape)


def same(got, want):
    return torch.equal(got.nan_to_num(1e30), want.to(got.dtype).nan_to_num(1e30)) and torch.equal(got.isnan(), want.isnan())


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("rows,k", [(1, 1), (1, 127), (3, 129), (2, 255), (129, 128), (5, 1000), (64, 136), (300, 2056), (1, 4096), (1030, 4104)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_codes_are_the_nearest(rows, k, dtype):
    o, g = ops(), gen(rows * 7 + k)
    x = normal(g, rows, k, dtype=dtype) * torch.exp2(torch.randint(-8, 8, (rows, k), generator=g, device=DEV)).to(dtype)
    made = o.f8_rows(x)
    assert same(made.values(F32), held(x, 1)) and same(made.values(BF16), held(x, 1))
    assert made.codes[-1, :rows, (k - 1) % 128 + 1:].count_nonzero() == 0
    w = o.f8_weight(x)
    assert same(w.values(F32), held(x, 128)) and same(w.values(BF16), held(x, 128))
    two = torch.cat([x, -3 * x])
    w = o.f8_weight(two, gated=True)
    assert w.shape == (2 * rows, k) and same(w.values(F32), held(two, 128))
    unaligned = torch.empty(rows * k + 1, dtype=dtype, device=DEV)[1:].view(rows, k).copy_(x)
    assert same(o.f8_rows(unaligned).values(F32), held(x, 1)) and same(o.f8_weight(unaligned).values(F32), held(x, 128))
    wide = torch.zeros(rows, k + 24, dtype=dtype, device=DEV)
    wide[:, 8:k + 8] = x                                          # rows further apart than they are long
    assert same(o.f8_weight(wide[:, 8:k + 8]).values(F32), held(x, 128))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ties_and_what_is_not_finite(dtype):
    """Every pair of a magnitude and a largest one among bfloat16's, so that every quotient that is a middle between two codes is among them."""
    o = ops()
    top = (128 + torch.arange(128, device=DEV)).to(F32)[:, None]  # mantissas
    x = (128 + torch.arange(128, device=DEV)).to(F32)[None, :]
    rows = []
    for e in range(0, 18):
        small = x * 2.0 ** -e
        rows.append(torch.cat([top, torch.where(small <= top, small, 0.0)[:, :127]], dim=1))
        rows.append(torch.cat([top, torch.where(small <= top, -small, 0.0)[:, 1:]], dim=1))
    m = torch.cat(rows)
    for s in (1.0, 2.0 ** -60, 2.0 ** 100):
        v = (m * s).to(dtype)
        assert same(o.f8_rows(v).values(F32), held(v, 1))
    if dtype == F32:                                              # a hair beside each of them
        for near in (torch.nextafter(m, torch.full_like(m, 1e30)), torch.nextafter(m, torch.full_like(m, -1e30))):
            near[:, 0] = m[:, 0]
            near = torch.where(near.abs() <= m[:, :1], near, 0.0)
            assert same(o.f8_rows(near).values(F32), held(near, 1))
    big, tiny, nan, inf = 3.3e38, 1e-40, float("nan"), float("inf")
    odd = torch.zeros(9, 256, device=DEV)
    odd[0, 3], odd[1], odd[2, 200], odd[3, 0], odd[4, 128:] = nan, tiny, -inf, big, -big
    odd[5], odd[6], odd[7, ::2] = 448 * LEAST, 447 * LEAST, -0.0
    odd[8, 7] = 2.0 ** -126
    odd = odd.to(dtype)
    assert same(o.f8_rows(odd).values(F32), held(odd, 1))
    wide = torch.ones(300, 300, dtype=dtype, device=DEV)
    wide[130, 5], wide[299, 299], wide[0, 200] = inf, nan, 0.0
    assert same(o.f8_weight(wide).values(F32), held(wide, 128))


def test_offsets_beyond_32_bits():
    o, g = ops(), gen(3)
    T, K = 33000, 66000                                           # 2.2e9 values
    x = torch.zeros(T, K, dtype=BF16, device=DEV)
    ends = [0, 127, 128, T // 2, T - 2, T - 1]
    for r in ends:
        x[r] = normal(g, K, dtype=BF16)
    made = o.f8_rows(x)
    assert same(made.values(BF16)[ends], held(x[ends], 1))
    del made
    w = o.f8_weight(x)
    got = w.values(BF16)
    assert same(got[:128], held(x[:128], 128)) and same(got[-104:], held(x[-104:], 128))


ROWS = (1, 7, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 300)


def near(K, carried):
    """K / 32 steps of the tensor core, each cut at 2^-23 of what the sum holds; a scale's product, its product with a tile's sum and the addition, 2^-24 each, for
    K / 128 tiles; the parts' additions."""
    return (K / 32 + 1.5 * K / 128 + 16) * 2.0 ** -23 * carried


def product(x, w):
    return x.to(F64) @ w.to(F64).T, x.to(F64).abs() @ w.to(F64).abs().T


@pytest.mark.parametrize("N,K", [(1, 1), (16, 32), (100, 200), (129, 128), (127, 1024), (1000, 1358), (640, 4104), (4096, 640), (6144, 4096), (2500, 12288)])
def test_product(N, K):
    o, g = ops(), gen(N + K)
    W = o.f8_weight(normal(g, N, K) * K ** -0.5)
    w = W.values(F32)
    for T in ROWS:
        x = normal(g, T, K, dtype=BF16) * (1 + 11 * (torch.rand(K, generator=g, device=DEV) < 0.01)).to(BF16)
        X = o.f8_rows(x)
        want, carried = product(X.values(F32), w)
        got = o.linear_f8(X, W)
        assert bool(((got.to(F64) - want).abs() <= near(K, carried)).all()), T
        assert torch.equal(o.linear_f8(x, W), got)                # the call takes the rows to 8 bits by itself, and gives the same again
        assert torch.equal(o.linear_f8(X, W, BF16), got.to(BF16))
        stream = normal(g, T, N)
        total = stream + got
        assert o.linear_f8(X, W, residual=stream) is stream and torch.equal(stream, total)
    assert o.stream_status(torch.device(DEV)).tolist() == [0, 0]


def middle(gate, up, act, limit):
    if act == 2:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        return gate * torch.sigmoid(1.702 * gate) * (up + 1)
    return (torch.nn.functional.gelu(gate, approximate="tanh") if act == 1 else gate * torch.sigmoid(gate)) * up


def half_step(n):
    """What rounding moves n by at most: 2^-4 of it, or half the smallest step of its block, 2^-10 of a scale."""
    b = blocks(n, 1)
    s = (b.abs().amax(dim=3, keepdim=True) / 448).expand_as(b)
    return torch.maximum(n.abs() * 2.0 ** -4, flat(s, *n.shape) * 2.0 ** -10)


@pytest.mark.parametrize("N,K", [(1, 32), (64, 128), (100, 200), (192, 520), (700, 1358), (4096, 640), (12288, 512), (1450, 4096)])
@pytest.mark.parametrize("activation,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("clamped_swish", 1.5)])
def test_gated_product(N, K, activation, limit):
    o, g = ops(), gen(N + K + 1)
    W = o.f8_weight(normal(g, 2 * N, K) * K ** -0.5, gated=True)
    w = W.values(F32)
    for T in ROWS:
        x = normal(g, T, K, dtype=BF16)
        X = o.f8_rows(x)
        y, carried = product(X.values(F32), w)
        gate, up = y[:, :N], y[:, N:]
        want = middle(gate, up, o.ACTIVATIONS[activation], limit)
        # the sums' own error, which no factor multiplies by more than 1.7 of the other side's; less than 32 roundings of 2^-24 in the activation
        off = near(K, carried)
        slack = 1.7 * (off[:, :N] * (up.abs() + 1) + off[:, N:] * gate.abs()) + 32 * 2.0 ** -24 * (gate.abs() + 1) * (up.abs() + 1)
        got = o.linear_silu_mul_f8(X, W, activation=activation, limit=limit)
        bound = half_step(want) * (1 + 2.0 ** -16) + 1.1 * slack + flat(blocks(slack, 1).amax(dim=3, keepdim=True).expand(-1, -1, -1, 128), T, N) * 2.0 ** -4
        assert bool(((got.values(F32).to(F64) - want).abs() <= bound).all()), T
        if N % 128:
            assert got.codes[-1, :T, N % 128:].count_nonzero() == 0
        again = o.linear_silu_mul_f8(x, W, activation=activation, limit=limit)
        assert torch.equal(again.codes[:, :T], got.codes[:, :T]) and torch.equal(again.scales[:T, :(N + 127) // 128], got.scales[:T, :(N + 127) // 128])
    assert o.stream_status(torch.device(DEV)).tolist() == [0, 0]


def experts_in_64_bits(x, gu, dn, ids, weights, act, limit, on_input, base):
    """(the result, a bound of what another rounding of a code may make of it, what the sums carry, the picks' rows added up as magnitudes)."""
    T, W = x.shape
    E, ff = dn.shape[0], dn.shape[2]
    out, steps, carried, rows = (torch.zeros(T, W, dtype=F64, device=DEV) for _ in range(4))
    if base is not None:
        out += base.to(F64)
        carried += base.to(F64).abs()
    v = held(x.to(F32), 1).to(F64)
    for e in range(E):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        if not len(token):
            continue
        wt = weights[token, choice, None].to(F64)
        y = (v[token] @ gu[e].to(F64).T) * (wt if on_input else 1)
        a = middle(y[:, :ff], y[:, ff:], act, limit)
        r = held(a.to(F32), 1).to(F64)
        down = dn[e].to(F64)
        f = 1 if on_input else wt
        out.index_add_(0, token, f * (r @ down.T))
        steps.index_add_(0, token, (f * (2 * half_step(a) @ down.abs().T)).abs())
        rows.index_add_(0, token, (f * (r @ down.T)).abs())
        carried.index_add_(0, token, (f * (r.abs() @ down.abs().T)).abs())
    return out, steps, carried, rows


EXPERTS = [(1, 8, 2, 1, 32), (1, 64, 8, 64, 128), (3, 4, 2, 100, 200), (17, 8, 2, 192, 520), (48, 64, 8, 128, 256), (70, 6, 3, 150, 136), (130, 3, 1, 700, 392),
           (200, 16, 4, 130, 300), (301, 8, 2, 1450, 1358), (600, 5, 5, 256, 640), (1100, 40, 6, 96, 264), (2000, 2, 1, 257, 512)]


@pytest.mark.parametrize("T,E,top,ff,W", EXPERTS)
@pytest.mark.parametrize("activation,limit,on_input", [("silu", 0.0, False), ("clamped_swish", 1.5, True)])
def test_experts(T, E, top, ff, W, activation, limit, on_input):
    o, g = ops(), gen(T + E + ff)
    gu, dn = normal(g, E, 2 * ff, W, dtype=BF16) * W ** -0.5, normal(g, E, W, ff, dtype=BF16) * ff ** -0.5
    x = normal(g, T, W, dtype=BF16)
    score, ids = torch.topk(normal(g, T, E) + normal(g, E), top, dim=1)
    ids, weights = ids.to(torch.int32), torch.softmax(score, dim=1)
    ids[torch.rand(T, top, generator=g, device=DEV) < 0.05] = -1  # picks without an expert
    G, D = o.f8_weight(gu, gated=True), o.f8_weight(dn)
    base = normal(g, T, W) if T % 2 else None
    want, steps, carried, rows = experts_in_64_bits(x, G.values(F32), D.values(F32), ids, weights, o.ACTIVATIONS[activation], limit, on_input, base)
    got = o.moe_f8(x, G, D, ids, weights, activation=activation, limit=limit, on_input=on_input, base=base)
    assert got.dtype == F32 and bool(((got.to(F64) - want).abs() <= steps + (near(ff, carried) + 2.0 ** -20 * carried)).all())
    # A code comes out a step off, 2^-3 at most, where its value is within 2^-18 of one of the 16 borders of an octave: one in 2^14 at most, or one
    # of these few if they are fewer; times sqrt of that share.  A row counts for itself, its picks not having one direction.
    share = max(2.0 ** -14, 1.0 / (T * top * ff))
    assert float((got.to(F64) - want).norm()) <= 2 * 2.0 ** -3 * share ** 0.5 * float((want if base is None else want - base.to(F64)).norm()) + 2.0 ** -20 * float(want.norm())
    again = o.moe_f8(x, G, D, ids, weights, activation=activation, limit=limit, on_input=on_input, base=base)
    assert torch.equal(again, got)                                # whatever order the rows were sorted in
    short = o.moe_f8(x, G, D, ids, weights, activation=activation, limit=limit, on_input=on_input, base=base, out_dtype=BF16)
    # each pick's row, and the sum, rounded to bfloat16: 2^-8 of it each; a row may be off by what it is made of
    assert bool(((short.to(F64) - got.to(F64)).abs() <= 2.0 ** -8 * 1.01 * (rows + steps + got.to(F64).abs())).all())
    wide = o.moe_f8(x.float(), G, D, ids, weights, activation=activation, limit=limit, on_input=on_input, base=base)
    assert torch.equal(wide, got)                                 # the same rows, made by a kernel of their own
    assert o.stream_status(torch.device(DEV)).tolist() == [0, 0]


def test_experts_nobody_picks_and_one_that_all_pick():
    o, g = ops(), gen(5)
    E, ff, W = 7, 136, 264
    G, D = o.f8_weight(normal(g, E, 2 * ff, W), gated=True), o.f8_weight(normal(g, E, W, ff))
    for T in (1, 20, 40, 120, 700):
        x, weights = normal(g, T, W, dtype=BF16), torch.rand(T, 1, generator=g, device=DEV)
        for e in (0, 6):
            ids = torch.full((T, 1), e, dtype=torch.int32, device=DEV)
            want, steps, carried, _ = experts_in_64_bits(x, G.values(F32), D.values(F32), ids, weights, 0, 0.0, False, None)
            got = o.moe_f8(x, G, D, ids, weights)
            assert bool(((got.to(F64) - want).abs() <= steps + near(ff, carried) + 2.0 ** -20 * carried).all()), (T, e)
        base = normal(g, T, W)
        none = torch.full((T, 1), -1, dtype=torch.int32, device=DEV)
        none[T // 2] = E
        assert torch.equal(o.moe_f8(x, G, D, none, weights, base=base), base)
        assert o.moe_f8(x, G, D, none, weights).count_nonzero() == 0
    assert o.moe_f8(x[:0], G, D, ids[:0], weights[:0]).shape == (0, W)
    assert o.linear_f8(x[:0], o.f8_weight(normal(g, 5, W))).shape == (0, 5)


def test_a_row_that_is_not_finite_stays_alone():
    o, g = ops(), gen(6)
    W = o.f8_weight(normal(g, 300, 400))
    for T in (5, 40, 300):
        x = normal(g, T, 400, dtype=BF16)
        clean = o.linear_f8(x, W)
        x[3, 7], x[1, 399] = float("nan"), float("inf")
        got = o.linear_f8(x, W)
        others = [r for r in range(T) if r not in (1, 3)]
        assert got[[1, 3]].isnan().all() and torch.equal(got[others], clean[others])


def test_refusals():
    o, g = ops(), gen(7)
    w, x = normal(g, 64, 96), normal(g, 4, 96, dtype=BF16)
    W, G = o.f8_weight(w), o.f8_weight(w, gated=True)
    S, SG = o.f8_weight(normal(g, 3, 96, 32)), o.f8_weight(normal(g, 3, 64, 96), gated=True)
    ids, weights = torch.zeros(4, 2, dtype=torch.int32, device=DEV), torch.ones(4, 2, device=DEV)
    for call in (lambda: o.f8_weight(w.half()), lambda: o.f8_weight(w[:63], gated=True), lambda: o.f8_weight(w.t()), lambda: o.f8_weight(w.cpu()), lambda: o.f8_weight(w[:0]),
                 lambda: o.f8_rows(x.half()), lambda: o.f8_rows(x[0]), lambda: o.f8_rows(x.t()), lambda: o.f8_rows(x.cpu()),
                 lambda: o.linear_f8(x[:, :95].contiguous(), W), lambda: o.linear_f8(x, G), lambda: o.linear_f8(x, w), lambda: o.linear_f8(x, S), lambda: o.linear_f8(x.half(), W),
                 lambda: o.linear_f8(x, W, torch.float16), lambda: o.linear_f8(x, W, residual=normal(g, 4, 63)), lambda: o.linear_f8(x, W, residual=normal(g, 4, 64, dtype=BF16)),
                 lambda: o.linear_f8(x.cpu(), W), lambda: o.linear_f8(None, W), lambda: o.linear_silu_mul_f8(x, W),
                 lambda: o.moe_f8(x, S, S, ids, weights), lambda: o.moe_f8(x, SG, SG, ids, weights), lambda: o.moe_f8(x, G, S, ids, weights),
                 lambda: o.moe_f8(x, SG, S, ids.long(), weights), lambda: o.moe_f8(x, SG, S, ids[:3], weights), lambda: o.moe_f8(x, SG, S, ids, weights.double()),
                 lambda: o.moe_f8(x, SG, S, ids, weights[:, :1]), lambda: o.moe_f8(x, SG, S, ids, weights, base=normal(g, 4, 95)), lambda: o.moe_f8(x[:, :64].contiguous(), SG, S, ids, weights),
                 lambda: o.moe_f8(x, SG, S, ids, weights, out_dtype=torch.float16), lambda: o.moe_f8(x, SG, o.f8_weight(normal(g, 3, 96, 40)), ids, weights)):
        with pytest.raises(o.KernelError):
            call()
    assert torch.isfinite(o.moe_f8(x, SG, S, ids, weights)).all()
