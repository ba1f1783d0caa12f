"""Microscaled rows, weights and products against their definition in 64 bits: blocks of 32, the smallest power of two as scale with
which the largest magnitude fits the format, codes to the nearest (ties to even)."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64, F32, BF16 = torch.float64, torch.float32, torch.bfloat16
TOP = {4: 6.0, 8: 448.0}
BITS, LEAST = {4: 1, 8: 3}, {4: 0, 8: -6}


def ops():
    from litellmengine_b200.csrc import ops as o
    return o


def scales(x, fmt):
    """float64 [rows, k] -> the scale of every value, NaN where the block holds something that is not finite."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % 32)).view(rows, -1, 32)
    most = b.abs().amax(-1)
    e = torch.floor(torch.log2(torch.where((most > 0) & most.isfinite(), most, 1.0) / TOP[fmt])) - 1
    for _ in range(3):                                            # the smallest exponent that is large enough
        e = torch.where(torch.exp2(e) * TOP[fmt] < most, e + 1, e)
    s = torch.exp2(torch.where(most > 0, e, -127.0).clamp(min=-127))
    s = torch.where(b.isfinite().all(-1), s, float("nan"))
    return s.repeat_interleave(32, dim=1)[:, :k]


def held(x, fmt):
    x = x.to(F64)
    s = scales(x, fmt)
    q = x / s
    step = torch.exp2(torch.floor(torch.log2(torch.where(q == 0, 1.0, q.abs()))).clamp(min=LEAST[fmt]) - BITS[fmt])
    return torch.round(q / step) * step * s                       # torch.round: ties to even


def same(got, want):
    want = want.to(got.dtype)                                     # exact, but for what reaches 2^128: the largest float32 rounds to that
    return torch.equal(got.to(F64).nan_to_num(1e300), want.to(F64).nan_to_num(1e300)) and torch.equal(got.isnan(), want.isnan())


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("rows,k", [(1, 1), (1, 31), (3, 33), (2, 127), (129, 128), (5, 1000), (64, 136), (300, 2056), (1, 4096)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_codes_are_the_nearest(rows, k, dtype):
    o, g = ops(), gen(rows * 7 + k)
    x = normal(g, rows, k, dtype=dtype) * torch.exp2(torch.randint(-8, 8, (rows, k), generator=g, device=DEV)).to(dtype)
    assert same(o.mx_rows(x).values(F32), held(x, 8))
    assert same(o.mx_weight(x).values(F32), held(x, 4))
    assert same(o.mx_rows(x).values(BF16), held(x, 8)) and same(o.mx_weight(x).values(BF16), held(x, 4))      # bfloat16 holds every value
    two = torch.cat([x, -x])
    w = o.mx_weight(two, gated=True)
    assert w.shape == (2 * rows, k) and same(w.values(F32), held(two, 4))
    unaligned = torch.empty(rows * k + 1, dtype=dtype, device=DEV)[1:].view(rows, k).copy_(x)
    assert same(o.mx_rows(unaligned).values(F32), held(x, 8)) and same(o.mx_weight(unaligned).values(F32), held(x, 4))


@pytest.mark.parametrize("fmt", [4, 8])
def test_borders(fmt):
    """Ties of every pair of neighbours, largest magnitudes at and just above what a scale takes, zeros of both signs, the
    smallest and largest float32, and blocks with something that is not finite beside blocks without."""
    o = ops()
    grid = [m * 2.0 ** (LEAST[fmt] - BITS[fmt]) for m in range(2 ** BITS[fmt])]
    e = LEAST[fmt]
    while 2.0 ** e <= TOP[fmt]:
        grid += [v for m in range(2 ** BITS[fmt]) if (v := (1 + m / 2 ** BITS[fmt]) * 2.0 ** e) <= TOP[fmt]]
        e += 1
    ties = [(a + b) / 2 for a, b in zip(grid, grid[1:])]
    near = [t * (1 + d) for t in ties for d in (2.0 ** -20, -2.0 ** -20)]
    blocks = []
    for values in (grid, ties, near):
        for at in range(0, len(values), 31):
            v = values[at:at + 31]
            blocks.append([TOP[fmt]] + v + [0.0] * (31 - len(v)))
    up = lambda v: torch.nextafter(torch.tensor(v), torch.tensor(3e38)).item()
    for s in (2.0 ** -100, 2.0 ** -3, 1.0, 2.0 ** 60):
        blocks += [[TOP[fmt] * s, s] + [0.0] * 30, [up(TOP[fmt] * s), -s] + [0.5 * s] * 30]
    big, tiny, nan, inf = 3.4028234663852886e38, 1.4e-45, float("nan"), float("inf")
    blocks += [[0.0] * 16 + [-0.0] * 16, [tiny] * 32, [1e-40, -3e-39] * 16, [big, -big, 1.0, 0.0] * 8, [nan] + [1.0] * 31, [1.0] * 32,
               [1.0] * 31 + [-inf], [inf, nan] * 16, [2.0] * 32]
    x = torch.tensor(blocks, device=DEV)
    x = torch.cat([x, -x, torch.flip(x, (1,))]).view(3 * len(blocks), 32)
    make = o.mx_rows if fmt == 8 else o.mx_weight
    assert same(make(x).values(F32), held(x, fmt))
    wide = x[:len(blocks)].reshape(1, -1)                         # the same blocks side by side: each its own scale
    assert same(make(wide).values(F32), held(wide, fmt))


def test_offsets_beyond_32_bits():
    o = ops()
    T, K = 33000, 66000                                           # 2.2e9 values
    x = torch.zeros(T, K, dtype=BF16, device=DEV)
    g = gen(3)
    ends = [0, 127, 128, T // 2, T - 2, T - 1]
    for r in ends:
        x[r] = normal(g, K, dtype=BF16)
    made = o.mx_rows(x)
    want = held(x[ends], 8)
    assert same(made.values(BF16)[ends], want)
    w = o.mx_weight(x)
    del made
    assert same(w.values(BF16)[ends], held(x[ends], 4))


def half_step(n, fmt=8):
    """What rounding moves n by at most: 2^-4 of it, or half the smallest step of its block; a scale may be the next one where the
    largest magnitude lies within 2^-18 of a border, which doubles that."""
    s = scales(n, fmt)
    s = torch.where(scales(n * (1 + 2.0 ** -18), fmt) > s, 2 * s, s)
    return torch.maximum(n.abs() * 2.0 ** -4, s * 2.0 ** -10)


@pytest.mark.parametrize("T,H", [(1, 4096), (3, 1), (2, 33), (130, 200), (257, 1450), (5, 8192), (2, 8200), (3, 20000), (1, 32768), (1024, 8), (1100, 1032),
                                 (3000, 2048), (1333, 4096), (1025, 8192), (1030, 1450),
                                 (639, 512), (640, 512), (700, 8192), (641, 264)])
@pytest.mark.parametrize("pending", ["none", "float32", "bfloat16", "parts"])
def test_norm(T, H, pending):
    o, g = ops(), gen(T + H)
    x, w = normal(g, T, H) * 3, 1 + 0.1 * normal(g, H)
    delta, total = None, x.clone()
    if pending == "parts":
        parts = normal(g, 3, T, H)
        delta = o.PartialSum(parts)
        for p in parts:
            total = total + p
    elif pending != "none":
        delta = normal(g, T, H).to(getattr(torch, pending))
        total = x + delta.float()
    # the stream is rounded after each addition; the norm is of what the sum is before that
    v = x.to(F64) + (0 if delta is None else delta.parts.to(F64).sum(0) if pending == "parts" else delta.to(F64))
    n = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w.to(F64)
    # less than 32 roundings of 2^-24 in all
    near = half_step(n) + n.abs() * 32 * 2.0 ** -24
    out = torch.empty_like(x)
    before = x.clone()
    got = o.rmsnorm_mx(x, w, 1e-6, delta=delta, sum_out=out)
    assert torch.equal(out, total) and torch.equal(x, before)
    assert bool(((got.values(F32).to(F64) - n).abs() <= near).all())
    assert got.codes[:, H:].count_nonzero() == 0
    again = o.rmsnorm_mx(x, w, 1e-6, delta=delta, sum_out=x)      # in place
    assert torch.equal(x, total) and torch.equal(again.values(F32), got.values(F32))
    if pending in ("float32", "bfloat16") and T < 1000:
        cut = o.rmsnorm_mx(before[:3].contiguous(), w, 1e-6, delta=delta[:3].contiguous()).values(F32)
        assert torch.equal(cut, got.values(F32)[:3])              # no row depends on the others
    rows = torch.tensor([T - 1, 0, T // 2, T // 2], dtype=torch.int32, device=DEV)
    picked = o.rmsnorm_mx(total, w, 1e-6, rows=rows).values(F32)
    assert T > 1000 or torch.equal(picked, o.rmsnorm_mx(total, w, 1e-6).values(F32)[rows.long()])
    n = total.to(F64)[rows.long()]
    n = n * torch.rsqrt(n.square().mean(-1, keepdim=True) + 1e-6) * w.to(F64)
    assert bool(((picked.to(F64) - n).abs() <= half_step(n) + n.abs() * 32 * 2.0 ** -24).all())


def test_norm_of_16_bits_and_of_rows_that_are_not_finite():
    o, g = ops(), gen(8)
    x, w = normal(g, 9, 520, dtype=BF16), torch.ones(520, device=DEV)
    n = x.to(F64) * torch.rsqrt(x.to(F64).square().mean(-1, keepdim=True) + 1e-5)
    out = torch.empty_like(x)
    got = o.rmsnorm_mx(x, w, 1e-5, delta=torch.zeros_like(x), sum_out=out).values(F32).to(F64)
    assert torch.equal(out, x) and bool(((got - n).abs() <= half_step(n) + n.abs() * 32 * 2.0 ** -24).all())
    x[2, 5] = float("nan")
    x[4] = 0
    got = o.rmsnorm_mx(x, w, 1e-5).values(F32)
    assert got[2].isnan().all() and got[4].count_nonzero() == 0 and got[[0, 1, 3, 5, 6, 7, 8]].isfinite().all()


def middle(gate, up, act, limit):
    if act == 2:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        return gate * torch.sigmoid(1.702 * gate) * (up + 1)
    return (torch.nn.functional.gelu(gate, approximate="tanh") if act == 1 else gate * torch.sigmoid(gate)) * up


@pytest.mark.parametrize("T,inter", [(1, 1), (1, 4096), (3, 33), (130, 200), (257, 1450), (40, 12288)])
@pytest.mark.parametrize("activation,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("clamped_swish", 1.5)])
def test_act(T, inter, activation, limit):
    o, g = ops(), gen(T + inter)
    act = o.ACTIVATIONS[activation]
    for given in (normal(g, T, 2 * inter), normal(g, T, 2 * inter, dtype=BF16), o.PartialSum(normal(g, 3, T, 2 * inter))):
        gu = given.parts.to(F64).sum(0) if isinstance(given, o.PartialSum) else given.to(F64)
        want = middle(gu[:, :inter], gu[:, inter:], act, limit)
        # exp, tanh and the products: less than 32 roundings of 2^-24 of the two factors (a tanh near -1 cancels: of the gate
        # itself), and 4 of each sum of parts, which moves the result by up to 1.2 times the other factor
        slack = 32 * 2.0 ** -24 * (gu[:, :inter].abs() + 1) * (gu[:, inter:].abs() + 1)
        got = o.silu_and_mul_mx(given, activation=activation, limit=limit)
        bound = torch.maximum(half_step(want), half_step(want.abs() + slack)) + slack
        assert bool(((got.values(F32).to(F64) - want).abs() <= bound).all())
        assert got.codes[:, inter:].count_nonzero() == 0


ROWS = (1, 7, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 300)


def carried(a, b):
    return a.to(F64).abs() @ b.to(F64).abs().T


@pytest.mark.parametrize("N,K", [(1, 1), (16, 32), (100, 200), (129, 128), (127, 1024), (1000, 1358), (640, 4104), (4096, 640), (6144, 4096), (2500, 12288)])
def test_product(N, K):
    o, g = ops(), gen(N + K)
    W = o.mx_weight(normal(g, N, K) * K ** -0.5)
    w = W.values(F32)
    for T in ROWS:
        x = normal(g, T, K, dtype=BF16) * (1 + 11 * (torch.rand(K, generator=g, device=DEV) < 0.01)).to(BF16)
        X = o.mx_rows(x)
        v = X.values(F32)
        got = o.linear_mx(X, W)
        # K / 32 steps of products that are exact in float32 and at most 8 parts, each sum cut or rounded at 2^-23 of what it holds
        near = (K / 32 + 24) * 2.0 ** -23 * carried(v, w)
        assert bool(((got.to(F64) - v.to(F64) @ w.to(F64).T).abs() <= near).all()), T
        assert torch.equal(o.linear_mx(x, W), got)                # the call takes the rows to 8 bits by itself, and gives the same again
        assert torch.equal(o.linear_mx(X, W, BF16), got.to(BF16))
        stream = normal(g, T, N)
        total = stream + got
        assert o.linear_mx(X, W, residual=stream) is stream and torch.equal(stream, total)
    assert o.stream_status(torch.device(DEV)).tolist() == [0, 0]


@pytest.mark.parametrize("N,K", [(1, 32), (64, 128), (100, 200), (192, 520), (700, 1358), (4096, 640), (12288, 512), (1450, 4096)])
@pytest.mark.parametrize("activation,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("clamped_swish", 1.5)])
def test_gated_product(N, K, activation, limit):
    o, g = ops(), gen(N + K)
    act = o.ACTIVATIONS[activation]
    plain = normal(g, 2 * N, K) * K ** -0.5
    W = o.mx_weight(plain, gated=True)
    w = W.values(F32)
    assert torch.equal(w, o.mx_weight(plain).values(F32))
    for T in ROWS:
        x = normal(g, T, K, dtype=BF16)
        X = o.mx_rows(x)
        v = X.values(F32)
        sums, off = v.to(F64) @ w.to(F64).T, (K / 32 + 24) * 2.0 ** -23 * carried(v, w)
        gate, up = sums[:, :N], sums[:, N:]
        want = middle(gate, up, act, limit)
        # as in test_act, and what the sums are off moves the result by at most 1.2 times the other factor
        slack = (32 * 2.0 ** -24 * (gate.abs() + 1) * (up.abs() + 1) + 1.2 * off[:, :N] * (up.abs() + 1) + 1.2 * off[:, N:] * (gate.abs() + 1))
        got = o.linear_silu_mul_mx(X, W, activation=activation, limit=limit)
        bound = torch.maximum(half_step(want), half_step(want.abs() + slack)) + slack
        assert bool(((got.values(F32).to(F64) - want).abs() <= bound).all()), T
        assert got.codes[:, N:].count_nonzero() == 0
        assert torch.equal(o.linear_silu_mul_mx(x, W, activation=activation, limit=limit).values(F32), got.values(F32))
    assert o.stream_status(torch.device(DEV)).tolist() == [0, 0]


def way(T, N, K, gated=False):
    o = ops()
    f = o._fn("microscaling", "llm_linear_mx_way", [o.c_int] * 5)
    return f(T, N, K, int(gated), torch.cuda.get_device_properties(0).multi_processor_count)


@pytest.mark.parametrize("T,N,K,tokens", [(2000, 2501, 1358, 192), (6013, 1003, 264, 192), (1500, 3000, 130, 128), (1201, 4104, 257, 192), (800, 4000, 2000, 128), (500, 4096, 1032, 128),
                                          (256, 12288, 520, 128), (90, 20000, 1358, 128), (130, 20000, 4104, 192), (577, 4096, 4096, 192)])
@pytest.mark.parametrize("gated", [False, True])
def test_pairs(T, N, K, tokens, gated):
    """Tiles of pairs of CTAs of every width, with ragged rows, features and K, rows whose scales begin in every word of a piece."""
    o, g = ops(), gen(T + N + K)
    n = N // 2 if gated else N
    W = o.mx_weight(normal(g, 2 * n if gated else n, K) * K ** -0.5, gated=gated)
    w = W.values(F32)
    x = normal(g, T, K) * torch.exp2(torch.randint(-3, 4, (T, 1), generator=g, device=DEV).float())      # every row its own scales
    X = o.mx_rows(x)
    v = X.values(F32)
    assert gated or way(T, n, K) == tokens
    sums, off = v.to(F64) @ w.to(F64).T, (K / 32 + 24) * 2.0 ** -23 * carried(v, w)
    if gated:
        gate, up = sums[:, :n], sums[:, n:]
        want = middle(gate, up, 0, 0)
        slack = (32 * 2.0 ** -24 * (gate.abs() + 1) * (up.abs() + 1) + 1.2 * off[:, :n] * (up.abs() + 1) + 1.2 * off[:, n:] * (gate.abs() + 1))
        got = o.linear_silu_mul_mx(X, W)
        assert bool(((got.values(F32).to(F64) - want).abs() <= torch.maximum(half_step(want), half_step(want.abs() + slack)) + slack).all())
        return
    got = o.linear_mx(X, W)
    assert bool(((got.to(F64) - sums).abs() <= off).all())
    assert torch.equal(o.linear_mx(X, W, BF16), got.to(BF16))
    stream = normal(g, T, n)
    total = stream + got
    assert torch.equal(o.linear_mx(X, W, residual=stream), total)
    room = torch.full((T + 2, n), 7.0, device=DEV)                # nothing beyond the result's rows is written
    room[1:-1].zero_()
    o.linear_mx(X, W, residual=room[1:-1])
    assert torch.equal(room[1:-1], got) and bool((room[0] == 7).all()) and bool((room[-1] == 7).all())


def test_scales_that_are_far_apart():
    """Blocks whose scales differ by up to 2^60 in one row: every product's scale is its own."""
    o, g = ops(), gen(5)
    x = normal(g, 20, 512) * torch.exp2(torch.randint(-30, 30, (20, 16), generator=g, device=DEV).float()).repeat_interleave(32, 1)
    w = normal(g, 300, 512) * torch.exp2(torch.randint(-30, 30, (300, 16), generator=g, device=DEV).float()).repeat_interleave(32, 1)
    X, W = o.mx_rows(x), o.mx_weight(w)
    v, u = X.values(F32), W.values(F32)
    got = o.linear_mx(X, W)
    assert bool(((got.to(F64) - v.to(F64) @ u.to(F64).T).abs() <= (512 / 32 + 24) * 2.0 ** -23 * carried(v, u)).all())


def test_rows_that_are_not_finite_stay_by_themselves():
    o, g = ops(), gen(6)
    W = o.mx_weight(normal(g, 200, 300))
    for T in (5, 200):
        x = normal(g, T, 300)
        want = o.linear_mx(x, W)
        x[3, 40] = float("inf")
        got = o.linear_mx(x, W)
        assert got[3].isnan().all() and torch.equal(got[:3], want[:3]) and torch.equal(got[4:], want[4:])
    w = normal(g, 200, 300)
    w[7, 299] = float("nan")                                      # in the block that ends inside a tile
    got = o.linear_mx(x[:3].contiguous(), o.mx_weight(w))
    assert got[:, 7].isnan().all() and got[:, :7].isfinite().all() and got[:, 8:].isfinite().all()


def feed_forward(o, h, delta, norm_w, gate_up, down, out):
    rows = o.rmsnorm_mx(h, norm_w, 1e-6, delta=delta, sum_out=out)
    return o.linear_mx(o.linear_silu_mul_mx(rows, gate_up), down, residual=out)


@pytest.mark.parametrize("T", [1, 24, 150, 600])
def test_a_feed_forward_of_them_captured_and_replayed(T):
    """Norm, gate and up, down and the residual's addition as a layer runs them: against 64 bits, on another stream, and as a graph
    replayed on new inputs beside eager calls."""
    o, g = ops(), gen(T)
    H, inter = 320, 712
    gate_up, down = o.mx_weight(normal(g, 2 * inter, H) * H ** -0.5, gated=True), o.mx_weight(normal(g, H, inter) * inter ** -0.5)
    norm_w = 1 + 0.1 * normal(g, H)
    h, delta, out = normal(g, T, H), normal(g, T, H), torch.empty(T, H, device=DEV)

    def reference():
        v = h.to(F64) + delta.to(F64)
        n = held((v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * norm_w.to(F64)), 8)
        s = n @ gate_up.values(F32).to(F64).T
        return v, held(middle(s[:, :inter], s[:, inter:], 0, 0), 8) @ down.values(F32).to(F64).T

    def check(got):
        v, y = reference()
        # codes that fall to the other side of a border are off by a whole step, 2^-3, instead of being right: fewer than one in
        # a hundred here (float32 sums are 2^-20 off, steps are 2^-3 apart), so the norm of the difference is below 2^-3 / 10 of y's
        assert float((got.to(F64) - v - y).norm() / y.norm()) < 2.0 ** -3 / 10
    eager = feed_forward(o, h, delta, norm_w, gate_up, down, out).clone()
    check(eager)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = torch.empty_like(out)
        feed_forward(o, h, delta, norm_w, gate_up, down, other)
    again = feed_forward(o, h, delta, norm_w, gate_up, down, out).clone()        # both streams at once
    torch.cuda.synchronize()
    assert torch.equal(other, eager) and torch.equal(again, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        feed_forward(o, h, delta, norm_w, gate_up, down, out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    h.copy_(normal(g, T, H))
    delta.copy_(normal(g, T, H))
    graph.replay()
    torch.cuda.synchronize()
    got = out.clone()
    check(got)
    assert torch.equal(feed_forward(o, h, delta, norm_w, gate_up, down, torch.empty_like(out)), got)


@pytest.mark.parametrize("T,N,K,gated", [(4, 4096, 4096, False), (100, 256, 2048, False), (300, 512, 4096, False), (4, 512, 2048, True),
                                         (2000, 4096, 1024, False), (700, 4001, 1024, False), (2000, 4096, 640, True)])
def test_a_wait_that_runs_out(T, N, K, gated):
    """Waits without tries: the status is set, the copies land before the blocks end, and the next products are right."""
    o, g = ops(), gen(9)
    W = o.mx_weight(normal(g, 2 * N if gated else N, K), gated=gated)
    X = o.mx_rows(normal(g, T, K))
    run = (lambda **k: o.linear_silu_mul_mx(X, W, **k).values(F32)) if gated else (lambda **k: o.linear_mx(X, W, **k))
    status = o.stream_status(torch.device(DEV))
    try:
        want = run()
        assert status.tolist() == [0, 0]
        run(waits=0)
        assert status.tolist()[0] == 9
        status.zero_()
        for _ in range(3):
            assert torch.equal(run(), want)
        assert status.tolist() == [0, 0]
    finally:
        status.zero_()


def test_refusals():
    o = ops()
    x, w = torch.zeros(4, 64, device=DEV), torch.zeros(128, 64, device=DEV)
    W, G, X, n = o.mx_weight(w), o.mx_weight(w, gated=True), o.mx_rows(x), torch.ones(64, device=DEV)

    def refuses(call, *a, **k):
        with pytest.raises(o.KernelError):
            call(*a, **k)
    refuses(o.linear_mx, X, G)                                    # a gated weight where a plain one is wanted, and the other way round
    refuses(o.linear_silu_mul_mx, X, W)
    refuses(o.linear_mx, X, w)
    refuses(o.linear_mx, o.mx_rows(x[:, :32].contiguous()), W)
    refuses(o.linear_mx, X, W, torch.float16)
    refuses(o.linear_mx, X, W, residual=torch.zeros(4, 128, dtype=BF16, device=DEV))
    refuses(o.linear_mx, X, W, residual=torch.zeros(4, 127, device=DEV))
    refuses(o.linear_mx, X, W, residual=torch.zeros(128, 4, device=DEV).t())
    refuses(o.linear_silu_mul_mx, X, G, activation="clamped_swish")
    refuses(o.mx_rows, x.half())
    refuses(o.mx_rows, x.t())
    refuses(o.mx_rows, x[0])
    refuses(o.mx_weight, w[:127].contiguous(), gated=True)
    refuses(o.mx_weight, w[:0])
    refuses(o.rmsnorm_mx, x, n[:63], 1e-6)
    refuses(o.rmsnorm_mx, x, n.to(BF16), 1e-6)
    refuses(o.rmsnorm_mx, x, n, 1e-6, delta=x[:3])
    refuses(o.rmsnorm_mx, x, n, 1e-6, sum_out=torch.empty_like(x, dtype=BF16))
    refuses(o.rmsnorm_mx, x, n, 1e-6, rows=torch.zeros(2, dtype=torch.int32, device=DEV), sum_out=x)
    refuses(o.rmsnorm_mx, x, n, 1e-6, rows=torch.zeros(2, dtype=torch.int64, device=DEV))
    refuses(o.rmsnorm_mx, torch.zeros(1, 32769, device=DEV), torch.ones(32769, device=DEV), 1e-6)
    refuses(o.silu_and_mul_mx, x[:, :63].contiguous())
    refuses(X.values, torch.float16)
    refuses(o.linear_mx, o.PartialSum(x[None]), W)
    refuses(o.linear, o.PendingRows(x, None, n, 1e-6, BF16), W)
    refuses(o.linear_silu_mul, o.PendingRows(x, None, n, 1e-6, BF16), G, BF16)
    assert o.linear_mx(o.mx_rows(x[:0]), W).shape == (0, 128) and o.linear_silu_mul_mx(x[:0], G).values().shape == (0, 64)
    assert W.nbytes == G.nbytes == 2 * (128 * 64 + 512)


def test_what_a_product_of_the_general_entry_comes_in():
    o, g = ops(), gen(12)
    x, W = normal(g, 3, 256), o.mx_weight(normal(g, 200, 256))
    want = o.linear_mx(x, W)
    for given, dtype, out in ((x, None, F32), (x, BF16, BF16), (x.to(BF16), None, BF16), (x.to(BF16), F32, F32), (o.mx_rows(x), None, BF16), (o.mx_rows(x), F32, F32)):
        got = o.linear(given, W, out_dtype=dtype)
        assert got.dtype == out
        if given.shape[0] and (isinstance(given, o.MxRows) or given.dtype == F32):
            assert torch.equal(got, want.to(out))


def test_a_copy_of_a_weight_is_a_weight_of_its_own():
    o, g = ops(), gen(13)
    x = normal(g, 5, 300)
    for gated in (False, True):
        W = o.mx_weight(normal(g, 260, 300), gated=gated)
        run = (lambda w: o.linear_silu_mul_mx(x, w).values(F32)) if gated else (lambda w: o.linear_mx(x, w))
        want, values = run(W), W.values(F32)
        other = copy.deepcopy(W)
        W.buffer.zero_()
        assert torch.equal(run(other), want) and torch.equal(other.values(F32), values) and bool((W.values(F32) == 0).all())


@pytest.mark.parametrize("T,H", [(5, 4096), (5, 520), (700, 2048)])
@pytest.mark.parametrize("pending", [False, True])
def test_norms_at_borders_between_codes(T, H, pending):
    """Rows whose normed values lie on, and one or two places beside, the borders between two codes or two scales, and in the lowest
    range: a float32 product falls to either side of them, the sums of 64 bits say to which."""
    o, g = ops(), gen(T + H)
    # a row's largest value, 7, is its blocks' scale; the rest are ties of e4m3 at that scale moved by up to two places
    ties = torch.tensor([(8 + m + 0.5) / 8 * 2.0 ** e for m in range(8) for e in range(-14, 2)] + [(m + 0.5) * 2.0 ** -15 for m in range(8)], device=DEV)
    x = ties[torch.randint(len(ties), (T, H), generator=g, device=DEV)]
    x = x * torch.where(torch.rand(T, H, generator=g, device=DEV) < 0.5, 1.0, -1.0)
    x = (x.view(torch.int32) + torch.randint(-2, 3, (T, H), generator=g, device=DEV, dtype=torch.int32)).view(F32)
    x[:, ::32] = 7.0
    # the mean of squares is made a power of four, so that the borders stay where they are, as near as one value more can do it
    want, last = 16.0, x[:, 1:].to(F64).square().sum(-1)
    rest = want * H - last
    x[:, 0] = torch.where(rest > 0, rest.clamp(min=0).sqrt(), 7.0).float()
    w = torch.ones(H, device=DEV)
    delta = None
    if pending:
        delta = normal(g, T, H)
        x = x - delta                                             # rounded: the sum of both is near the border, and its remainder says where
    v = x.to(F64) + (0 if delta is None else delta.to(F64))
    n = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-12) * w.to(F64)
    got = o.rmsnorm_mx(x, w, 1e-12, delta=delta).values(F32).to(F64)
    # half a step of each value, and what a sum of squares in float32 leaves: fewer than 32 roundings of 2^-24
    assert bool(((got - n).abs() <= half_step(n) + n.abs() * 32 * 2.0 ** -24).all())
    # and hardly any code differs from the rounded exact value: those within 2^-22 of a border
    sure = (held(n * (1 + 2.0 ** -21), 8) == held(n * (1 - 2.0 ** -21), 8)) & (scales(n * (1 + 2.0 ** -21), 8) == scales(n * (1 - 2.0 ** -21), 8))
    assert torch.equal(got[sure], held(n, 8)[sure])
