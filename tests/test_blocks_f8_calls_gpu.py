"""Products of 8 bits as callers use them: in captured graphs, on streams of their own, from stacks that lie apart, with tokens that pick an expert twice, and
with bounded waits that run out."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64, F32, BF16 = torch.float64, torch.float32, torch.bfloat16


def ops():
    from litellmengine_b200.csrc import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


#: one token of eight picks, a batch whose rows the products make, sorted rows of every item, a sorting by several blocks
TOKENS = (1, 4, 5, 40, 100, 300, 600)


def feed_forward(o, x, W, D, S, SD, ids, weights):
    y = o.linear_f8(o.linear_silu_mul_f8(x, W), D)
    o.moe_f8(x, S, SD, ids, weights, base=y)
    return y + o.moe_f8(x, S, SD, ids, weights, base=y, out_dtype=BF16).float()


@pytest.mark.parametrize("T", TOKENS)
def test_captured_graphs_with_their_own_inputs(T):
    """Two graphs of the same weights, captured one after the other and replayed on two streams at once, with inputs that change between replays."""
    o, g = ops(), gen(T)
    E, top, ff, K = 16, 8, 264, 520
    W, D = o.f8_weight(normal(g, 2 * ff, K) * K ** -0.5, gated=True), o.f8_weight(normal(g, K, ff) * ff ** -0.5)
    S, SD = o.f8_weight(normal(g, E, 2 * ff, K) * K ** -0.5, gated=True), o.f8_weight(normal(g, E, K, ff) * ff ** -0.5)

    def inputs():
        score, ids = torch.topk(normal(g, T, E), top, dim=1)
        return normal(g, T, K, dtype=BF16), ids.to(torch.int32), torch.softmax(score, dim=1)
    held = [inputs(), inputs()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for (x, ids, weights), s in zip(held, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            feed_forward(o, x, W, D, S, SD, ids, weights)
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                outs.append(feed_forward(o, x, W, D, S, SD, ids, weights))
            graphs.append(graph)
    for _ in range(5):
        for mine in held:
            for a, b in zip(mine, inputs()):
                a.copy_(b)
        want = [feed_forward(o, x, W, D, S, SD, ids, weights) for x, ids, weights in held]
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    assert o.stream_status(torch.device(DEV)).tolist() == [0, 0]


def test_calls_in_a_row_on_one_stream():
    """Launches that begin before the one in front has ended: what each reads of the one in front is there."""
    o, g = ops(), gen(2)
    K = 1024
    W = [o.f8_weight(normal(g, K, K) * K ** -0.5) for _ in range(3)]
    for T in (3, 16, 20, 64, 130, 1500):
        x = normal(g, T, K, dtype=BF16)
        y = x
        for w in W * 8:
            y = o.linear_f8(y, w, BF16)
        z = x
        for w in W * 8:
            torch.cuda.synchronize()
            z = o.linear_f8(z, w, BF16)
        assert torch.equal(y, z), T


def test_stacks_that_lie_apart_and_copies():
    o, g = ops(), gen(3)
    room = normal(g, 5, 300, 264)
    stack = room[1::2, 8:264, 4:260]                              # matrices, rows and first values apart
    assert not stack.is_contiguous()
    S, want = o.f8_weight(stack), o.f8_weight(stack.contiguous())
    assert torch.equal(S.values(F32), want.values(F32)) and torch.equal(S.scales[..., :2], want.scales[..., :2])
    G = o.f8_weight(stack, gated=True)
    assert torch.equal(G.values(F32), want.values(F32))
    one = o.f8_weight(room[2, :, :200])
    x = normal(g, 9, 200, dtype=BF16)
    y = o.linear_f8(x, one)
    other = copy.deepcopy(one)
    assert other.buffer.data_ptr() != one.buffer.data_ptr() and torch.equal(o.linear_f8(x, other), y)
    other.buffer.zero_()
    assert o.linear_f8(x, other).count_nonzero() == 0 and torch.equal(o.linear_f8(x, one), y)


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 5), (130, 131), (257, 1358), (1003, 1357)])
def test_values_of_odd_sizes(rows, k):
    """Nothing beyond the matrix is written, wherever its rows begin."""
    o, g = ops(), gen(rows + k)
    w = o.f8_weight(normal(g, rows, k))
    for dtype in (F32, BF16):
        n = rows * k
        room = torch.full((n + 16,), 7.0, dtype=dtype, device=DEV)
        want = w.values(dtype)
        for first in (0, 1, 2, 8):
            room.fill_(7.0)
            out = room[first:first + n]
            o._check(o._mx_call("llm_f8_values")(w.buffer.data_ptr(), w.buffer.data_ptr() + w.scales_behind, out.data_ptr(), o._dt(out), rows, rows, k, w.tiles[0], 0, 1,
                                                 o._stream()), "values")
            assert torch.equal(out.view(rows, k), want)
            assert bool((room[:first] == 7).all()) and bool((room[first + n:] == 7).all())


@pytest.mark.parametrize("E,top,ff,W", [(4, 8, 2056, 4104), (1, 1, 64, 12288), (6, 3, 300, 136), (64, 8, 1024, 2048)])
def test_a_token_alone_gives_what_it_gives_among_others(E, top, ff, W):
    """Picks that stay as they are against the same picks sorted; an expert that is picked twice counts twice."""
    o, g = ops(), gen(E + ff)
    G, D = o.f8_weight(normal(g, E, 2 * ff, W, dtype=BF16) * W ** -0.5, gated=True), o.f8_weight(normal(g, E, W, ff, dtype=BF16) * ff ** -0.5)
    T = 6
    x, weights, base = normal(g, T, W, dtype=BF16), torch.rand(T, top, generator=g, device=DEV), normal(g, T, W)
    ids = torch.randint(-1, E + 1, (T, top), generator=g, device=DEV, dtype=torch.int32)
    ids[0] = 0
    for on_input in (False, True):
        whole = o.moe_f8(x, G, D, ids, weights, base=base, on_input=on_input)
        for n in (1, 2, 3, 4):
            for first in range(0, T - n + 1):
                part = slice(first, first + n)
                got = o.moe_f8(x[part], G, D, ids[part], weights[part], base=base[part], on_input=on_input)
                # K of the products is cut otherwise: the sums' order; a code may then be another, 2^-3 of a value of the middle
                assert float((got - whole[part]).abs().max()) <= 2.0 ** -6 * float((whole[part] - base[part]).abs().max()) + 2.0 ** -20 * float(whole.abs().max())
                assert torch.equal(got, o.moe_f8(x[part], G, D, ids[part], weights[part], base=base[part], on_input=on_input))


@pytest.mark.parametrize("T", [1, 5, 11, 20, 41, 50, 64, 65, 100, 130, 200, 300])
def test_one_expert_is_a_feed_forward(T):
    """A stack of one expert that every token picks with weight one, against the same matrices' products."""
    o, g = ops(), gen(T)
    ff, W = 264, 520
    up, down = normal(g, 2 * ff, W) * W ** -0.5, normal(g, W, ff) * ff ** -0.5
    x = normal(g, T, W, dtype=BF16)
    ids, weights = torch.zeros(T, 1, dtype=torch.int32, device=DEV), torch.ones(T, 1, device=DEV)
    got = o.moe_f8(x, o.f8_weight(up[None], gated=True), o.f8_weight(down[None]), ids, weights)
    want = o.linear_f8(o.linear_silu_mul_f8(x, o.f8_weight(up, gated=True)), o.f8_weight(down))
    # K may be cut otherwise: the sums' order; a code may then be another, 2^-3 of a value of the middle
    assert float((got - want).abs().max()) <= 2.0 ** -6 * float(want.abs().max())
    # one code in 2^14, or one of these few, a step off, twice its share of the norm
    assert float((got - want).norm()) <= 2 * 2.0 ** -3 * max(2.0 ** -14, 1.0 / (T * ff)) ** 0.5 * float(want.norm())


@pytest.mark.parametrize("T", [33, 64, 65, 100, 128, 300])
def test_rows_of_wide_weights(T):
    """Tiles of 128 rows by one CTA: more tiles of weights than there are SMs, results of any alignment and added ones; up features that lie in two blocks."""
    from test_blocks_f8_gpu import blocks, flat, half_step, middle, near, product
    o, g = ops(), gen(T + 7)
    for N, K in ((19201, 200), (20480, 1024)):
        W, x = o.f8_weight(normal(g, N, K) * K ** -0.5), normal(g, T, K, dtype=BF16)
        X = o.f8_rows(x)
        want, carried = product(X.values(F32), W.values(F32))
        got = o.linear_f8(X, W)
        assert bool(((got.to(F64) - want).abs() <= near(K, carried)).all())
        assert torch.equal(o.linear_f8(x, W), got) and torch.equal(o.linear_f8(X, W, BF16), got.to(BF16))
        stream = normal(g, T, N)
        total = stream + got
        assert o.linear_f8(X, W, residual=stream) is stream and torch.equal(stream, total)
    for N, K in ((9700, 200), (10240, 640)):
        W, X = o.f8_weight(normal(g, 2 * N, K) * K ** -0.5, gated=True), o.f8_rows(normal(g, T, K, dtype=BF16))
        y, carried = product(X.values(F32), W.values(F32))
        gate, up, off = y[:, :N], y[:, N:], near(K, carried)
        want = middle(gate, up, 0, 0.0)
        slack = 1.7 * (off[:, :N] * (up.abs() + 1) + off[:, N:] * gate.abs()) + 32 * 2.0 ** -24 * (gate.abs() + 1) * (up.abs() + 1)
        bound = half_step(want) * (1 + 2.0 ** -16) + 1.1 * slack + flat(blocks(slack, 1).amax(dim=3, keepdim=True).expand(-1, -1, -1, 128), T, N) * 2.0 ** -4
        assert bool(((o.linear_silu_mul_f8(X, W).values(F32).to(F64) - want).abs() <= bound).all())
    assert o.stream_status(torch.device(DEV)).tolist() == [0, 0]


@pytest.mark.parametrize("T,E,top,ff,W", [(1, 16, 12, 96, 264), (2, 40, 9, 264, 520), (3, 20, 20, 130, 136), (4, 4097, 2, 8, 16), (300, 24, 17, 96, 264), (4300, 8, 8, 64, 136)])
def test_more_picks_and_experts(T, E, top, ff, W):
    """More picks a token than a cluster adds up, more than are in flight together, more tokens than the sorting keeps in registers; more experts than a call routes to are refused."""
    from test_blocks_f8_gpu import test_experts
    if E <= 4096:
        return test_experts(T, E, top, ff, W, "silu", 0.0, False)
    o, g = ops(), gen(E)
    G, D = o.f8_weight(normal(g, E, 2 * ff, W), gated=True), o.f8_weight(normal(g, E, W, ff))
    with pytest.raises(o.KernelError):
        o.moe_f8(normal(g, T, W, dtype=BF16), G, D, torch.zeros(T, top, dtype=torch.int32, device=DEV), torch.ones(T, top, device=DEV))


def test_another_stream_and_a_wrong_operand():
    o, g = ops(), gen(4)
    W = o.f8_weight(normal(g, 300, 520))
    x = normal(g, 70, 520, dtype=BF16)
    want = o.linear_f8(x, W)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = o.linear_f8(x, W)
    s.synchronize()
    assert torch.equal(got, want)
    for call in (lambda: o.linear_f8(x.t().contiguous().t(), W), lambda: o.linear_f8(o.f8_rows(x), W, residual=torch.zeros(300, 70, device=DEV).t()),
                 lambda: o.f8_weight(torch.zeros(4, 4, 0, device=DEV)), lambda: o.f8_rows(torch.zeros(4, 0, device=DEV))):
        with pytest.raises(o.KernelError):
            call()


#: (T, N, K, gated, a matrix that the product takes to 8 bits itself): tiles of 16, 32 and 64 rows with K whole and cut, CTAs of 128 rows, pairs of CTAs with one
#: tile and several
SIZES = [(4, 4096, 4096, False, False), (4, 512, 2048, True, False), (3, 1000, 4104, False, True), (16, 700, 12288, True, True), (30, 1024, 4096, False, False),
         (64, 12288, 1024, False, False), (64, 512, 4096, True, False), (250, 700, 4096, False, False), (2000, 4096, 1024, False, False), (2000, 4096, 640, True, False),
         (2000, 2050, 640, True, False), (600, 4096, 4096, False, False), (700, 4001, 1024, False, False), (100, 20480, 512, False, False), (100, 10240, 512, True, False), (4, 128, 65536, False, False), (40, 200, 65536, False, False)]
#: tries of a wait: from none to enough for most waits, so that products stop in front of their first stage, among the stages, and not at all
TRIES = [0, 1, 2, 3] + [2 ** n for n in range(2, 14)]


@pytest.mark.parametrize("T,N,K,gated,plain", SIZES)
def test_what_is_under_way_ends_with_the_product(T, N, K, gated, plain):
    """Whatever the number of tries: the status says that a wait ran out or the result is right, and the products behind it are."""
    o, g = ops(), gen(T + N + K)
    W = o.f8_weight(normal(g, 2 * N if gated else N, K) * K ** -0.5, gated=gated)
    x = normal(g, T, K, dtype=BF16)
    X = x if plain else o.f8_rows(x)
    run = (lambda **k: o.linear_silu_mul_f8(X, W, **k).values(F32)) if gated else (lambda **k: o.linear_f8(X, W, **k))
    status = o.stream_status(torch.device(DEV))
    want, ran_out = run(), []
    assert status.tolist() == [0, 0]
    try:
        for tries in TRIES:
            for _ in range(3):
                got, code = run(waits=tries), status.tolist()[0]
                assert code == 10 or (code == 0 and torch.equal(got, want)), tries
                status.zero_()
                ran_out.append((tries, code))
                assert torch.equal(run(), want) and status.tolist() == [0, 0], tries
    finally:
        status.zero_()
    assert ran_out[0] == (0, 10)


@pytest.mark.parametrize("T,N,K,plain", [(T, N, K, plain) for T, N, K, gated, plain in SIZES if not gated] + [(129, 4096, 4096, False), (5000, 2560, 1024, False)])
def test_what_was_not_computed_is_not_added(T, N, K, plain):
    """A stream that a product was to be added to: without any tries as it was; with some, every value as it was or with its whole sum."""
    o, g = ops(), gen(T + N + K + 1)
    W = o.f8_weight(normal(g, N, K) * K ** -0.5)
    x = normal(g, T, K, dtype=BF16)
    X = x if plain else o.f8_rows(x)
    before = normal(g, T, N)
    total = o.linear_f8(X, W, residual=before.clone())
    status = o.stream_status(torch.device(DEV))
    assert status.tolist() == [0, 0] and not torch.equal(total, before)
    try:
        for tries in TRIES:
            stream = before.clone()
            o.linear_f8(X, W, residual=stream, waits=tries)
            code = status.tolist()[0]
            status.zero_()
            assert code == 10 or (code == 0 and torch.equal(stream, total)), tries
            added = stream != before
            assert bool((stream[added] == total[added]).all()), tries
            assert tries > 0 or (code == 10 and not bool(added.any()))
    finally:
        status.zero_()


@pytest.mark.parametrize("T", TOKENS)
def test_experts_that_give_up(T):
    o, g = ops(), gen(T)
    E, top, ff, K = 16, 8, 264, 1032
    S, SD = o.f8_weight(normal(g, E, 2 * ff, K) * K ** -0.5, gated=True), o.f8_weight(normal(g, E, K, ff) * ff ** -0.5)
    score, ids = torch.topk(normal(g, T, E), top, dim=1)
    x, ids, weights = normal(g, T, K, dtype=BF16), ids.to(torch.int32), torch.softmax(score, dim=1)
    want = o.moe_f8(x, S, SD, ids, weights)
    status = o.stream_status(torch.device(DEV))
    try:
        for tries in TRIES:
            got, code = o.moe_f8(x, S, SD, ids, weights, waits=tries), status.tolist()[0]
            assert code == 10 or (code == 0 and torch.equal(got, want)), tries
            assert tries > 0 or code == 10
            status.zero_()
            assert torch.equal(o.moe_f8(x, S, SD, ids, weights), want) and status.tolist() == [0, 0], tries
    finally:
        status.zero_()


@pytest.mark.parametrize("T", [4, 20, 64, 250, 2000])
def test_a_result_that_was_not_computed_is_not_written(T):
    """The kernels' own entries with room that the test filled: without tries nothing of it changes."""
    o, g = ops(), gen(T)
    W, G, X = o.f8_weight(normal(g, 700, 512)), o.f8_weight(normal(g, 1400, 512), gated=True), o.f8_rows(normal(g, T, 512))
    status = o.stream_status(torch.device(DEV))
    try:
        made = o.F8Rows(T, 700, torch.device(DEV))
        made.buffer.fill_(77)
        rc = o._mx_call("llm_linear_f8_silu_mul")(G.described(), X.buffer.data_ptr(), X.padded, None, 0, made.buffer.data_ptr(), made.padded, T, 0, 0.0, 0,
                                                  status.data_ptr(), o._stream())
        assert rc == 0 and status.tolist()[0] == 10 and bool((made.buffer == 77).all())
        status.zero_()
        room = torch.full((T, 700), 77.0, device=DEV)
        rc = o._mx_call("llm_linear_f8")(W.described(), X.buffer.data_ptr(), X.padded, None, 0, room.data_ptr(), 0, False, T, 0, status.data_ptr(), o._stream())
        assert rc == 0 and status.tolist()[0] == 10 and bool((room == 77).all())
    finally:
        status.zero_()
