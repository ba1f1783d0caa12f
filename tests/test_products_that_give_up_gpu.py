"""Microscaled products whose bounded waits run out: who learns of it, and what stands behind them."""
import pytest
import torch

import tiny_models as tm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def ops():
    from litellmengine_b200.csrc import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def test_a_runner_on_cuda_without_an_index_learns_of_it():
    from litellmengine_b200.config import config_from_dict
    from litellmengine_b200.engine import ModelRunner
    from litellmengine_b200.weights import DictSource
    o, g = ops(), gen(1)
    w = tm.make_weights(tm.TINY_A, 0, bf16_exact=True)
    runner = ModelRunner.from_config(config_from_dict(tm.TINY_A), dtype="bfloat16", device="cuda", page_size=4, max_total_tokens=64, max_requests=2,
                                     source=DictSource({k: (v.to(BF16) if v.dim() == 2 else v) for k, v in w.items()}), weight_format="mxfp4")
    runner.check_status()
    x, W = o.mx_rows(normal(g, 3, 256)), o.mx_weight(normal(g, 128, 256))
    o.linear_mx(x, W, waits=0)
    with pytest.raises(RuntimeError, match="device status 9"):
        runner.check_status()
    runner.check_status()


#: single CTAs of every width with K whole and cut, a matrix that the product takes to 8 bits itself, pairs of CTAs with one tile and several
SIZES = [(4, 4096, 4096, False, False), (4, 512, 2048, True, False), (3, 1000, 4104, False, True), (16, 700, 12288, True, True), (30, 1024, 4096, False, False),
         (64, 12288, 1024, False, False), (64, 512, 4096, True, False), (2000, 4096, 1024, False, False), (2000, 4096, 640, True, False),
         (600, 4096, 4096, False, False), (700, 4001, 1024, False, False),
         # few tiles and a long K: waits for the sums run out among the stages
         (4, 128, 65536, False, False), (40, 200, 65536, False, False), (20, 64, 65536, True, False), (2, 128, 65536, False, True)]
#: tries of a wait: from none to enough for most waits, so that products stop in front of their first stage, among the stages, and not at all
TRIES = [0, 1, 2, 3] + [2 ** n for n in range(2, 14)]


@pytest.mark.parametrize("T,N,K,gated,plain", SIZES)
def test_what_is_under_way_ends_with_the_product(T, N, K, gated, plain):
    """Whatever the number of tries: the status says that a wait ran out or the result is right, and the products behind it are."""
    o, g = ops(), gen(T + N + K)
    W = o.mx_weight(normal(g, 2 * N if gated else N, K) * K ** -0.5, gated=gated)
    x = normal(g, T, K, dtype=BF16)
    X = x if plain else o.mx_rows(x)
    run = (lambda **k: o.linear_silu_mul_mx(X, W, **k).values(F32)) if gated else (lambda **k: o.linear_mx(X, W, **k))
    status = o.stream_status(torch.device(DEV))
    want, ran_out = run(), []
    assert status.tolist() == [0, 0]
    try:
        for tries in TRIES:
            for _ in range(3):
                got, code = run(waits=tries), status.tolist()[0]
                assert code == 9 or (code == 0 and torch.equal(got, want)), tries
                status.zero_()
                ran_out.append((tries, code))
                assert torch.equal(run(), want) and status.tolist() == [0, 0], tries
    finally:
        status.zero_()
    assert ran_out[0] == (0, 9)
    print(T, N, K, gated, plain, "ran out:", [t for t, c in ran_out if c])


@pytest.mark.parametrize("T,N,K,plain", [(T, N, K, plain) for T, N, K, gated, plain in SIZES if not gated] + [(129, 4096, 4096, False), (5000, 2560, 1024, False)])
def test_what_was_not_computed_is_not_added(T, N, K, plain):
    """A stream that a product was to be added to: without any tries as it was; with some, every value as it was or with its whole sum."""
    o, g = ops(), gen(T + N + K + 1)
    W = o.mx_weight(normal(g, N, K) * K ** -0.5)
    x = normal(g, T, K, dtype=BF16)
    X = x if plain else o.mx_rows(x)
    before = normal(g, T, N)
    total = o.linear_mx(X, W, residual=before.clone())
    status = o.stream_status(torch.device(DEV))
    assert status.tolist() == [0, 0] and not torch.equal(total, before)
    some = 0
    try:
        for tries in TRIES:
            stream = before.clone()
            o.linear_mx(X, W, residual=stream, waits=tries)
            code = status.tolist()[0]
            status.zero_()
            assert code == 9 or (code == 0 and torch.equal(stream, total)), tries
            added = stream != before
            assert bool((stream[added] == total[added]).all()), tries
            assert tries > 0 or (code == 9 and not bool(added.any()))
            some += code == 9 and bool(added.any())
    finally:
        status.zero_()
    print(T, N, K, plain, "added in part:", some)


@pytest.mark.parametrize("T,N,K,gated", [(4, 4096, 4096, False), (60, 512, 2048, True), (2000, 4096, 1024, False), (2000, 4096, 640, True), (700, 4001, 1024, False)])
def test_a_result_that_was_not_computed_is_not_written(T, N, K, gated):
    """The kernels' own entries with room that the test filled: without tries nothing of it changes."""
    o, g = ops(), gen(T + N + K + 2)
    W, X = o.mx_weight(normal(g, 2 * N if gated else N, K), gated=gated), o.mx_rows(normal(g, T, K))
    status = o.stream_status(torch.device(DEV))
    at = W.buffer.data_ptr()
    try:
        if gated:
            room = o.MxRows(T, N, torch.device(DEV))
            room.buffer.fill_(77)
            rc = o._mx_call("llm_linear_mx_silu_mul")(X.buffer.data_ptr(), None, 0, at, at + W.scales_behind, room.buffer.data_ptr(), T, N, K, 0, 0.0, 0, status.data_ptr(),
                                                      o._stream())
            kept = bool((room.buffer == 77).all())
        else:
            room = torch.full((T, N), 77.0, device=DEV)
            rc = o._mx_call("llm_linear_mx")(X.buffer.data_ptr(), None, 0, at, at + W.scales_behind, room.data_ptr(), 0, False, T, N, K, 0, status.data_ptr(), o._stream())
            kept = bool((room == 77).all())
        assert rc == 0 and status.tolist()[0] == 9 and kept
    finally:
        status.zero_()
