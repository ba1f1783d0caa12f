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
         (600, 4096, 4096, False, False), (700, 4001, 1024, False, False)]
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
