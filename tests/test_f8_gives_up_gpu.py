"""Products of 8 bits whose bounded waits run out: who learns of it, and in which words."""
import pytest
import torch

import tiny_models as tm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("device", ["cuda", "cuda:0"])
@pytest.mark.parametrize("T", [3, 40, 300])
def test_a_runner_learns_of_it(device, T):
    from litellmengine_b200.config import config_from_dict
    from litellmengine_b200.csrc import ops as o
    from litellmengine_b200.engine import ModelRunner
    from litellmengine_b200.weights import DictSource
    w = tm.make_weights(tm.TINY_A, 0, bf16_exact=True)
    runner = ModelRunner.from_config(config_from_dict(tm.TINY_A), dtype="bfloat16", device=device, page_size=4, max_total_tokens=64, max_requests=2,
                                     source=DictSource({k: (v.to(torch.bfloat16) if v.dim() == 2 else v) for k, v in w.items()}), weight_format="fp8")
    runner.check_status()
    x, W = o.f8_rows(torch.ones(T, 256, device=DEV)), o.f8_weight(torch.ones(128, 256, device=DEV))
    o.linear_f8(x, W, waits=0)
    with pytest.raises(RuntimeError, match="device status 10: a wait on a barrier in a product of 8 bits .* ran out"):
        runner.check_status()
    runner.check_status()


@pytest.mark.parametrize("T,E,top,ff,W", [(300, 16, 8, 264, 1032), (1700, 16, 8, 264, 1032), (1700, 2, 1, 128, 520)])
def test_experts_with_larger_items(T, E, top, ff, W):
    """Items of 128 rows and of 256, by how many picks an expert has: the status says that a wait ran out or the result is right, and the call behind it is."""
    from litellmengine_b200.csrc import ops as o
    g = torch.Generator(device=DEV).manual_seed(T + E)
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEV)
    G, D = o.f8_weight(normal(E, 2 * ff, W) * W ** -0.5, gated=True), o.f8_weight(normal(E, W, ff) * ff ** -0.5)
    score, ids = torch.topk(normal(T, E), top, dim=1)
    x, ids, weights = normal(T, W).to(torch.bfloat16), ids.to(torch.int32), torch.softmax(score, dim=1)
    want = o.moe_f8(x, G, D, ids, weights, out_dtype=torch.bfloat16)
    status = o.stream_status(torch.device(DEV))
    assert status.tolist() == [0, 0]
    try:
        for tries in [0, 1, 2, 3] + [2 ** n for n in range(2, 14)]:
            got, code = o.moe_f8(x, G, D, ids, weights, out_dtype=torch.bfloat16, waits=tries), status.tolist()[0]
            assert code == 10 or (code == 0 and tries > 0 and torch.equal(got, want)), tries
            status.zero_()
            assert torch.equal(o.moe_f8(x, G, D, ids, weights, out_dtype=torch.bfloat16), want) and status.tolist() == [0, 0], tries
    finally:
        status.zero_()
