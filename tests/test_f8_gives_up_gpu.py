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
