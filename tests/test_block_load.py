"""The ways of saying in what a block holds its matrices."""
import pytest
import torch

import tiny_models as tm
from litellmengine_b200.config import config_from_dict
from litellmengine_b200.csrc import ops
from litellmengine_b200.parts.block import Block

BF16 = torch.bfloat16


@pytest.fixture
def block_and_tensors(monkeypatch):
    monkeypatch.setattr(ops, "mx_weight", lambda w, gated=False: ("4 bits", gated))
    monkeypatch.setattr(ops, "f8_weight", lambda w, gated=False: ("8 bits", gated))
    plan = config_from_dict(tm.TINY_A).plan()
    spec = plan.blocks[0]
    w = {n: t.to(BF16) if t.dim() == 2 else t for n, t in tm.make_weights(tm.TINY_A, 0, bf16_exact=True).items()}
    block = Block(spec, plan.hidden_size, BF16, torch.device("cpu"))
    return block, {n: w[f"{spec.weight_prefix}.{n}"] for n, ps in block.parameters().items() if f"{spec.weight_prefix}.{n}" in w}


@pytest.mark.parametrize("args,kw,held", [((), {}, None), ((False,), {}, None), ((), {"in_4_bits": False}, None), (("stored",), {}, None),
                                          ((True,), {}, "4 bits"), ((), {"in_4_bits": True}, "4 bits"), ((), {"weight_format": "mxfp4"}, "4 bits"),
                                          (("mxfp4",), {"in_4_bits": True}, "4 bits"), (("fp8",), {}, "8 bits"), ((), {"weight_format": "fp8"}, "8 bits")])
def test_formats(block_and_tensors, args, kw, held):
    block, t = block_and_tensors
    assert block.load(t, *args, **kw) == (4 if held else 0)
    matrices = (block.mixer.w_qkv, block.mixer.w_o, block.feed_forward.w_gate_up, block.feed_forward.w_down)
    assert all((m[0] == held if held else isinstance(m, torch.Tensor)) for m in matrices)
    assert [type(p) for p in block.parts_in_4_bits()] == [type(p) for p in block.parts_that_hold("mxfp4")] != []


def test_two_formats_at_once_are_refused(block_and_tensors):
    block, t = block_and_tensors
    for bad in ({"weight_format": "fp8", "in_4_bits": True}, {"weight_format": "fp4"}):
        with pytest.raises(ValueError):
            block.load(t, **bad)
