"""Limits of products of 8 bits: refused before anything is replaced, and the same on both sides of the library."""
import os
import re

import pytest
import torch

from litellmengine_b200.csrc import ops

BF16 = torch.bfloat16


def defined(name, file):
    with open(os.path.join(os.path.dirname(ops.__file__), file), encoding="utf-8") as f:
        return re.search(rf"^#define {re.escape(name)} +(.+?) *(?://.*)?$", f.read(), re.M).group(1)


def experts(E):
    from litellmengine_b200.config.specs import FeedForwardSpec
    from litellmengine_b200.parts.feed_forward import RoutedExperts
    params = (("experts", E), ("top", 2), ("activation", "silu"), ("score", "softmax"))
    part = RoutedExperts(FeedForwardSpec(kind="moe", intermediate_size=1, params=params), 2, BF16, "cpu")
    part.load({n: torch.ones(ps.shape, dtype=BF16) for n, ps in part.parameters().items()})
    return part


def test_more_experts_than_a_call_routes_to_are_refused_when_they_would_be_held(monkeypatch):
    assert ops.F8_MOST_EXPERTS == int(defined("F8_MOST_EXPERTS", "f8_blocks.cuh"))
    monkeypatch.setattr(ops, "f8_weight", lambda w, gated=False: ("8 bits", tuple(w.shape)))
    part = experts(ops.F8_MOST_EXPERTS + 1)
    before = part.w_gate_up, part.w_down
    with pytest.raises(ValueError, match="4097 routed experts.* 4096 "):
        part.hold_in_8_bits()
    assert part.w_gate_up is before[0] and part.w_down is before[1]
    part = experts(ops.F8_MOST_EXPERTS)
    assert part.hold_in_8_bits() == 2 and part.w_gate_up == ("8 bits", (4096, 2, 2))


def test_rows_that_a_product_makes_itself():
    """Python leaves out the room for rows where the library says that the product makes them: the same numbers on both sides."""
    gated, others = re.fullmatch(r"\(\(GATED\) \? (\d+) : (\d+)\)", defined("F8_PLAIN_ROWS(GATED)", "gemm_f8_tcgen05.cu")).groups()
    assert (int(others), int(gated)) == (ops.F8_PLAIN_ROWS, ops.F8_PLAIN_ROWS_GATED)
