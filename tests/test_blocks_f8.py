"""Products of 8 bits under float32 scales, as far as they need no device: sizes of what is held, refusals, which parts hold their matrices so, the command line's option."""
import pytest
import torch

from litellmengine_b200 import cli
from litellmengine_b200.csrc import ops

BF16 = torch.bfloat16
CPU = torch.device("cpu")


def refuses(call, *args, **kw):
    with pytest.raises(ops.KernelError):
        call(*args, **kw)


def test_sizes_of_rows_and_weights():
    assert [ops.f8_padded_rows(t) for t in (1, 16, 17, 32, 33, 64, 65, 128, 129, 257)] == [16, 16, 32, 32, 64, 64, 128, 128, 256, 384]
    rows = ops.F8Rows(70, 700, CPU)
    assert rows.shape == (70, 700) and rows.codes.shape == (6, 128, 128) and rows.scales.shape == (128, 8) and rows.scales.dtype == torch.float32
    w = ops.F8Weight((300, 700), False, CPU)
    assert w.codes.shape == (1, 4, 6, 128, 128) and w.scales.shape == (1, 4, 3, 8) and w.nbytes == 4 * (6 * 128 * 128 + 3 * 8 * 4)
    g = ops.F8Weight((5, 2 * 65, 100), True, CPU)
    assert g.experts == 5 and g.codes.shape == (5, 2, 1, 128, 128) and g.scales.shape == (5, 2, 3, 4)


def test_nothing_runs_without_a_device():
    x, w = torch.zeros(4, 64, dtype=BF16), torch.zeros(32, 64)
    W, G, S = ops.F8Weight((32, 64), False, CPU), ops.F8Weight((3, 32, 64), True, CPU), ops.F8Weight((3, 64, 16), False, CPU)
    ids, weights = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    for call in (lambda: ops.f8_weight(w), lambda: ops.f8_rows(x), lambda: ops.linear_f8(x, W), lambda: ops.linear_f8(ops.F8Rows(4, 64, CPU), W), lambda: W.values(),
                 lambda: ops.F8Rows(4, 64, CPU).values(), lambda: ops.linear(x, W), lambda: ops.moe_f8(x, G, S, ids, weights)):
        refuses(call)


def test_refusals_that_come_before_the_device():
    x = torch.zeros(4, 64, dtype=BF16)
    W, G, S = ops.F8Weight((32, 64), False, CPU), ops.F8Weight((32, 64), True, CPU), ops.F8Weight((3, 32, 64), False, CPU)
    for call in (lambda: ops.linear_f8(x, G), lambda: ops.linear_f8(x, S), lambda: ops.linear_f8(x[:, :63], W), lambda: ops.linear_silu_mul_f8(x, W), lambda: ops.linear_f8("x", W),
                 lambda: ops.linear_f8(x, torch.zeros(32, 64))):
        refuses(call)
    with pytest.raises(KeyError):
        ops.linear_silu_mul_f8(x, G, activation="relu")


def test_a_residual_that_the_product_does_not_take_is_declined():
    W = ops.F8Weight((32, 64), False, CPU)
    x = torch.zeros(4, 64, dtype=BF16)
    for residual in (torch.ones(4, 32, dtype=BF16), torch.ones(32, 4).t(), torch.ones(4, 31), torch.ones(5, 32)):
        assert ops.linear_into(x, W, residual) is False and bool((residual == 1).all())
    refuses(ops.linear_into, x, W, torch.ones(4, 32))             # one that it takes: no device here


def test_a_copy_of_a_weight_is_described_for_itself():
    import copy
    w = ops.F8Weight((32, 64), False, CPU)
    w._described = (w.buffer.data_ptr(), 1, None)
    other = copy.deepcopy(w)
    assert w.described() == 1 and "_described" not in other.__dict__ and other.buffer.data_ptr() != w.buffer.data_ptr() and other.shape == w.shape


def test_matrices_are_held_in_8_bits_by_parts_that_say_so_of_their_own_forward(monkeypatch):
    import tiny_models as tm
    from litellmengine_b200.config import config_from_dict
    from litellmengine_b200.parts import registry
    from litellmengine_b200.parts.feed_forward import SwiGLU
    from litellmengine_b200.parts.model import Model
    from litellmengine_b200.weights import DictSource

    class Own(SwiGLU):
        def forward(self, x, **k):
            return x @ self.w_down.t()

    class Again(Own):
        def hold_in_8_bits(self):
            return super().hold_in_8_bits()

    monkeypatch.setattr(ops, "f8_weight", lambda w, gated=False: ("8 bits", gated))
    w = {n: t.to(BF16) if t.dim() == 2 else t for n, t in tm.make_weights(tm.TINY_A, 0, bf16_exact=True).items()}
    kind = next(k for k, c in registry._KINDS["feed_forward"].items() if c is SwiGLU)
    for cls, held in ((SwiGLU, True), (Own, False), (Again, True)):
        monkeypatch.setitem(registry._KINDS["feed_forward"], kind, cls)
        model = Model(config_from_dict(tm.TINY_A).plan(), device="cpu", weight_format="fp8")
        model.load_weights(DictSource(w))
        for block in model.blocks:
            assert block.mixer.w_qkv == ("8 bits", False) and type(block.feed_forward) is cls
            assert isinstance(block.feed_forward.w_down, tuple) == held and isinstance(block.feed_forward.w_gate_up, tuple) == held


def test_experts_are_held_as_stacks(monkeypatch):
    """What of the stored matrices each stack is made of, with and without a shared expert behind the routed ones."""
    from litellmengine_b200.config.specs import FeedForwardSpec
    from litellmengine_b200.parts.feed_forward import RoutedExperts
    monkeypatch.setattr(ops, "f8_weight", lambda w, gated=False: (w.clone(), gated))
    for shared in (0, 24):
        params = [("experts", 3), ("top", 2), ("activation", "silu"), ("score", "softmax")] + ([("shared", shared), ("shared_gate", True)] if shared else [])
        part = RoutedExperts(FeedForwardSpec(kind="moe", intermediate_size=16, params=tuple(params)), 40, BF16, "cpu")
        t = {n: torch.randn(ps.shape).to(BF16) for n, ps in part.parameters().items()}
        part.load(t)
        assert part.hold_in_8_bits() == (4 if shared else 2)
        (gu, gated), (dn, plain) = part.w_gate_up, part.w_down
        assert gated and not plain
        for e in range(3):
            assert torch.equal(gu[e], torch.cat([t[f"e{e}.gate"], t[f"e{e}.up"]])) and torch.equal(dn[e], t[f"e{e}.down"])
        if shared:
            assert torch.equal(part.w_shared_gate_up[0], torch.cat([t["shared.gate"], t["shared.up"]])) and torch.equal(part.w_shared_down[0], t["shared.down"])


def test_weight_format():
    assert cli.parse_args(["--model", "m", "--weight-format=fp8"]).weight_format == "fp8"
    with pytest.raises(cli.ArgError, match="--weight-format"):
        cli.parse_args(["--model", "m", "--weight-format", "fp8", "--dtype", "float32"])


def test_a_block_refuses_a_weight_format_that_it_does_not_know():
    from litellmengine_b200.parts.block import Block
    block = Block.__new__(Block)
    for unknown in ("fp4", True, None):
        with pytest.raises(ValueError):
            block.parts_that_hold(unknown)
