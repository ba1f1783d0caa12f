"""What loading a model of 4-bit weights leaves undone: tiled copies of matrices that are about to be replaced."""
import pytest
import torch

import tiny_models as tm
from litellmengine_b200.config import config_from_dict
from litellmengine_b200.csrc import ops
from litellmengine_b200.parts.feed_forward import SwiGLU
from litellmengine_b200.parts.model import Model
from litellmengine_b200.weights import DictSource


def weights(cfg):
    return {n: t.to(torch.bfloat16) if t.dim() == 2 else t for n, t in tm.make_weights(cfg, 0, bf16_exact=True).items()}


@pytest.fixture
def loads(monkeypatch):
    """(the bytes a model announces, [(a matrix' shape, whether it may have a copy)]) of the models that are loaded; copies are allowed to all."""
    said = {"bytes": [], "copies": []}

    def begin(matrix_bytes, device):
        said["bytes"].append(matrix_bytes)
        ops._tiled_allowed = True
        return True

    monkeypatch.setattr(ops, "_tiled_allowed", True)
    monkeypatch.setattr(ops, "begin_model", begin)
    monkeypatch.setattr(ops, "prepare_streaming", lambda w: said["copies"].append((tuple(w.shape), ops._tiled_allowed)))
    monkeypatch.setattr(ops, "mx_weight", lambda w, gated=False: ("4 bits", tuple(w.shape)))
    return said


def test_only_what_stays_has_copies(loads):
    cfg, w = tm.TINY_A, weights(tm.TINY_A)
    layers = [t for n, t in w.items() if t.dim() == 2 and ".layers." in n]
    rest = [t for n, t in w.items() if t.dim() == 2 and ".layers." not in n]
    for f in ("stored", "mxfp4"):
        Model(config_from_dict(cfg).plan(), device="cpu", weight_format=f).load_weights(DictSource(w))
    head = (cfg["vocab_size"], cfg["hidden_size"])
    stored, held = loads["copies"][:len(loads["copies"]) // 2], loads["copies"][len(loads["copies"]) // 2:]
    assert [s for s, _ in stored] == [s for s, _ in held] and all(may for _, may in stored)
    assert held[-1] == (head, True) and not any(may for _, may in held[:-1])       # the output head comes last
    assert loads["bytes"][0] - loads["bytes"][1] == sum(2 * t.numel() - t.numel() * 17 // 32 for t in layers)
    assert loads["bytes"][0] == sum(2 * t.numel() for t in layers + rest)
    assert ops._tiled_allowed is True


def test_parts_that_keep_their_matrices_keep_their_copies(loads, monkeypatch):
    monkeypatch.delattr(SwiGLU, "hold_in_4_bits")
    cfg, w = tm.TINY_A, weights(tm.TINY_A)
    Model(config_from_dict(cfg).plan(), device="cpu", weight_format="mxfp4").load_weights(DictSource(w))
    inter, hidden = cfg["intermediate_size"], cfg["hidden_size"]
    assert {s for s, may in loads["copies"] if may} >= {(2 * inter, hidden), (hidden, inter)}
    assert [may for s, may in loads["copies"]].count(False) == 2 * cfg["num_hidden_layers"]
    mine = [t.numel() for n, t in w.items() if "self_attn" in n and t.dim() == 2]
    assert mine and loads["bytes"] == [sum(2 * t.numel() for t in w.values() if t.dim() == 2) - sum(2 * n - n * 17 // 32 for n in mine)]


def test_an_error_while_loading_leaves_the_rule_as_it_was(loads):
    with pytest.raises(RuntimeError):
        with ops.no_tiled_copies():
            assert ops._tiled_allowed is False
            raise RuntimeError
    assert ops._tiled_allowed is True


@pytest.mark.gpu
def test_no_copy_outlives_the_matrix(monkeypatch):
    """A source whose tensors are on the device and stay: the matrices' copies would stay with them."""
    monkeypatch.setattr(ops, "_TILED_POLICY", "on")
    cfg = dict(tm.TINY_E, hidden_size=256, intermediate_size=512, num_hidden_layers=2)
    w = {n: t.to("cuda:0") for n, t in weights(cfg).items()}
    ops.release_streaming()
    kept = {}
    for f in ("stored", "mxfp4"):
        model = Model(config_from_dict(cfg).plan(), device="cuda:0", weight_format=f)
        model.load_weights(DictSource(w))
        kept[f] = [v.numel() for v in ops._tiled.values()]
        head = ops._tiled[model.output.data_ptr()]
        del model
        ops.release_streaming()
    assert len(kept["stored"]) == 2 * 4 + 1 and kept["mxfp4"] == [head.numel()]
    # and a feed-forward whose residual the product does not take gives its result instead
    ff = Model(config_from_dict(cfg).plan(), device="cuda:0", weight_format="mxfp4")
    ff.load_weights(DictSource(w))
    ff = ff.blocks[0].feed_forward
    x = torch.randn(5, 256, generator=torch.Generator("cuda:0").manual_seed(1), device="cuda:0").to(torch.bfloat16)
    want, stream = ff.forward(x), torch.zeros(5, 256, dtype=torch.bfloat16, device="cuda:0")
    assert torch.equal(ff.forward(x, residual=stream), want) and stream.count_nonzero() == 0
    assert ff.forward(x, residual=torch.zeros_like(want)) is None
