"""Models whose matrices are held in 8 bits under a float32 scale per block of 128 x 128: the Qwen3 ones against the plain code's own functions with weights and
products' inputs rounded to the format, in every way of cutting the work; other designs, those with routed experts among them, against themselves with the
same weights in 16 bits; generation, captured steps, the command line, refusals."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_qwen3 as pq
import replay_helpers as rh
import tiny_models as tm
from test_blocks_f8_gpu import held

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"


def runner_for(config, weights, page, pool, weight_format="fp8", **kw):
    from litellmengine_b200.config import config_from_dict
    from litellmengine_b200.engine import ModelRunner
    from litellmengine_b200.weights import DictSource
    src = DictSource({k: (v.to(torch.bfloat16) if v.dim() == 2 else v) for k, v in weights.items()})
    return ModelRunner.from_config(config_from_dict(config), dtype="bfloat16", device=DEV, source=src, page_size=page, max_total_tokens=pool,
                                   weight_format=weight_format, **kw)


def plain_rows(cfg, w, reqs):
    """As the engine computes: rows of 8 bits, made of bfloat16 but for the feed-forward's middle, in front of every product of a layer; weights of 8 bits, the
    blocks of fused matrices counted through them; queries, keys, values and attention's output in bfloat16, the head in bfloat16."""
    act = lambda x: held(x, 1)
    w = {n: t.to(torch.bfloat16).float() if t.dim() == 2 else t.float() for n, t in w.items()}
    for layer in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{layer}"
        for group in ([f"{p}.self_attn.{k}_proj.weight" for k in "qkv"], [f"{p}.self_attn.o_proj.weight"], [f"{p}.mlp.gate_proj.weight", f"{p}.mlp.up_proj.weight"],
                      [f"{p}.mlp.down_proj.weight"]):
            for n, t in zip(group, held(torch.cat([w[n] for n in group]), 128).split([len(w[n]) for n in group])):
                w[n] = t
    eps, nq, d = cfg["rms_norm_eps"], cfg["num_attention_heads"], cfg["head_dim"]
    weights = pq.to_bf16 if rh.rounds_attention_weights(cfg) else None
    out = {}
    for r, ids in reqs.items():
        h = pq.embedding(torch.as_tensor(ids), pq.to_bf16(w["model.embed_tokens.weight"]))
        positions = torch.arange(len(ids), dtype=torch.int32)
        for layer in range(cfg["num_hidden_layers"]):
            p = f"model.layers.{layer}"
            q, k, v = pq.attention_qkv(act(pq.to_bf16(pq.rms_norm(h, w[f"{p}.input_layernorm.weight"], eps))), positions, w, f"{p}.self_attn", cfg, pq.to_bf16)
            a = pq.to_bf16(pq.causal_attention(q, k, v, act=weights)).reshape(len(ids), nq * d)
            h = h + act(a) @ w[f"{p}.self_attn.o_proj.weight"].T
            x = act(pq.to_bf16(pq.rms_norm(h, w[f"{p}.post_attention_layernorm.weight"], eps)))
            m = pq.silu_and_mul(x @ w[f"{p}.mlp.gate_proj.weight"].T, x @ w[f"{p}.mlp.up_proj.weight"].T)
            h = h + act(m) @ w[f"{p}.mlp.down_proj.weight"].T
        head = pq.to_bf16(w.get("lm_head.weight", w["model.embed_tokens.weight"]))
        out[r] = (pq.to_bf16(pq.rms_norm(h, w["model.norm.weight"], eps)) @ head.T).numpy()
    return out


def off(got, ref):
    """2-norm of the difference over that of the reference, all rows together."""
    keys = sorted(got)
    a, b = np.stack([got[k] for k in keys]), np.stack([ref[k[0]][k[1]] for k in keys])
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


# A value that another order of sums puts on the other side of a border comes out a whole step off, at most 2^-3 of it.  What is rounded to bfloat16 first (the
# norms' and attention's output) may differ by 2^-8, which a step of 2^-3 feels one time in 32: 2^-3 sqrt(2^-5) = 0.022 of the 2-norm of a product's input.  Two layers of
# four such inputs, in quadrature: 0.062.
FLIPS = 0.062


@pytest.mark.parametrize("name", ["A", "B", "C", "D", "E", "F"])
def test_every_way_of_cutting(name):
    cfg = getattr(tm, f"TINY_{name}")
    page = getattr(tm, f"TINY_{name}_PAGE")
    w = tm.make_weights(cfg, getattr(tm, f"TINY_{name}_SEED"), bf16_exact=True)
    lengths = [1, 7, 33, 70, 90] if cfg["max_position_embeddings"] < 200 else [2, 16, 65, 129, 200]
    reqs = rh.requests_for(cfg, lengths, 3)
    ref = plain_rows(cfg, w, reqs)
    for steps in (rh.trace_whole(reqs), rh.trace_tail_decode(reqs, 24), rh.trace_portions(reqs, seed=3), rh.trace_mixed(reqs, seed=5, max_live=4)):
        runner = runner_for(cfg, w, page, rh.peak_tokens(steps, page), max_requests=4, max_tokens_per_step=256)
        got = rh.run_trace(runner, steps)
        runner.check_status()
        assert len(got) == sum(lengths)
        assert off(got, ref) < FLIPS * (cfg["num_hidden_layers"] / 2) ** 0.5, name


def test_captured_steps_give_what_launched_ones_give():
    """Decode steps of five requests: replayed graphs and kernels launched one by one, the same bits."""
    cfg, w = tm.TINY_E, tm.make_weights(tm.TINY_E, tm.TINY_E_SEED, bf16_exact=True)
    from litellmengine_b200.engine import PagedGenerateEngine
    prompts = [tm.random_tokens(cfg, n, 80 + n) for n in (3, 9, 17, 40, 65)]
    outs = []
    for graphs in (True, False):
        runner = runner_for(cfg, w, tm.TINY_E_PAGE, 1024, max_requests=5, max_tokens_per_step=256, use_graphs=graphs)
        engine = PagedGenerateEngine(runner)
        outs.append(engine.generate(prompts, max_new_tokens=24))
        assert bool(runner.graph_replays) == graphs
    assert outs[0] == outs[1]


def with_the_same_weights(runner, other):
    """The matrices that `runner` holds in 8 bits, in 16 bits, into `other`: how many."""
    from litellmengine_b200.csrc import ops
    from litellmengine_b200.parts.feed_forward import RoutedExperts

    def into(p, q):
        n = 0
        if isinstance(p, RoutedExperts):
            gu, dn = p.w_gate_up.values(), p.w_down.values()
            gu, dn = gu.reshape(-1, p.hidden), dn.permute(1, 0, 2).reshape(p.hidden, -1)
            if p.joined is not None:
                gu, dn = torch.cat([gu, p.w_shared_gate_up.values()]), torch.cat([dn, p.w_shared_down.values()], dim=1)
                q.w_shared_down = p.w_shared_down.values()
            q.w_gate_up, q.w_down, n = gu.contiguous(), dn.contiguous(), 2
            return n + (into(p.shared, q.shared) if p.shared is not None else 0)
        for name, v in vars(p).items():
            if isinstance(v, ops.F8Weight):
                setattr(q, name, v.values())
                n += 1
        return n

    return sum(into(p, q) for a, b in zip(runner.model.blocks, other.model.blocks) for p, q in zip(a.parts(), b.parts()))


def random_weights(module, name):
    m = __import__(module)
    cfg = getattr(m, name)
    return m, cfg, getattr(m, f"{name}_PAGE"), m.random_weights(cfg, getattr(m, f"{name}_RANK"), 5) if module == "tobovik_models" else m.random_weights(cfg, 5)


@pytest.mark.parametrize("module,name", [("komazen_models", "KOMA_C"), ("komazen_models", "KOMA_F"), ("tobovik_models", "TOBO_C"), ("tobovik_models", "TOBO_D")])
def test_other_designs_against_themselves_in_16_bits(module, name):
    """Gated attention, clamped and gelu feed-forwards, other norms and arrangements, no routers: the same model with the same weights in 16 bits differs by the
    rounding of products' inputs to 8 bits.  That is off by 2^-4 / sqrt(3) of a value at most in quadrature, 0.036; four inputs a layer and up to four
    layers: 0.15, twice that for what sharp attention makes of it."""
    m, cfg, page, w = random_weights(module, name)
    reqs = {f"r{i}": m.random_tokens(cfg, n, 50 + i) for i, n in enumerate((3, 20, 61))}
    steps = rh.trace_mixed(reqs, seed=2, max_live=3)
    kw = dict(max_requests=3, max_tokens_per_step=128)
    runner, other = (runner_for(cfg, w, page, 512, weight_format=f, **kw) for f in ("fp8", "stored"))
    assert with_the_same_weights(runner, other) >= 2
    got, want = rh.run_trace(runner, steps), rh.run_trace(other, steps)
    ref = {r: np.stack([want[(r, p)] for p in range(len(t))]) for r, t in reqs.items()}
    assert 0 < off(got, ref) < 0.3
    runner.check_status()


@pytest.mark.parametrize("module,name", [("gubidra_models", "GUBI_A"), ("gubidra_models", "GUBI_B"), ("vugedra_models", "VUG_A"), ("vugedra_models", "VUG_B"), ("pukatar_models", "PUK_A"),
                                         ("pukatar_models", "PUK_B"), ("purivik_models", "PUR_A"), ("purivik_models", "PUR_B")])
def test_designs_with_routed_experts(module, name):
    """Every feed-forward of a design (each kind of router, shared expert and activation) against the same part with the same weights in 16 bits, for the
    same tokens: its input and its middle are rounded to 8 bits, by 2^-4 of a value at most, the input's share up to 1.7 times that behind a gate (a gate's
    slope is at most 1.1, and a row has two factors): 0.0625 (1.7 + 1) = 0.17 of the 2-norm, where all of them are rounded as far as can be.  (Two models as wholes say nothing: a router picks another expert for a hidden state that is a hair off.)  The
    model itself runs a mixed trace, the same twice."""
    from litellmengine_b200.csrc import ops
    m, cfg, page, w = random_weights(module, name)
    kw = dict(max_requests=3, max_tokens_per_step=128)
    runner, other = (runner_for(cfg, w, page, 512, weight_format=f, **kw) for f in ("fp8", "stored"))
    assert with_the_same_weights(runner, other) >= 2
    g = torch.Generator(device=DEV).manual_seed(7)
    routed = 0
    for a, b in zip(runner.model.blocks, other.model.blocks):
        p, q = a.feed_forward, b.feed_forward
        if p is None:
            continue
        routed += hasattr(p, "w_router")
        for T in (1, 3, 20, 70, 300):
            x = torch.randn(T, p.hidden, generator=g, device=DEV).to(torch.bfloat16)
            got, want = ops.as_tensor(p.forward(x)).float(), ops.as_tensor(q.forward(x)).float()
            assert 0 < float((got - want).norm() / want.norm()) < 0.17, T
    assert routed
    reqs = {f"r{i}": m.random_tokens(cfg, n, 50 + i) for i, n in enumerate((3, 20, 61))}
    steps = rh.trace_mixed(reqs, seed=2, max_live=3)
    got, again = rh.run_trace(runner, steps), rh.run_trace(runner_for(cfg, w, page, 512, **kw), steps)
    runner.check_status()
    assert all(np.isfinite(got[k]).all() and np.array_equal(got[k], again[k]) for k in got) and len(got) == 84


def test_weights_take_half_of_their_bytes():
    cfg = dict(tm.TINY_E, hidden_size=256, intermediate_size=512, num_hidden_layers=1)
    w = tm.make_weights(cfg, 4, bf16_exact=True)
    a, b = (runner_for(cfg, w, 16, 64, weight_format=f).model for f in ("fp8", "stored"))
    layer = sum(t.numel() for n, t in w.items() if t.dim() == 2 and ".layers." in n)
    scales = 3 * 4 * sum(-(-t.shape[0] // 128) * 4 * -(-t.shape[1] // 512) for n, t in w.items() if t.dim() == 2 and ".layers." in n)
    assert b.weight_bytes() - a.weight_bytes() == 2 * layer - layer - scales
    assert a.weight_format == "fp8"


def test_the_command_line(tmp_path):
    from litellmengine_b200.config import config_from_dict
    from litellmengine_b200.weights import write_random_model
    folder = str(tmp_path / "m")
    write_random_model(config_from_dict(tm.TINY_D), folder, seed=3)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "litellmengine"), "--model", folder, "--input-ids", "3,1,4,1,5", "--max-tokens", "6",
                        "--temperature", "0", "--weight-format", "fp8"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert "fp8" in r.stdout and "New token ids:" in r.stdout


def test_refusals(monkeypatch):
    from litellmengine_b200.config import config_from_dict
    from litellmengine_b200.parts.attention import AttentionMixer
    from litellmengine_b200.parts.feed_forward import SwiGLU
    from litellmengine_b200.parts.model import Model
    cfg, w = tm.TINY_A, tm.make_weights(tm.TINY_A, 0, bf16_exact=True)
    with pytest.raises(ValueError, match="weight_format"):
        runner_for(cfg, w, 4, 64, weight_format="fp9")
    with pytest.raises(ValueError, match="bfloat16"):
        Model(config_from_dict(cfg).plan(), dtype="float32", device=DEV, weight_format="fp8")
    monkeypatch.delattr(AttentionMixer, "hold_in_8_bits")
    monkeypatch.delattr(SwiGLU, "hold_in_8_bits")
    with pytest.raises(ValueError, match="no part"):
        runner_for(cfg, w, 4, 64)
