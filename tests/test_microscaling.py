"""Refusals of the microscaled operators, which need no device."""
import ctypes

import pytest
import torch

from litellmengine_b200.csrc import build, ops


def refuses(call, *a, **k):
    with pytest.raises(ops.KernelError):
        call(*a, **k)


def test_tensors_that_are_on_no_device():
    x, w = torch.zeros(4, 64), torch.ones(64)
    refuses(ops.mx_rows, x)
    refuses(ops.mx_weight, x)
    refuses(ops.mx_weight, x, gated=True)
    refuses(ops.rmsnorm_mx, x, w, 1e-6)
    refuses(ops.rmsnorm_mx, x, w, 1e-6, delta=x, sum_out=x)
    refuses(ops.silu_and_mul_mx, x)
    refuses(ops.linear_mx, x, w)
    refuses(ops.linear_silu_mul_mx, x, torch.zeros(8, 64))


def lib(family):
    return ctypes.CDLL(build.ensure_built(family))


P, SIZE, DTYPE, ALIGN = 4096, -1, -2, -3          # an aligned address that nothing reads: every call below is refused before its launch


def test_sizes_types_and_addresses_of_rows():
    m, f, ll = lib("microscaling"), ctypes.c_float, ctypes.c_longlong
    v = ctypes.c_void_p
    rows = lambda dt=1, r=P, T=4, K=64: m.llm_mx_rows(v(P), dt, v(r), T, K, v(0))
    assert rows(T=0) == 0 and rows(K=0) == SIZE and rows(K=(1 << 20) + 1) == SIZE and rows(r=P + 8) == ALIGN and rows(dt=2) == DTYPE
    weight = lambda dt=1, t=P, s=P, N=4, K=64: m.llm_mx_weight(v(P), dt, v(t), v(s), N, K, 0, v(0))
    assert weight(N=0) == SIZE and weight(K=0) == SIZE and weight(N=(1 << 24) + 1) == SIZE and weight(dt=3) == DTYPE and weight(t=P + 1) == ALIGN
    norm = lambda dt=0, parts=1, H=64, sum_out=0, rws=0, r=P: m.llm_mx_rmsnorm(v(P), dt, v(P), 0, parts, ll(0), v(P), f(1e-6), v(sum_out), v(r), v(rws), 4, H, v(0))
    assert norm(H=0) == SIZE and norm(parts=0) == SIZE and norm(sum_out=P, rws=P) == SIZE and norm(dt=2) == DTYPE and norm(r=P + 2) == ALIGN and norm(H=32769) == SIZE
    act = lambda dt=1, parts=1, inter=64, kind=0, limit=0.0, r=P: m.llm_mx_silu_and_mul(v(P), dt, parts, ll(0), v(r), 4, inter, kind, f(limit), v(0))
    assert act(inter=0) == SIZE and act(kind=3) == SIZE and act(kind=2) == SIZE and act(parts=0) == SIZE and act(dt=5) == DTYPE and act(r=P + 8) == ALIGN
    values = lambda fmt=8, dt=1, gated=0, K=64: m.llm_mx_values(v(P), v(P), fmt, v(P), dt, 4, K, gated, v(0))
    assert values(fmt=6) == SIZE and values(gated=1) == SIZE and values(dt=2) == DTYPE and values(K=0) == SIZE
    assert [m.llm_mx_weight_tiles(n, g) for n, g in ((1, 0), (128, 0), (129, 0), (1, 1), (128, 1), (129, 1))] == [2, 2, 2, 2, 2, 4]


def test_sizes_types_and_addresses_of_products():
    m, f = lib("microscaling"), ctypes.c_float
    v = ctypes.c_void_p
    y = lambda x=P, plain=0, xd=1, w=P, dt=0, add=0, T=4, N=64, K=64, status=P: m.llm_linear_mx(v(x), v(plain), xd, v(w), v(P), v(P), dt, add, T, N, K, 1, v(status), v(0))
    assert y(T=0) == 0 and y(N=0) == SIZE and y(K=0) == SIZE and y(K=(1 << 20) + 1) == SIZE and y(T=(1 << 24) + 1) == SIZE
    assert y(x=P + 8) == ALIGN and y(w=P + 16) == ALIGN and y(status=0) == ALIGN and y(dt=2) == DTYPE and y(dt=1, add=1) == DTYPE and y(plain=P, xd=2) == DTYPE
    g = lambda kind=0, limit=0.0, T=4, N=64, made=P: m.llm_linear_mx_silu_mul(v(P), v(0), 0, v(P), v(P), v(made), T, N, 64, kind, f(limit), 1, v(P), v(0))
    assert g(T=0) == 0 and g(N=0) == SIZE and g(kind=3) == SIZE and g(kind=2) == SIZE and g(kind=-1) == SIZE and g(made=P + 8) == ALIGN
    assert y(x=0) == ALIGN and y(x=0, plain=P, T=17) == ALIGN 
    takes = lambda T=16, dt=1, K=64, at=P: m.llm_linear_mx_takes(v(at), dt, T, K)
    assert takes(T=ops.MX_PLAIN_ROWS) and not takes(T=ops.MX_PLAIN_ROWS + 1) and not takes(dt=0) and not takes(K=36) and not takes(at=P + 8)
    assert [ops.mx_padded_rows(t) for t in (1, 16, 17, 33, 65, 128, 129, 384, 385)] == [16, 16, 32, 64, 128, 128, 384, 384, 768]


def test_matrices_are_held_in_4_bits_by_parts_that_say_so_of_their_own_forward(monkeypatch):
    """A part that derives from one with `hold_in_4_bits` and has a forward of its own keeps its matrices, unless it says so again."""
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
        def hold_in_4_bits(self):
            return super().hold_in_4_bits()

    monkeypatch.setattr(ops, "mx_weight", lambda w, gated=False: ("4 bits", gated))
    w = {n: t.to(torch.bfloat16) if t.dim() == 2 else t for n, t in tm.make_weights(tm.TINY_A, 0, bf16_exact=True).items()}
    kind = next(k for k, c in registry._KINDS["feed_forward"].items() if c is SwiGLU)
    for cls, held in ((SwiGLU, True), (Own, False), (Again, True)):
        monkeypatch.setitem(registry._KINDS["feed_forward"], kind, cls)
        model = Model(config_from_dict(tm.TINY_A).plan(), device="cpu", weight_format="mxfp4")
        model.load_weights(DictSource(w))
        for block in model.blocks:
            assert block.mixer.w_qkv == ("4 bits", False) and type(block.feed_forward) is cls
            assert isinstance(block.feed_forward.w_down, tuple) == held and isinstance(block.feed_forward.w_gate_up, tuple) == held


def test_a_residual_that_the_product_does_not_take_is_declined():
    """As with stored weights: False, and nothing done, for a residual that is not float32, not contiguous or of another shape."""
    W = ops.MxWeight(32, 64, False, torch.device("cpu"))
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for residual in (torch.ones(4, 32, dtype=torch.bfloat16), torch.ones(4, 32, dtype=torch.float64), torch.ones(32, 4).t(), torch.ones(4, 64)[:, ::2], torch.ones(4, 31),
                     torch.ones(5, 32), torch.ones(128)):
        assert ops.linear_into(x, W, residual) is False and bool((residual == 1).all())
    refuses(ops.linear_into, x, W, torch.ones(4, 32))             # one that it takes: no device here
