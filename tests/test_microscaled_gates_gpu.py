"""Gated microscaled products of few rows at the borders between two codes and two scales: gate and up values that are exact in float32, whose
activation comes out within 2^-21 of a border, so that float32 falls to either side and 64 bits say to which."""
import pytest
import torch

from test_microscaling_gpu import held, middle, scales

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64, F32 = torch.float64, torch.float32
#: gate values are whole multiples of 2^-11 (12 bits), up values of 2^-12 (16 bits): digits of 16, one a block of 32
G_BITS, U_BITS, G_DIGITS, U_DIGITS = 11, 12, 3, 4


def ops():
    from litellmengine_b200.csrc import ops as o
    return o


def pairs_at_borders(g, count, borders, act, limit):
    """`count` pairs (gate, up) in float64, of many drawn those whose activation is nearest to one of the borders; which border that is."""
    n = 4000 * count
    whole = torch.randint(1 << 9, 1 << 12, (n,), generator=g, device=DEV)          # gates of 0.25 to 2
    gate = whole.to(F64) * 2.0 ** -G_BITS * torch.where(torch.rand(n, generator=g, device=DEV) < 0.5, 1.0, -1.0)
    want = borders[torch.randint(len(borders), (n,), generator=g, device=DEV)]
    one = middle(gate, torch.zeros_like(gate), act, limit) if act == 2 else middle(gate, torch.ones_like(gate), act, limit)      # what multiplies up (+ 1)
    up = torch.round((want / one - (1 if act == 2 else 0)) * 2.0 ** U_BITS).clamp(1 - 2 ** 16, 2 ** 16 - 1) * 2.0 ** -U_BITS
    made = middle(gate, up, act, limit)
    far = (made / want - 1).abs()
    # nearer than 2^-44 is left out: the oracle's own exp
    best = torch.argsort(torch.where(far > 2.0 ** -44, far, 1.0))[:count]
    return gate[best], up[best], far[best]


def pairs_beside(border, above, act, limit):
    """The sixteen pairs, of one for every gate, whose activation is nearest to the border from above or below."""
    gate = torch.arange(1 << 9, 1 << 12, dtype=F64, device=DEV) * 2.0 ** -G_BITS
    gate = torch.cat([gate, -gate])
    one = middle(gate, torch.zeros_like(gate), act, limit) if act == 2 else middle(gate, torch.ones_like(gate), act, limit)
    up = (border / one - (1 if act == 2 else 0)) * 2.0 ** U_BITS
    up = torch.cat([torch.floor(up), torch.ceil(up)]) * 2.0 ** -U_BITS
    gate = torch.cat([gate, gate])
    far = middle(gate, up, act, limit) / border - 1
    far = torch.where(up.abs() < 16, far if above else -far, -1.0)
    best = torch.argsort(torch.where(far > 2.0 ** -44, far, 1.0))[:16]
    assert float(far[best].max()) < 2.0 ** -20
    return gate[best], up[best]


def rows_of(gate, up):
    """[T, 32] pairs -> the matrix [T, blocks * 32] whose products with `weights_of` are them: digit i of feature j in block i, column j."""
    blocks = []
    for v, bits, digits in ((gate, G_BITS, G_DIGITS), (up, U_BITS, U_DIGITS)):
        whole, sign = (v.abs() * 2.0 ** bits).to(torch.int64), torch.sign(v)
        blocks += [((whole >> (4 * i)) & 15).to(F64) * 2.0 ** (4 * i - bits) * sign for i in range(digits)]
    return torch.cat(blocks, dim=1).to(F32)


def weights_of():
    one, none = torch.eye(32, device=DEV), torch.zeros(32, 32, device=DEV)
    gate = torch.cat([one] * G_DIGITS + [none] * U_DIGITS, dim=1)
    up = torch.cat([none] * G_DIGITS + [one] * U_DIGITS, dim=1)
    return gate, up


def check(gate, up, activation, limit):
    """Every code of act(gate) * up is the nearest to the exact value, for gate and up [T, 32] as sums of a product."""
    o = ops()
    x = rows_of(gate, up)
    w_gate, w_up = weights_of()
    both = torch.cat([w_gate, w_up])
    X, W, plain = o.mx_rows(x), o.mx_weight(both, gated=True), o.mx_weight(both)
    assert torch.equal(X.values(F32), x)                          # digits of 16 at powers of two: nothing is rounded
    sums = o.linear_mx(X, plain).to(F64)
    assert torch.equal(sums[:, :32], gate) and torch.equal(sums[:, 32:], up)
    want = held(middle(gate, up, o.ACTIVATIONS[activation], limit), 8)
    got = o.linear_silu_mul_mx(X, W, activation=activation, limit=limit).values(F32).to(F64)
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("T", [1, 7, 16, 17, 32, 40, 64])
@pytest.mark.parametrize("activation,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("clamped_swish", 1000.0)])
def test_gates_at_borders_between_codes(T, activation, limit):
    o = ops()
    g, act = torch.Generator(device=DEV).manual_seed(T + len(activation)), o.ACTIVATIONS[activation]
    # the block's largest value, near 448 * 2^-9 = 0.875, is on one side or the other of the border between two scales; the rest are ties of e4m3 at
    # that scale, from its lowest normal value on (and, where the next scale is taken, of the one below, which are ties there too)
    ties = torch.tensor([(8 + m + 0.5) / 8 * 2.0 ** (e - 9) for m in range(8) for e in range(-5, 8)], dtype=F64, device=DEV)
    gate, up, far = pairs_at_borders(g, 31 * T, ties, act, limit)
    order = torch.randperm(31 * T, generator=g, device=DEV)
    top_gate, top_up, top_far = pairs_at_borders(g, T, torch.tensor([0.875], dtype=F64, device=DEV), act, limit)
    gate, up = (torch.cat([a[:, None], b[order].view(T, 31)], dim=1) for a, b in ((top_gate, gate), (top_up, up)))
    assert float(torch.cat([far, top_far]).max()) < 2.0 ** -21
    check(gate, up, activation, limit)
    single = middle(gate.to(F32), up.to(F32), act, limit)
    if T >= 16:                                                   # in float32 these come out differently: the test is one of what is carried beyond it
        assert not torch.equal(held(single, 8), held(middle(gate, up, act, limit), 8))
    # the same with largest values on both sides of that border in turn
    rows, sides = torch.arange(T, device=DEV), [pairs_beside(0.875, above, act, limit) for above in (False, True)]
    for n, v in enumerate((gate, up)):
        v[:, 0] = torch.where(rows % 2 == 0, sides[0][n][rows % 16], sides[1][n][rows % 16])
    if T > 1:
        assert len(torch.unique(scales(middle(gate, up, act, limit), 8))) == 2
    check(gate, up, activation, limit)
