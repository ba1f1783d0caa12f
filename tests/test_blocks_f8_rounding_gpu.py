"""Where products of 8 bits round: results of routed experts once, whatever way their rows take; rows made of gate and up values to the nearest code of the float32 values."""
import pytest
import torch

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


#: picks as they are (up to 4 tokens), and sorted into items of 16, 128 and 256 rows; results of whole, aligned pieces of eight values, of four, and of any size
ROUNDED_ONCE = [(1, 64, 8, 64, 128), (4, 8, 2, 72, 136), (4, 8, 2, 130, 131), (2, 12, 9, 64, 128), (5, 64, 8, 64, 128), (17, 8, 2, 192, 520), (48, 64, 8, 128, 256),
                (130, 3, 1, 200, 393), (301, 8, 2, 450, 358), (600, 5, 5, 256, 640), (90, 2, 2, 64, 12), (2000, 2, 1, 257, 515),
                (2000, 2, 1, 256, 512), (900, 3, 3, 130, 264)]


@pytest.mark.parametrize("T,E,top,ff,W", ROUNDED_ONCE)
def test_a_bfloat16_result_of_experts_is_the_float32_one_rounded_once(T, E, top, ff, W):
    o, g = ops(), gen(T + E + ff)
    G, D = o.f8_weight(normal(g, E, 2 * ff, W, dtype=BF16) * W ** -0.5, gated=True), o.f8_weight(normal(g, E, W, ff, dtype=BF16) * ff ** -0.5)
    x, weights, base = normal(g, T, W, dtype=BF16), torch.rand(T, top, generator=g, device=DEV), normal(g, T, W)
    ids = torch.randint(-1, E + 1, (T, top), generator=g, device=DEV, dtype=torch.int32)
    for rows in (x, x.float()):
        for add in (None, base):
            want = o.moe_f8(rows, G, D, ids, weights, base=add)
            got = o.moe_f8(rows, G, D, ids, weights, base=add, out_dtype=BF16)
            assert got.dtype == BF16 and torch.equal(got, want.to(BF16))


def nearly_middles(g, N, K):
    """A gated weight and the column that rows of one value pick: quotients of its gate and up values, 448 * 256 the largest product, lie on middles between two
    codes (12 x 14, 10 x 10 and 12 x 9 among the mantissas' products) or, by the roundings of float32, a hair beside them."""
    codes = torch.tensor([m / 8 * 2.0 ** e for e in range(5, 9) for m in range(8, 16) if m / 8 * 2.0 ** e <= 448], device=DEV)
    pick = lambda most: codes[codes <= most][torch.randint(0, int((codes <= most).sum()), (N,), generator=g, device=DEV)]
    w = torch.zeros(2 * N, K, device=DEV)
    w[:N, 0], w[N:, 0] = pick(448), pick(256) * torch.where(torch.rand(N, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    w[N:, 0] *= torch.exp2(-torch.randint(0, 17, (N,), generator=g, device=DEV).float() * (torch.rand(N, generator=g, device=DEV) < 0.3))      # down to the lowest codes
    w[:N][::128, 0], w[N:][::128, 0] = 448.0, 256.0               # every 128 of the result's features have the largest product
    w[:, 1] = 448.0                                               # every block of the weight has the scale's largest; the rows are zero there
    return w * 1.37


@pytest.mark.parametrize("T,N,K", [(1, 256, 128), (4, 200, 128), (5, 256, 256), (16, 200, 200), (30, 640, 128), (50, 256, 128), (64, 200, 130), (100, 9728, 128), (100, 9700, 128),
                                   (1000, 9728, 128), (1000, 9700, 136)])
def test_codes_of_gate_and_up(T, N, K):
    """Gates so large that their sigmoid is one: gate times up in float32 is what the codes and scales are of.  In tiles of up to 64 rows as `f8_rows` makes them of
    a matrix; in those of 128 and 256 the nearest to the quotient as float32 has it."""
    o, g = ops(), gen(T + N)
    w = nearly_middles(g, N, K)
    x = torch.zeros(T, K, device=DEV, dtype=BF16)
    x[:, 0] = (1 + torch.rand(T, generator=g, device=DEV)).to(BF16)
    y = o.linear_f8(x, o.f8_weight(w))                            # one tile of K has numbers: no sums that another order would change
    assert float(y[:, :N].min()) > 32
    v = y[:, :N] * y[:, N:]
    made, tiles = o.f8_rows(v), (N + 127) // 128
    want = made.codes[:, :T]
    if T > 64:
        b = torch.nn.functional.pad(v, (0, -N % 128)).view(T, tiles, 128)
        most = b.abs().amax(dim=2, keepdim=True)
        want = (b * (torch.full_like(most, 448.0) / most)).to(torch.float8_e4m3fn).view(torch.uint8).transpose(0, 1)
    W = o.f8_weight(w, gated=True)
    for rows in (x, o.f8_rows(x)):
        got = o.linear_silu_mul_f8(rows, W)
        assert torch.equal(got.scales[:T, :tiles], made.scales[:T, :tiles])
        wrong = int((got.codes[:, :T] != want).sum())
        assert wrong == 0, f"{wrong} of {T * N} codes"


def test_codes_of_experts_items():
    """The same rows through a stack of one expert, whose items of 16 rows are settled too: the down product of an identity gives the codes' values back."""
    o, g = ops(), gen(9)
    N = 128
    w = nearly_middles(g, N, 128)
    D = o.f8_weight(torch.eye(N, device=DEV)[None])
    for T in (3, 6, 16):
        x = torch.zeros(T, 128, device=DEV, dtype=BF16)
        x[:, 0] = (1 + torch.rand(T, generator=g, device=DEV)).to(BF16)
        y = o.linear_f8(x, o.f8_weight(w))
        ids, weights = torch.zeros(T, 1, dtype=torch.int32, device=DEV), torch.ones(T, 1, device=DEV)
        want = o.linear_f8(o.f8_rows(y[:, :N] * y[:, N:]), o.f8_weight(torch.eye(N, device=DEV)))
        for rows in (x, x.float()):
            assert torch.equal(o.moe_f8(rows, o.f8_weight(w[None], gated=True), D, ids, weights), want)


def test_float32_values_a_hair_beside_every_middle():
    """Blocks of every order of magnitude and any largest value, with values at, and up to three of float32's steps beside, each middle between two codes."""
    from test_blocks_f8_gpu import held, same
    o, g = ops(), gen(11)
    codes = [m * 2.0 ** -9 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if e < 8 or m < 7]
    middles = torch.tensor([(a + b) / 2 for a, b in zip(codes, codes[1:])], dtype=torch.float64, device=DEV)
    assert len(middles) == 126
    low = torch.tensor([2.0 ** -126, 448 * 2.0 ** -126, 449 * 2.0 ** -126], device=DEV)
    top = torch.cat([(1 + torch.rand(4000, generator=g, device=DEV)) * torch.exp2(torch.randint(-117, 128, (4000,), generator=g, device=DEV).float()), low,
                     torch.nextafter(low, low * 2), torch.nextafter(low, low * 0), torch.tensor([3.4028234e38, 1.0, 448.0], device=DEV)])
    rows = (middles * top.to(torch.float64)[:, None] / 448).to(F32)
    rows = (rows.view(torch.int32) + torch.randint(-3, 4, rows.shape, generator=g, device=DEV, dtype=torch.int32)).clamp(min=0).view(F32)
    rows = torch.minimum(rows, top[:, None]) * torch.where(torch.rand(rows.shape, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    x = torch.cat([top[:, None], rows, -top[:, None]], dim=1)
    assert x.shape[1] == 128
    assert same(o.f8_rows(x).values(F32), held(x, 1))
