"""Where products of 8 bits round: results of routed experts once, whatever way their rows take."""
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
                (130, 3, 1, 200, 393), (301, 8, 2, 450, 358), (600, 5, 5, 256, 640), (90, 2, 2, 64, 12), (2000, 2, 1, 257, 515)]


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
