"""The builds of the 16-bit experts on pairs of CTAs as they run on a prompt: several units a pair of CTAs, so that the ring of
stages and the two accumulators pass from unit to unit; and a layer's prompt form down to its fp32 rows."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16

ROWS, COUNTS = 5200, (3101, 2092, 7)                # items of 256 pairs, the last of an expert partly filled, one of 7 pairs
DIMS, WIDTH = 1800, 1032                            # 29 and 17 blocks of 64 inputs, the last partly filled; 6 or 8 stages


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def whole(seed, *shape, most=3, dtype=BF):
    return torch.randint(-most, most + 1, shape, generator=gen(seed), device=DEV).to(dtype)


def normal(seed, *shape, scale=1.0, dtype=BF):
    return (torch.randn(shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def plan_of(tile):
    from tensorfold_b200 import experts, experts16

    picks = torch.repeat_interleave(torch.arange(3), torch.tensor(COUNTS))[torch.randperm(ROWS, generator=torch.Generator().manual_seed(1))]
    plan = experts16.Plan(ROWS, 1, 3, DEV)
    plan.decode_tile = tile
    experts.route(picks.to(torch.int32).view(ROWS, 1).to(DEV), plan)
    return plan, picks.to(DEV)


def units(columns, tile):
    """Units of a launch: items times tiles of 256 weight rows."""

    return sum(-(-c // tile) for c in COUNTS) * -(-columns // 256)


@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_down_on_many_units_is_exact(dtype, tile):
    """Whole numbers, fp32 rows: sums below 1032 * 9 < 2^24, exact in any order."""

    from tensorfold_b200 import experts16

    down = whole(3, 3, DIMS, WIDTH, dtype=dtype)
    ex = experts16.make([torch.zeros((3, WIDTH, DIMS), dtype=dtype, device=DEV)], down)
    plan, picks = plan_of(tile)
    pairs_of_ctas = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert units(DIMS, tile) > 2 * pairs_of_ctas
    act, y = whole(4, ROWS, WIDTH, dtype=dtype), torch.full((ROWS, DIMS), float("nan"), device=DEV)
    experts16.down(act, ex, plan, y, ROWS)
    for e in range(3):
        assert torch.equal(y[picks == e].double(), act[picks == e].double() @ down[e].double().t()), e
    half = torch.full((ROWS, DIMS), float("nan"), dtype=dtype, device=DEV)
    experts16.down(act, ex, plan, half, ROWS)
    assert torch.equal(half, y.to(dtype))


@pytest.mark.parametrize("swiglu", [True, False], ids=["swiglu", "relu2"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gate_up_on_many_units_gives_the_small_build_s_bits(dtype, swiglu):
    """Items of 128 and 256 pairs against items of 32, each walked by one CTA; those against 64 bits, within the bound of a sum of
    K products off by a truncated fp32 step each, through the activation, and one rounding."""

    from tensorfold_b200 import experts16

    up = [normal(5 + i, 3, WIDTH, DIMS, scale=DIMS ** -0.5, dtype=dtype) for i in range(2 if swiglu else 1)]
    ex = experts16.make(up, torch.zeros((3, DIMS, WIDTH), dtype=dtype, device=DEV))
    x, got = normal(8, ROWS, DIMS, dtype=dtype), {}
    pairs_of_ctas = torch.cuda.get_device_properties(0).multi_processor_count // 2
    for tile in (32, 128, 256):
        plan, picks = plan_of(tile)
        assert tile == 32 or units(len(up) * WIDTH, tile) > pairs_of_ctas
        got[tile] = torch.full((ROWS, WIDTH), float("nan"), dtype=dtype, device=DEV)
        experts16.gate_up(x, ex, plan, got[tile], ROWS)
    assert torch.equal(got[128], got[32]) and torch.equal(got[256], got[32])
    for e in range(3):
        xe = x[picks == e].double()
        s = [(xe @ m[e].double().t(), (xe.abs() @ m[e].double().abs().t()) * DIMS * 2.0 ** -23) for m in up]
        if swiglu:
            (g, eg), (u, eu) = s
            silu = g * torch.sigmoid(g)
            want = silu * u
            room = 1.1 * u.abs() * eg + silu.abs() * eu + 1.1 * eg * eu + want.abs() * (8 + 1.2 * g.abs()) * 2.0 ** -23
        else:
            a, ea = s[0]
            want = a.clamp(min=0) ** 2
            room = 2 * a.abs() * ea + ea ** 2 + want * 2.0 ** -23
        room = room * 1.01 + want.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25
        assert ((got[32][picks == e].double() - want).abs() <= room).all(), e


@pytest.mark.parametrize("rows", [40, 700])
@pytest.mark.parametrize("prefill", [False, True])
def test_a_layer_sums_fp32_rows(prefill, rows):
    """Either form of a layer is the weighted sum of ``down``'s fp32 rows, bit for bit: nothing is rounded between."""

    from tensorfold_b200 import experts, experts16, moe

    ex = experts16.make([normal(1, 12, 128, 256, scale=0.1), normal(2, 12, 128, 256, scale=0.1)], normal(3, 12, 256, 128, scale=0.1))
    layer, x = moe.Routed(normal(4, 12, 256, scale=0.05), ex, 4, shared=False), normal(5, rows, 256)
    buf = moe.MoEBuffers(rows, moe._Shape(layer), DEV, prefill=prefill, shared=False, dtype=BF)
    out = torch.empty((rows, 256), dtype=BF, device=DEV)
    moe.layer(x, layer, buf, out)
    plan = experts16.Plan(rows, 4, 12, DEV)
    experts.route(buf.pick, plan)
    act, y = torch.empty((rows * 4, 128), dtype=BF, device=DEV), torch.empty((rows, 4, 256), device=DEV)
    experts16.gate_up(x, ex, plan, act, rows)
    experts16.down(act, ex, plan, y.view(-1, 256), rows)
    assert torch.equal(out, moe.combine(y, buf.wts)) and torch.equal(out, moe.run(x, layer, prefill=prefill))
    assert torch.equal(out, moe.picked(x, ex, buf.pick, buf.wts))
