"""Low-rank adapters of many requests (``tensorfold_b200.adapters``; ``qmm`` and ``Exl3Linear`` with ``adapters=``): against
64-bit products, exact integers, rows alone, odd sizes, rows without an adapter, special values, streams and graphs."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32

# (type, rows, inputs, columns, adapters, rank): both sides of the sorted form's least rows, inputs of a part of a warp's
# run and of several, columns of a part of eight and of a warp's 32, every build of the rank
CASES = [(BF, 1, 64, 32, 1, 8), (BF, 1, 2048, 333, 4, 16), (HF, 3, 200, 40, 5, 24), (BF, 64, 1032, 257, 7, 64),
         (HF, 65, 8, 1, 3, 1), (BF, 96, 520, 96, 3, 16), (BF, 97, 520, 96, 3, 16), (BF, 200, 2056, 130, 2, 33), (HF, 500, 328, 1000, 40, 128),
         (BF, 130, 4104, 64, 1, 100), (HF, 77, 4096, 48, 9, 5)]
IDS = [f"{'bf16' if c[0] == BF else 'fp16'}-m{c[1]}-k{c[2]}-n{c[3]}-i{c[4]}-r{c[5]}" for c in CASES]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(seed, *shape, scale=1.0, dtype=BF):
    return (torch.randn(shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def whole(seed, *shape, most=2, dtype=BF):
    return torch.randint(-most, most + 1, shape, generator=gen(seed), device=DEV).to(dtype)


def ids_of(rows, count, seed=3):
    ids = torch.randint(-1, count + 1, (rows,), generator=torch.Generator().manual_seed(seed))   # -1 and count: none
    if rows == 1:
        ids[0] = count - 1
    return ids.to(torch.int32).to(DEV)


def build(case, seed=11, make=normal):
    from tensorfold_b200 import adapters

    dtype, _, k, n, count, rank = case
    if make is whole:
        a, b, scale = whole(seed, count, rank, k, dtype=dtype), whole(seed + 1, count, n, rank, dtype=dtype), 2.0
    else:
        a, b = normal(seed, count, rank, k, scale=k ** -0.5, dtype=dtype), normal(seed + 1, count, n, rank, scale=0.3, dtype=dtype)
        scale = torch.rand((count,), generator=gen(seed), device=DEV) + 0.5
    return adapters.make(a, b, scale)


def plan_of(ids, count):
    from tensorfold_b200 import adapters

    plan = adapters.Plan(max(1, ids.shape[0]), count, DEV)
    adapters.route(ids, plan)
    return plan


def reference(x, ad, ids, base, out_type):
    """The formula in 64 bits, and how far the kernel's rows may be: the low-rank sums are off by at most K truncated fp32
    steps of 2^-23 of the sum of magnitudes, and one for the scale; they are split into two parts of t bits each with a
    rest below half a step of the second, after scaling the row's largest value into [1, 2): 2^-16 (bf16: 8 + 8 bits; with a
    third part under fp32 rows 2^-24) of a value, or for fp16 2^-22 of it or, where the second part is below fp16's normal
    range, 2^-25 of the row's largest; the columns' sums add 3 R steps, the base one; then one rounding of half a step."""

    want, room = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64, device=DEV)
    k, rank = ad.k, ad.a.shape[1]
    for m, i in enumerate(ids.tolist()):
        if not 0 <= i < ad.count:
            continue
        a, b, sc = ad.a[i].double(), ad.b[i].double(), ad.scale[i].double()
        s, mag = sc * (a @ x[m].double()), sc.abs() * (a.abs() @ x[m].double().abs())
        es = mag * (k + 1) * 2.0 ** -23
        es = es + (s.abs() * 2.0 ** (-24 if out_type == F32 else -16) if ad.dtype == BF else s.abs() * 2.0 ** -22 + s.abs().max() * 2.0 ** -25)
        delta = b @ s
        want[m] += delta
        parts = b.abs() @ (s.abs() + es)
        room[m] = (b.abs() @ es + parts * 3 * rank * 2.0 ** -23 + want[m].abs() * 2.0 ** -24) * 1.01
    if out_type != F32:
        room = room + want.abs() * torch.finfo(out_type).eps / 2 + 2.0 ** -25
    return want, room


@pytest.mark.parametrize("base_type,out_type", [(F32, F32), (F32, None), (None, None)], ids=["f32-f32", "f32-16", "16-16"])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_against_64_bits(case, base_type, out_type, pdl):
    from tensorfold_b200 import adapters

    dtype, rows, k, n, count, _ = case
    ad, ids = build(case), ids_of(rows, count)
    x, base = normal(5, rows, k, dtype=dtype), normal(6, rows, n, dtype=base_type or dtype)
    plan = plan_of(ids, count)
    got = adapters.add(x, ad, plan, base, dtype=out_type or dtype)
    want, room = reference(x, ad, ids, base, out_type or dtype)
    assert got.dtype == (out_type or dtype) and ((got.double() - want).abs() <= room).all()
    none = (ids < 0) | (ids >= count)
    assert torch.equal(got[none], base[none].to(got.dtype))
    if base.dtype == got.dtype:                                        # in place: the same bits
        assert adapters.add(x, ad, plan, base, base) is base and torch.equal(base, got)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_whole_numbers_come_out_exactly(case):
    from tensorfold_b200 import adapters

    dtype, rows, k, n, count, _ = case
    ad, ids = build(case, make=whole), ids_of(rows, count)
    x, base = whole(5, rows, k, most=1, dtype=dtype), whole(6, rows, n, most=100, dtype=F32)
    got = adapters.add(x, ad, plan_of(ids, count), base)
    want, _ = reference(x, ad, ids, base, F32)
    # the low-rank sums are below 2^14 (4104 inputs of magnitude 2, doubled), so that two parts of eight bits hold them
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_a_row_does_not_depend_on_the_call(case):
    """Rows alone, a few together and in another order; padded ranks; the same bits."""

    from tensorfold_b200 import adapters

    dtype, rows, k, n, count, rank = case
    ad, ids = build(case, 21), ids_of(rows, count, 7)
    x, base = normal(8, rows, k, dtype=dtype), normal(9, rows, n, dtype=F32)
    got = adapters.add(x, ad, plan_of(ids, count), base)
    for lo, hi in {(0, 1), (rows // 2, rows // 2 + 1), (0, min(rows, 64)), (rows - 1, rows)}:
        part = adapters.add(x[lo:hi], ad, plan_of(ids[lo:hi].clone(), count), base[lo:hi])
        assert torch.equal(part, got[lo:hi]), (lo, hi)
    perm = torch.randperm(rows, generator=torch.Generator().manual_seed(2)).to(DEV)
    again = adapters.add(x[perm].contiguous(), ad, plan_of(ids[perm].contiguous(), count), base[perm].contiguous())
    assert torch.equal(again, got[perm])
    many = torch.cat([ids, ids])
    twice = adapters.add(torch.cat([x, x]), ad, plan_of(many, count), torch.cat([base, base]))
    assert torch.equal(twice, torch.cat([got, got]))


def test_many_rows_of_one_adapter_and_of_none():
    from tensorfold_b200 import adapters

    case = (BF, 1000, 264, 200, 3, 16)
    ad, x, base = build(case, 31), normal(1, 1000, 264), normal(2, 1000, 200, dtype=F32)
    for ids in (torch.full((1000,), 1), torch.full((1000,), -7), torch.arange(1000) // 700 - 1):
        ids = ids.to(torch.int32).to(DEV)
        got = adapters.add(x, ad, plan_of(ids, 3), base, dtype=BF)
        want, room = reference(x, ad, ids, base, BF)
        assert ((got.double() - want).abs() <= room).all()


@pytest.mark.parametrize("rows", [5, 120])
def test_strides_and_alignments(rows):
    """Strided rows of x, base and out at any alignment; what lies between the rows of out stays."""

    from tensorfold_b200 import adapters

    case = (HF, rows, 136, 75, 4, 16)
    ad, ids = build(case, 41), ids_of(rows, 4)
    plan = plan_of(ids, 4)
    for pad in (0, 1, 4, 5, 8):
        x = normal(1, rows, 136 + 2 * pad, dtype=HF)[:, pad:pad + 136]
        wide_b, wide_o = normal(2, rows, 75 + pad, dtype=HF), torch.full((rows, 75 + 2 * pad), 9.0, dtype=HF, device=DEV)
        base, out = wide_b[:, :75], wide_o[:, pad:pad + 75]
        assert adapters.add(x, ad, plan, base, out) is out
        assert torch.equal(out, adapters.add(x.contiguous(), ad, plan, base.contiguous()))
        assert (wide_o[:, :pad] == 9).all() and (wide_o[:, pad + 75:] == 9).all()


@pytest.mark.parametrize("rows", [6, 99])
def test_special_values_stay_in_their_rows(rows):
    """NaN and infinities in one row's inputs or in one adapter; rows far apart in size; tiny and huge low-rank values."""

    from tensorfold_b200 import adapters

    case = (HF, rows, 128, 64, 3, 16)
    ad = build(case, 51)
    ids = (torch.arange(rows) % 3).to(torch.int32).to(DEV)
    x, base = normal(1, rows, 128, dtype=HF), torch.zeros((rows, 64), device=DEV)
    plan = plan_of(ids, 3)
    got = adapters.add(x, ad, plan, base)
    bad = x.clone()
    bad[3, 5], bad[4, 6] = float("nan"), float("inf")
    out = adapters.add(bad, ad, plan, base)
    keep = torch.tensor([i not in (3, 4) for i in range(rows)], device=DEV)
    assert torch.equal(out[keep], got[keep]) and not torch.isfinite(out[3:5]).any()
    # powers of two through the scale alone: the low-rank values leave fp16's range at both ends, their rows scale exactly
    for power in (-60, -20, 16, 40):
        ad.scale.mul_(2.0 ** power)
        assert torch.equal(adapters.add(x, ad, plan, base), got * 2.0 ** power), power
        ad.scale.mul_(2.0 ** -power)
    ad.a[1, 2, 7] = float("nan")
    out = adapters.add(x, ad, plan, base)
    assert torch.isnan(out[ids == 1]).all() and torch.equal(out[ids != 1], got[ids != 1])
    ad.clear(1)
    assert torch.equal(adapters.add(x, ad, plan, base + 1)[ids == 1], (base + 1)[ids == 1])


def test_slots_are_replaced_between_calls(pdl):
    """A slot filled again in front of a call: the call sees the new adapter, of another rank."""

    from tensorfold_b200 import adapters

    case = (BF, 40, 256, 128, 4, 32)
    ad, x, base = build(case, 61), normal(1, 40, 256), normal(2, 40, 128, dtype=F32)
    ids = (torch.arange(40) % 4).to(torch.int32).to(DEV)
    plan = plan_of(ids, 4)
    got = []
    for turn in range(4):
        ad.put(2, normal(70 + turn, 8 * turn + 3, 256, scale=0.1), normal(80 + turn, 128, 8 * turn + 3), 0.5)
        got.append((adapters.add(x, ad, plan, base), ad.a.clone(), ad.b.clone(), ad.scale.clone()))
    for out, a, b, scale in got:
        assert torch.equal(out, adapters.add(x, adapters.make(a, b, scale), plan, base))


@pytest.mark.parametrize("rows", [16, 300])
def test_graph_replays_follow_the_ids_on_their_own_plans(rows):
    """Two captured calls with plans of their own, on another stream: replays follow the ids and the rows."""

    from tensorfold_b200 import adapters

    stream, held = torch.cuda.Stream(), []
    for i, (k, n) in enumerate(((256, 96), (512, 200))):
        ad = build((BF, rows, k, n, 6, 16), 91 + i)
        x, base, ids = normal(1, rows, k), normal(2, rows, n, dtype=F32), ids_of(rows, 6, i)
        plan, out = adapters.Plan(rows, 6, DEV), torch.empty((rows, n), dtype=BF, device=DEV)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            adapters.route(ids, plan)
            adapters.add(x, ad, plan, base, out)
        held.append((ad, x, base, ids, plan, out, graph, k))
    for turn in range(3):
        for ad, x, base, ids, plan, out, graph, k in held:
            x.copy_(normal(100 + turn, rows, k))
            ids.copy_(ids_of(rows, 6, 20 + turn))
            graph.replay()
            got = out.clone()
            assert torch.equal(got, adapters.add(x, ad, plan_of(ids.clone(), 6), base, dtype=BF))


@pytest.mark.parametrize("rows", [1, 45, 300])
def test_beside_a_4_bit_projection(rows, pdl):
    """``qmm.matmul`` and ``prefill_matmul`` with adapters: the fp32 product with each row's adapter, rounded once."""

    from tensorfold_b200 import adapters, qmm
    from test_qmm_gpu import mlx

    q = qmm.pack(*mlx(200, 512, 7), 64)                                # 200 columns: a padded projection
    ad = build((BF, rows, 512, 200, 5, 16), 17)
    x, ids = normal(1, rows, 512), ids_of(rows, 5)
    plan = plan_of(ids, 5)
    for product in (qmm.matmul, qmm.prefill_matmul):
        base = product(x, q, f32=True)
        for f32 in (False, True):
            want = adapters.add(x, ad, plan, base, dtype=F32 if f32 else BF)
            assert torch.equal(product(x, q, f32=f32, adapters=ad, plan=plan), want)
            out = torch.empty_like(want)
            assert product(x, q, f32=f32, adapters=ad, plan=plan, out=out) is out and torch.equal(out, want)
    with pytest.raises(ValueError, match="whole product"):
        qmm.matmul(x, q, reduce=False, adapters=ad, plan=plan)
    with pytest.raises(ValueError, match="takes the plan"):
        qmm.matmul(x, q, adapters=ad)
    with pytest.raises(ValueError, match="beside a projection"):
        qmm.matmul(x, q, adapters=build((BF, rows, 512, 192, 5, 16)), plan=plan)
    with pytest.raises(ValueError, match="comes first"):
        qmm.matmul(x, q, adapters=ad, plan=adapters.Plan(rows, 5, DEV))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_beside_an_exl3_projection(dtype):
    from tensorfold_b200 import adapters, synthetic
    from tensorfold_b200.exl3.linear import Exl3Linear

    layer = Exl3Linear.from_tensors(*synthetic.exl3_matrix(3, 256, 384, 4), "3inst", normal(4, 384, dtype=HF))
    ad = build((dtype, 20, 256, 384, 5, 16), 17)
    x, ids = normal(1, 20, 256, dtype=dtype), ids_of(20, 5)
    plan = plan_of(ids, 5)
    want = adapters.add(x, ad, plan, layer(x, out_dtype=F32), dtype=dtype)
    assert torch.equal(layer(x, adapters=ad, plan=plan), want)
    out = torch.empty_like(want)
    assert layer(x, out, adapters=ad, plan=plan) is out and torch.equal(out, want)
    with pytest.raises(ValueError, match="takes the plan"):
        layer(x, adapters=ad)


def test_the_layer_of_a_step():
    """The set as a program runs it: a 4-bit projection with the batch's adapters, whose rows then route to 16-bit
    experts; one plan of the ids for the step, everything in one graph."""

    from tensorfold_b200 import adapters, experts16, moe, qmm
    from test_qmm_gpu import dequant64, mlx

    rows = 24
    words = mlx(256, 512, 9)
    q, ad = qmm.pack(*words, 64), build((BF, rows, 512, 256, 6, 16), 19)
    up = [normal(20 + i, 8, 128, 256, scale=0.1) for i in range(2)]
    down = normal(25, 8, 256, 128, scale=0.1)
    layer = moe.Routed(normal(26, 8, 256, scale=0.05), experts16.make(up, down), 2, shared=False)
    x, ids = normal(27, rows, 512), ids_of(rows, 6)
    plan, buf = adapters.Plan(rows, 6, DEV), moe.MoEBuffers(rows, moe._Shape(layer), DEV, shared=False, dtype=BF)
    h, out = torch.empty((rows, 256), dtype=BF, device=DEV), torch.empty((rows, 256), dtype=BF, device=DEV)

    def step():
        adapters.route(ids, plan)
        qmm.matmul(x, q, adapters=ad, plan=plan, out=h)
        moe.layer(h, layer, buf, out)

    step()
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    x.copy_(normal(28, rows, 512))
    ids.copy_(ids_of(rows, 6, 5))
    graph.replay()
    base = (x.double() @ dequant64(*words).t())
    want_h, room = reference(x, ad, ids, base, BF)
    # the product's own arithmetic: K steps of 2^-23 of the sum of magnitudes
    room = room + (x.double().abs() @ dequant64(*words).abs().t()) * 512 * 2.0 ** -23
    assert ((h.double() - want_h).abs() <= room).all()
    want = torch.zeros((rows, 256), dtype=torch.float64, device=DEV)
    for r in range(rows):
        for s in range(2):
            e = int(buf.pick[r, s])
            g, u = up[0][e].double() @ h[r].double(), up[1][e].double() @ h[r].double()
            want[r] += buf.wts[r, s].double() * (down[e].double() @ (g * torch.sigmoid(g) * u))
    assert (out.double() - want).norm() <= 2.0 ** -8 * want.norm()          # roundings of the activations and of the sum


def test_refusals_on_the_gpu():
    from tensorfold_b200 import adapters

    ad, ids = build((BF, 8, 64, 40, 3, 16)), ids_of(8, 3)
    plan = plan_of(ids, 3)
    x, base = normal(1, 8, 64), normal(2, 8, 40, dtype=F32)
    buf = torch.zeros((8, 80), device=DEV)
    for kw, why in (({"x": x.to(HF)}, "as the adapters"), ({"x": x[:, :56]}, "as the adapters"), ({"x": x[:7]}, "comes first"),
                    ({"base": base[:7]}, "base"), ({"base": base.double()}, "base"), ({"base": base[:, :39]}, "base"),
                    ({"base": base.cpu()}, "x's device"), ({"out": base[:, :39]}, "out"),
                    ({"base": base[:1].expand(8, 40)}, "must not overlap"),
                    ({"base": buf[:, :40], "out": buf[:, 8:48]}, "must not overlap"),
                    ({"base": base, "out": base.view(torch.bfloat16)[:, :40]}, "must not overlap"),
                    ({"out": base, "dtype": BF}, "not torch.bfloat16"), ({"plan": adapters.Plan(8, 3, DEV)}, "comes first")):
        with pytest.raises(ValueError, match=why):
            adapters.add(**{"x": x, "ad": ad, "plan": plan, "base": base, **kw})
    other = adapters.Plan(8, 4, DEV)
    adapters.route(ids, other)
    with pytest.raises(ValueError, match="a plan of 4 adapters for 3"):
        adapters.add(x, ad, other, base)
    with pytest.raises(ValueError, match="do not fit a plan"):
        adapters.route(ids_of(9, 3), plan)
    assert adapters.add(x[:0], ad, plan_of(ids[:0], 3), base[:0]).shape == (0, 40)
