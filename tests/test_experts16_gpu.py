"""Grouped experts on 16-bit weights (``tensorfold_b200.experts16``, ``moe.picked``): against 64-bit products, exact
integers, rows alone, plans of other items, odd sizes, masked and special values, streams and graphs."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16

# (dtype, SwiGLU, limit, experts, D, NI, slots, rows): K of one block, of a part of one, of several and a part; columns of
# a part of 16, of a part of a tile, of several tiles; experts with no pair, one, more than an item's
CASES = [
    (BF, True, 0.0, 5, 64, 64, 2, 1),
    (BF, True, 2.0, 7, 200, 136, 3, 17),
    (BF, False, 0.0, 3, 264, 40, 1, 300),
    (HF, True, 0.0, 12, 136, 328, 4, 33),
    (HF, False, 0.0, 2, 8, 8, 2, 5),
    (HF, True, 0.5, 40, 72, 24, 6, 64),
    (BF, True, 0.0, 2, 712, 200, 2, 700),
    (BF, True, 0.0, 1, 512, 256, 1, 129),
]
IDS = [f"{'bf16' if c[0] == BF else 'fp16'}-{'swiglu' if c[1] else 'relu2'}-e{c[3]}-d{c[4]}-n{c[5]}-r{c[7]}" for c in CASES]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(seed, *shape, scale=1.0, dtype=BF):
    return (torch.randn(shape, generator=gen(seed), device=DEV) * scale).to(dtype)


def whole(seed, *shape, most=3, dtype=BF):
    return torch.randint(-most, most + 1, shape, generator=gen(seed), device=DEV).to(dtype)


def picks_of(rows, slots, count, seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.stack([torch.randperm(count, generator=g)[:slots] for _ in range(rows)]).to(torch.int32).to(DEV)


def weights(case, seed=11, make=normal):
    dtype, swiglu, _, e, d, n, _, _ = case
    kw = {} if make is whole else {"scale": 0.1}
    up = [make(seed + i, e, n, d, dtype=dtype, **kw) for i in range(2 if swiglu else 1)]
    return up, make(seed + 5, e, d, n, dtype=dtype, **kw)


def run(ex, x, picks, tile=None, y_type=torch.float32):
    from tensorfold_b200 import experts, experts16

    rows, slots = picks.shape
    plan = experts16.Plan(rows, slots, ex.count, DEV)
    if tile is not None:
        plan.decode_tile = tile
    experts.route(picks, plan)
    act = torch.full((rows * slots, ex.width), 77.0, dtype=ex.dtype, device=DEV)
    y = torch.full((rows * slots, ex.dims), 77.0, dtype=y_type, device=DEV)
    experts16.gate_up(x, ex, plan, act, rows)
    experts16.down(act, ex, plan, y, rows)
    return act, y


def ref_gate_up(case, up, x, picks):
    """Activations [R * slots, NI] in 64 bits, and how far the kernel's may be: K additions of exact products, each off
    by at most a truncated fp32 step (2^-23 of the sum of magnitudes), through the activation; the fast exponential and
    division (2 + 1.2 |g| and 2 steps of 2^-23, a few more for the products); one rounding of half a step."""

    dtype, swiglu, limit, e, d, n, slots, rows = case
    pk = picks.reshape(-1).long()
    xs = x.double().repeat_interleave(picks.shape[1], 0)
    want, room = [], []
    for i in range(pk.numel()):
        s = [(m[pk[i]].double() @ xs[i], m[pk[i]].double().abs() @ xs[i].abs() * d * 2.0 ** -23) for m in up]
        if swiglu:
            (g, eg), (u, eu) = s
            if limit:
                g, u = g.clamp(max=limit), u.clamp(-limit, limit)
            silu = g * torch.sigmoid(g)
            v = silu * u
            r = 1.1 * u.abs() * eg + silu.abs() * eu + 1.1 * eg * eu + v.abs() * (8 + 1.2 * g.abs()) * 2.0 ** -23
        else:
            a, ea = s[0]
            v = a.clamp(min=0) ** 2
            r = 2 * a.abs() * ea + ea ** 2 + v * 2.0 ** -23
        want.append(v)
        room.append(r * 1.01 + v.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25)      # 2^-25: half of fp16's least step
    return torch.stack(want), torch.stack(room)


def ref_down(down, act, picks, dtype):
    pk = picks.reshape(-1).long()
    want = torch.stack([down[pk[i]].double() @ act[i].double() for i in range(pk.numel())])
    room = torch.stack([down[pk[i]].double().abs() @ act[i].double().abs() for i in range(pk.numel())])
    room = room * act.shape[1] * 2.0 ** -23
    if dtype != torch.float32:
        room = room * 1.01 + want.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25
    return want, room


@pytest.mark.parametrize("e,n,k", [(3, 40, 72), (2, 128, 64), (1, 200, 8), (5, 16, 520), (2, 304, 1032)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("mats", [1, 2])
def test_pack_round_trip(e, n, k, dtype, mats):
    from tensorfold_b200 import experts16

    ms = [normal(i, e, n, k, dtype=dtype) for i in range(mats)]
    packed = experts16.pack(*ms)
    assert packed.shape == (e, mats * ((n + 15) // 16 * 16), (k + 63) // 64 * 64) and packed.dtype == dtype
    back = experts16._unpack(packed, mats, n, k)
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(back, ms))
    assert torch.count_nonzero(packed) == sum(torch.count_nonzero(m) for m in ms)       # zeros behind the sizes


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_against_64_bits(case, pdl):
    from tensorfold_b200 import experts16

    dtype, _, limit, e, d, n, slots, rows = case
    up, down = weights(case)
    ex = experts16.make(up, down, limit=limit)
    x, picks = normal(5, rows, d, dtype=dtype), picks_of(rows, slots, e)
    for y_type in (torch.float32, dtype):
        act, y = run(ex, x, picks, y_type=y_type)
        want, room = ref_gate_up(case, up, x, picks)
        assert ((act.double() - want).abs() <= room).all()
        want, room = ref_down(down, act, picks, y_type)
        assert ((y.double() - want).abs() <= room).all()
    back = experts16.unpack(ex)
    assert all(torch.equal(a, b) for a, b in zip(back[0], up)) and torch.equal(back[1], down)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_whole_numbers_come_out_exactly(case):
    """Small whole numbers: every sum is exact in fp32, so the down projection's rows are equal, bit for bit."""

    from tensorfold_b200 import experts, experts16

    dtype, _, _, e, d, n, slots, rows = case
    up, down = weights(case, make=whole)
    ex = experts16.make(up, down)
    picks = picks_of(rows, slots, e)
    act = whole(9, rows * slots, n, dtype=dtype)
    plan = experts16.Plan(rows, slots, e, DEV)
    experts.route(picks, plan)
    y = torch.empty((rows * slots, d), dtype=torch.float32, device=DEV)
    experts16.down(act, ex, plan, y, rows)
    want = torch.stack([down[p].double() @ a for p, a in zip(picks.reshape(-1).long(), act.double())])
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_a_pair_does_not_depend_on_the_call(case):
    """Rows alone, other item sizes and another order of the rows: the same bits."""

    from tensorfold_b200 import experts16

    dtype, _, limit, e, d, n, slots, rows = case
    up, down = weights(case, 21)
    ex = experts16.make(up, down, limit=limit)
    x, picks = normal(6, rows, d, dtype=dtype), picks_of(rows, slots, e, 8)
    act, y = run(ex, x, picks)
    for tile in (8, 16, 48, 64, 65, 256):
        a, b = run(ex, x, picks, tile)
        assert torch.equal(a, act) and torch.equal(b, y), tile
    for r in {0, rows // 2, rows - 1}:
        a, b = run(ex, x[r:r + 1], picks[r:r + 1])
        assert torch.equal(a, act[r * slots:(r + 1) * slots]) and torch.equal(b, y[r * slots:(r + 1) * slots]), r
    perm = torch.randperm(rows, generator=torch.Generator().manual_seed(1)).to(DEV)
    a, b = run(ex, x[perm].contiguous(), picks[perm].contiguous())
    at = (perm[:, None] * slots + torch.arange(slots, device=DEV)).reshape(-1)
    assert torch.equal(a, act[at]) and torch.equal(b, y[at])


def test_one_expert_takes_every_pair():
    """Many items of one expert, the last one partly filled."""

    from tensorfold_b200 import experts16

    case = (BF, True, 0.0, 3, 128, 72, 1, 1000)
    up, down = weights(case, 31)
    ex = experts16.make(up, down)
    x, picks = normal(7, 1000, 128), torch.full((1000, 1), 2, dtype=torch.int32, device=DEV)
    act, y = run(ex, x, picks)
    want, room = ref_gate_up(case, up, x, picks)
    assert ((act.double() - want).abs() <= room).all()
    want, room = ref_down(down, act, picks, torch.float32)
    assert ((y.double() - want).abs() <= room).all()


def test_values_behind_a_row_and_in_other_rows_do_not_leak():
    """NaN and infinities behind the inputs of a strided row, and in other pairs' rows, stay where they are."""

    from tensorfold_b200 import experts16

    case = (BF, True, 0.0, 4, 200, 136, 2, 24)
    up, down = weights(case, 41)
    ex = experts16.make(up, down)
    wide = normal(8, 24, 264)
    picks = picks_of(24, 2, 4)
    clean = wide[:, :200].clone()
    act, y = run(ex, wide[:, :200], picks)
    assert torch.equal(run(ex, clean, picks)[0], act)
    wide[:, 200:] = float("nan")
    assert torch.equal(run(ex, wide[:, :200], picks)[0], act)
    wide[5, 3], wide[6, 7] = float("nan"), float("inf")
    a, b = run(ex, wide[:, :200], picks)
    keep = torch.ones(48, dtype=torch.bool, device=DEV)
    keep[10:14] = False
    assert torch.equal(a[keep], act[keep]) and torch.equal(b[keep], y[keep])
    assert torch.isnan(a[10:12]).all() and not torch.isfinite(a[12:14]).all()
    one = weights(case, 41)
    one[0][0][2, 5, 9] = float("inf")                                    # one weight: its column of its expert alone
    a, _ = run(experts16.make(*one), clean, picks)
    hit = (picks.reshape(-1) == 2)
    assert torch.equal(a[~hit], act[~hit]) and torch.equal(a[hit][:, :5], act[hit][:, :5])
    assert torch.equal(a[hit][:, 6:], act[hit][:, 6:])


def test_relu2_and_clip_keep_nan():
    from tensorfold_b200 import experts16

    for swiglu, limit in ((False, 0.0), (True, 1.0)):
        case = (HF, swiglu, limit, 2, 64, 32, 1, 4)
        up, down = weights(case, 51)
        x = normal(9, 4, 64, dtype=HF)
        x[1, 0] = float("nan")
        act, _ = run(experts16.make(up, down, limit=limit), x, picks_of(4, 1, 2))
        assert torch.isnan(act[1]).all() and torch.isfinite(act[[0, 2, 3]]).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_slots_that_take_no_part(dtype):
    """Picks outside 0..E-1 (a padded batch): their pairs' rows stay as they are, their weights count for nothing, a row
    without any comes out as zeros."""

    from tensorfold_b200 import experts, experts16, moe

    case = (dtype, True, 0.0, 6, 136, 72, 3, 20)
    up, down = weights(case, 61)
    ex = experts16.make(up, down)
    x, picks = normal(10, 20, 136, dtype=dtype), picks_of(20, 3, 6)
    wts = torch.rand((20, 3), generator=gen(2), device=DEV)
    full = picks.clone()
    picks[4, 1], picks[7], picks[9, 0], picks[19] = -1, -5, 6, 1 << 30
    out = (picks < 0) | (picks >= 6)
    wts[out] = float("nan")
    act, y = run(ex, x, picks)
    act0, y0 = run(ex, x, full)
    gone = out.reshape(-1)
    assert (act[gone] == 77).all() and (y[gone] == 77).all()
    assert torch.equal(act[~gone], act0[~gone]) and torch.equal(y[~gone], y0[~gone])
    buf = moe.buffers(ex, 32, 3)
    buf.y.fill_(float("nan"))
    buf.act.fill_(float("nan"))
    got = moe.picked(x, ex, picks, wts, buf=buf)
    w = torch.where(out, torch.zeros_like(wts), wts).double()
    # the sum over the slots: three fp32 steps, and bf16's rounding
    want = (y0.view(20, 3, -1).double() * w[..., None]).sum(1)
    room = (y0.view(20, 3, -1).double().abs() * w[..., None]).sum(1) * 3 * 2.0 ** -24
    if got.dtype == BF:
        room = room * 1.01 + want.abs() * torch.finfo(BF).eps / 2
    assert got.dtype == (BF if dtype == BF else torch.float32)
    assert ((got.double() - want).abs() <= room).all()
    assert (got[7] == 0).all() and (got[19] == 0).all()


@pytest.mark.parametrize("rows,slots,count", [(1, 1, 1), (1, 8, 9), (4, 8, 128), (32, 1, 3), (3, 7, 5), (2, 16, 70), (1, 32, 2),
                                              (31, 1, 1), (11, 3, 64)])
def test_few_pairs_need_no_plan(rows, slots, count):
    """Up to 32 pairs the launches sort the picks themselves, repeated and absent ones among them: the bits of the same
    rows in a call of more pairs, which plans; the plan's tables are left alone."""

    from tensorfold_b200 import experts16, moe

    case = (BF, True, 0.0, count, 136, 72, slots, rows)
    ex = experts16.make(*weights(case, 73))
    g = torch.Generator().manual_seed(rows * slots)
    picks = torch.randint(-1, count + 1, (rows, slots), generator=g).to(torch.int32).to(DEV)
    x, wts = normal(3, rows, 136), torch.rand((rows, slots), generator=gen(4), device=DEV)
    many = 33 // (rows * slots) + 1
    want = moe.picked(x.repeat(many, 1), ex, picks.repeat(many, 1), wts.repeat(many, 1))
    buf = moe.buffers(ex, rows, slots)
    for t in (buf.plan.items, buf.plan.members, buf.plan.counts):
        t.fill_(-9)
    got = moe.picked(x, ex, picks, wts, buf=buf)
    assert rows * slots > 32 or all((t == -9).all() for t in (buf.plan.items, buf.plan.members, buf.plan.counts))
    assert torch.equal(got, want[:rows]) and torch.equal(want[-rows:], want[:rows])


@pytest.mark.parametrize("tile", [32, 64, 256])
def test_a_plan_of_more_rows_than_the_call(tile):
    """Fewer rows than were routed: their pairs' rows, and nothing behind them."""

    from tensorfold_b200 import experts, experts16

    case = (BF, True, 0.0, 3, 136, 72, 2, 90)
    up, down = weights(case, 77)
    ex = experts16.make(up, down)
    x, picks = normal(4, 90, 136), picks_of(90, 2, 3)
    act, y = run(ex, x, picks)
    plan = experts16.Plan(90, 2, 3, DEV)
    plan.decode_tile = tile
    experts.route(picks, plan)
    got = torch.full((180, 72), 55.0, dtype=BF, device=DEV)
    rows = torch.full((180, 136), 55.0, device=DEV)
    experts16.gate_up(x[:41], ex, plan, got[:82], 41)
    experts16.down(got[:82], ex, plan, rows[:82], 41)
    assert torch.equal(got[:82], act[:82]) and (got[82:] == 55).all()
    assert torch.equal(rows[:82], y[:82]) and (rows[82:] == 55).all()


def test_a_plan_without_pairs_and_calls_without_rows():
    from tensorfold_b200 import experts16, moe

    case = (BF, True, 0.0, 4, 64, 40, 2, 8)
    ex = experts16.make(*weights(case, 71))
    none = torch.full((8, 2), -1, dtype=torch.int32, device=DEV)
    act, y = run(ex, normal(11, 8, 64), none)
    assert (act == 77).all() and (y == 77).all()
    got = moe.picked(normal(11, 8, 64), ex, none, torch.ones((8, 2), device=DEV))
    assert (got == 0).all()
    got = moe.picked(normal(11, 0, 64), ex, none[:0], torch.ones((0, 2), device=DEV))
    assert got.shape == (0, 64)


def test_the_layer_takes_either_kind_of_experts(pdl):
    """``moe.run``, ``layer``, ``Runner`` and ``picked`` on one layer: the same picks, the same bits; the routed sum."""

    from tensorfold_b200 import experts16, moe

    case = (BF, True, 0.0, 12, 256, 128, 4, 40)
    up, down = weights(case, 81)
    ex = experts16.make(up, down)
    for shared in (False, True):
        rows_w = normal(12, 12, 256, scale=0.05)
        layer = moe.Routed(rows_w, ex, 4, shared=shared)
        x = normal(13, 40, 256)
        got = moe.run(x, layer)
        buf = moe.MoEBuffers(40, moe._Shape(layer), DEV, shared=shared, dtype=BF)
        out = torch.empty_like(got)
        assert moe.layer(x, layer, buf, out) == 6 and torch.equal(out, got)
        assert torch.equal(moe.Runner(layer, 40)(x), got)
        pick, wts = buf.pick[:40].contiguous(), buf.wts[:40].contiguous()
        assert torch.equal(moe.picked(x, ex, pick, wts), got)
        want, _ = ref_gate_up(case, up, x, pick)
        y = torch.stack([down[p].double() @ a for p, a in zip(pick.reshape(-1).long(), want)]).view(40, -1, 256)
        want = (y * wts.double()[..., None]).sum(1)
        assert (got.double() - want).norm() <= 2.0 ** -8 * want.norm()      # one rounding of the activations, one of the sum
        prompt = moe.run(x, layer, prefill=True)
        assert (prompt.double() - want).norm() <= 2.0 ** -7 * want.norm()   # and one of the rows


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_picked_on_4_bit_experts(prefill, shared):
    """A 4-bit layer's own picks and weights through ``picked``: the layer's bits; slots that take no part."""

    from tensorfold_b200 import experts, moe, synthetic

    shape = synthetic.SMALL_SHARED if shared else synthetic.SMALL
    gate, up, down = synthetic.affine_layer(shape, DEV)
    layer = moe.Routed(synthetic.router_rows(shape, DEV), experts.make([gate, up], down, 64), shape.top_k, shared=shared)
    x = synthetic.activations(shape, 21, DEV)
    buf = moe.MoEBuffers(21, moe._Shape(layer), DEV, prefill=prefill, shared=shared)
    want = torch.empty((21, shape.dims), dtype=BF, device=DEV)
    moe.layer(x, layer, buf, want)
    pick, wts = buf.pick[:21].contiguous(), buf.wts[:21].contiguous()
    mine = moe.buffers(layer.experts, 21, pick.shape[1], prefill=prefill)
    assert torch.equal(moe.picked(x, layer.experts, pick, wts, buf=mine), want)
    pick[3], wts[3] = -1, float("nan")
    got = moe.picked(x, layer.experts, pick, wts, buf=mine)
    assert (got[3] == 0).all() and torch.equal(got[:3], want[:3]) and torch.equal(got[4:], want[4:])


def test_graph_replays_follow_the_picks_on_their_own_scratch():
    """Two captured layers with buffers of their own, replayed in turn on other picks and rows, on another stream."""

    from tensorfold_b200 import experts16, moe

    case = (BF, True, 0.0, 9, 136, 72, 3, 30)
    ex = experts16.make(*weights(case, 91))
    stream = torch.cuda.Stream()
    held = []
    for rows in (30, 70):
        x, picks, wts = normal(1, rows, 136), picks_of(rows, 3, 9, rows), torch.rand((rows, 3), generator=gen(rows), device=DEV)
        buf, out = moe.buffers(ex, rows, 3), torch.empty((rows, 136), dtype=BF, device=DEV)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            moe.picked(x, ex, picks, wts, buf=buf, out=out)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            moe.picked(x, ex, picks, wts, buf=buf, out=out)
        held.append((rows, x, picks, wts, out, graph))
    for turn in range(3):
        for rows, x, picks, wts, out, graph in held:
            x.copy_(normal(100 + turn, rows, 136))
            picks.copy_(picks_of(rows, 3, 9, 50 + turn))
            graph.replay()
            got = out.clone()
            assert torch.equal(got, moe.picked(x, ex, picks, wts))


def test_two_streams_at_once():
    """Blocks of different sizes on two streams, launched in turn without waiting, each with its own scratch."""

    from tensorfold_b200 import experts16, moe

    jobs = []
    for i, (rows, e, d, n, slots) in enumerate([(400, 6, 512, 264, 2), (3, 9, 256, 136, 4)]):
        ex = experts16.make(*weights((BF, True, 0.0, e, d, n, slots, rows), 101 + i))
        x, picks, wts = normal(i, rows, d), picks_of(rows, slots, e, i), torch.rand((rows, slots), generator=gen(i), device=DEV)
        jobs.append((x, ex, picks, wts, moe.buffers(ex, rows, slots), torch.cuda.Stream(), moe.picked(x, ex, picks, wts)))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k, (x, ex, picks, wts, buf, stream, _want) in enumerate(jobs):
            with torch.cuda.stream(stream):
                got[k].append(moe.picked(x, ex, picks, wts, buf=buf))
    torch.cuda.synchronize()
    for k, job in enumerate(jobs):
        assert all(torch.equal(g, job[-1]) for g in got[k])


def test_offsets_past_32_bits():
    """An output of more than 2^32 bytes: its last rows and columns are the right ones."""

    from tensorfold_b200 import experts, experts16

    n, rows = 65536, 33000
    up = whole(1, 1, n, 8, dtype=BF)
    ex = experts16.Experts16(experts16.pack(up), up, n, 8, False)
    plan = experts16.Plan(rows, 1, 1, DEV)
    experts.route(torch.zeros((rows, 1), dtype=torch.int32, device=DEV), plan)
    x = whole(2, rows, 8)
    out = torch.zeros((rows, n), dtype=BF, device=DEV)
    experts16.gate_up(x, ex, plan, out, rows)
    at = torch.tensor([0, 1, 16383, 16384, 32767, 32768, rows - 1], device=DEV)
    want = (x[at].float() @ up[0].float().t()).clamp(min=0) ** 2
    assert torch.equal(out[at], want.to(BF))


def test_refusals_on_the_gpu():
    from tensorfold_b200 import experts, experts16, moe

    case = (BF, True, 0.0, 4, 64, 40, 2, 8)
    up, down = weights(case, 95)
    ex = experts16.make(up, down)
    plan = experts16.Plan(8, 2, 4, DEV)
    picks = picks_of(8, 2, 4)
    experts.route(picks, plan)
    x, act = normal(1, 8, 64), torch.empty((16, 40), dtype=BF, device=DEV)
    y = torch.empty((16, 64), device=DEV)
    for bad in (x.to(HF), x.float(), x[:, :56], x[:7], torch.empty_strided((8, 64), (1, 8), dtype=BF, device=DEV),
                normal(1, 8, 68)[:, 4:], normal(1, 8 * 64 + 8).as_strided((8, 64), (64, 1), 1)):
        with pytest.raises(ValueError, match="x: at least"):
            experts16.gate_up(bad, ex, plan, act, 8)
    for bad in (act.float(), act[:15], torch.empty((16, 48), dtype=BF, device=DEV)[:, :40]):
        with pytest.raises(ValueError, match="out: contiguous"):
            experts16.gate_up(x, ex, plan, bad, 8)
    with pytest.raises(ValueError, match="do not fit a plan"):
        experts16.gate_up(normal(1, 9, 64), ex, plan, torch.empty((18, 40), dtype=BF, device=DEV), 9)
    with pytest.raises(ValueError, match="a plan of 5 experts for 4"):
        experts16.down(act, ex, experts16.Plan(8, 2, 5, DEV), y, 8)
    with pytest.raises(ValueError, match="experts16.Plan"):
        experts16.down(act, ex, experts.Plan(8, 2, 4, DEV, prefill=True), y, 8)
    with pytest.raises(ValueError, match="one device"):
        experts16.down(act, ex, plan, y.cpu(), 8)
    wts = torch.ones((8, 2), device=DEV)
    for kw in ({"wts": wts.double()}, {"wts": wts[:, :1]}, {"picks": picks.long()}, {"picks": picks[:, :1]}, {"x": x[:7]},
               {"out": torch.empty((8, 64), dtype=HF, device=DEV)}, {"buf": moe.buffers(ex, 4, 2)},
               {"buf": moe.buffers(ex, 8, 3)}, {"picks": picks.cpu()}):
        with pytest.raises(ValueError):
            moe.picked(**{"x": x, "ex": ex, "picks": picks, "wts": wts, **kw})


@pytest.mark.parametrize("stacked", [True, False])
@pytest.mark.parametrize("shared", [True, False])
def test_a_layer_from_a_checkpoint(tmp_path, stacked, shared):
    """``load.routed16``: the layer built from the file equals the layer built from the tensors, shared expert last."""

    from safetensors.torch import save_file
    from tensorfold_b200 import experts16, load, moe

    e, d, n = 5, 64, 40
    gate, up = (normal(i, e + 1, n, d, scale=0.1) for i in (1, 2))
    down, rows = normal(3, e + 1, d, n, scale=0.1), normal(4, e + 1, d, scale=0.1)
    tensors = {"l.mlp.gate.weight": rows[:e]}
    if shared:
        tensors["l.mlp.shared_expert_gate.weight"] = rows[e:]
    for proj, m in (("gate_proj", gate), ("up_proj", up), ("down_proj", down)):
        if stacked:
            tensors[f"l.mlp.switch_mlp.{proj}.weight"] = m[:e]
        else:
            tensors.update({f"l.mlp.experts.{i}.{proj}.weight": m[i] for i in range(e)})
        if shared:
            tensors[f"l.mlp.shared_expert.{proj}.weight"] = m[e]
    save_file({k: v.cpu().contiguous() for k, v in tensors.items()}, str(tmp_path / "model.safetensors"))
    layer = load.routed16(load.Checkpoint(tmp_path), "l.mlp.", 2, DEV)
    have = e + 1 if shared else e
    want = moe.Routed(rows[:have], experts16.make([gate[:have], up[:have]], down[:have]), 2, shared=shared)
    assert layer.shared == shared and layer.count == e and torch.equal(layer.router, want.router)
    assert torch.equal(layer.experts.up, want.experts.up) and torch.equal(layer.experts.down, want.experts.down)
    x = normal(5, 9, d)
    assert torch.equal(moe.run(x, layer), moe.run(x, want))
