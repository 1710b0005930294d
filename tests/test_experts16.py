"""Refusals of the 16-bit experts and of the low-rank adapters that need no GPU, and their kernels' order of reads."""

from types import SimpleNamespace

import pytest
import torch

from test_wait_order import CSRC, kernels, untied

BF, HF = torch.bfloat16, torch.float16


def test_entry_points_refuse_bad_arguments_before_any_launch():
    from tensorfold_b200 import _lib

    g16 = [2, 0, 16, 64, 8, 2, 16, 3, 64, 32, 16, 16, 16, 16, 0.0, 4, 64, 0]
    cases = [("tfb_pack16", (0, 0, 16, 1, 16, 64, 0), "null pointer"),
             ("tfb_pack16", (16, 0, 16, 1, 16, 60, 0), "does not pack"),
             ("tfb_pack16", (16, 24, 16, 1, 16, 64, 0), "16-byte aligned"),
             ("tfb_unpack16", (16, 16, 0, 0, 16, 64, 0), "does not pack")]
    for at, value, why in ((2, 0, "null pointer"), (8, 60, "multiples of 8"), (9, 0, "columns"), (3, 56, "x rows"),
                           (3, 68, "x rows"), (2, 24, "16-byte aligned"), (5, -1, "bad slots"), (16, 257, "items of 1..256"),
                           (16, 0, "items of 1..256"), (7, 0, "expert count"), (0, 4, "no kernel for epilogue 4"), (4, 1 << 31, "x rows")):
        bad = list(g16)
        bad[at] = value
        cases.append(("tfb_experts16", tuple(bad), why))
    block = [0, 16, 64, 4, 16, 2, 16, 16, 1, 0.0, 16, 3, 64, 32, 16, 16, 16, 4, 64, 16, 16, 16, 0, 0]
    for at, value, why in ((1, 0, "null pointer"), (4, 0, "null pointer"), (20, 0, "null pointer"), (2, 60, "x rows"), (5, 0, "bad slots"),
                           (12, 60, "multiples of 8"), (13, 36, "multiples of 8"), (18, 300, "items of 1..256"), (11, 0, "expert count"),
                           (11, 1025, "at most 1024 experts")):
        bad = list(block)
        bad[at] = value
        cases.append(("tfb_experts16_block", tuple(bad), why))
    ad = [0, 16, 64, 16, 16, 16, 16, 64, 32, 16, 4, 2, 0, 0, 0, 0, 16, 0, 32, 32, 1, 32, 0]
    for at, value, why in ((1, 0, "null pointer"), (9, 0, "null pointer"), (12, 16, "a whole plan or none"),
                           (6, 12, "ranks up to 128"), (6, 136, "ranks up to 128"), (7, 60, "multiples of 8"),
                           (2, 60, "16-byte aligned"), (17, 3, "fp32 \\(0\\)"), (20, -1, "fp32 \\(0\\)"), (18, 31, "bad sizes"),
                           (11, 0, "bad sizes"), (19, 16, "in place needs one layout")):
        bad = list(ad)
        bad[at] = value
        cases.append(("tfb_adapters", tuple(bad), why))
    for name, args, why in cases:
        with pytest.raises(ValueError, match=why):
            _lib.call(name, *args)


def test_calls_without_work_launch_nothing():
    from tensorfold_b200 import _lib

    _lib.call("tfb_experts16", 0, 0, 16, 64, 0, 2, 16, 3, 64, 32, 16, 16, 16, 16, 0.0, 4, 64, 0)
    _lib.call("tfb_experts16", 0, 0, 16, 64, 8, 2, 16, 3, 64, 32, 16, 16, 16, 16, 0.0, 0, 64, 0)
    _lib.call("tfb_experts16_block", 0, 16, 64, 0, 16, 2, 16, 16, 1, 0.0, 16, 3, 64, 32, 16, 16, 16, 4, 64, 16, 16, 16, 0, 0)
    _lib.call("tfb_adapters", 0, 16, 64, 16, 16, 16, 16, 64, 32, 16, 0, 2, 0, 0, 0, 0, 16, 0, 32, 32, 1, 32, 0)


def test_weights_that_do_not_fit_together_are_refused():
    from tensorfold_b200 import experts16

    w = torch.zeros((2, 16, 24), dtype=BF)
    down = torch.zeros((2, 24, 16), dtype=BF)
    for up, dn, why in (([w.float(), w], down, "bf16 or fp16"), ([w, w.half()], down, "one dtype"),
                        ([w[:, :, :20]], down, "multiples of 8"), ([w, w, w], down, "alone"), ([], down, "alone"),
                        ([w], down[:1], "down must be"), ([w[0]], down, "bf16 or fp16"), ([w, w], down, "CUDA"),
                        ([w[:0]], down[:0], "multiples of 8")):
        with pytest.raises(ValueError, match=why):
            experts16.make(up, dn)
    with pytest.raises(ValueError, match="gate and up differ"):
        experts16.pack(w, torch.zeros((2, 8, 24), dtype=BF))


def test_the_4_bit_operators_refuse_16_bit_experts():
    from tensorfold_b200 import experts, experts16

    ex = experts16.Experts16(torch.zeros((2, 16, 64), dtype=BF), torch.zeros((2, 16, 64), dtype=BF), 16, 16, False)
    plan, x = experts.Plan(4, 1, 2, "cpu"), torch.zeros((4, 16), dtype=BF)
    for call in (lambda: experts.gate_up(x, ex, plan, x, 4), lambda: experts.down(x, ex, plan, x, 4),
                 lambda: experts.down_combine(x, ex, plan, x, 4, x, x, x)):
        with pytest.raises(ValueError, match="run through experts16"):
            call()


def test_item_sizes():
    from tensorfold_b200 import experts16

    assert experts16.item_pairs(8, 128) < experts16.item_pairs(128 * 1024, 128) == experts16.ITEM
    assert experts16.Plan(4, 2, 8, "cpu").tile == experts16.item_pairs(8, 8)


def test_cpu_tensors_are_refused():
    from tensorfold_b200 import adapters, experts16, moe

    ex = experts16.Experts16(torch.zeros((2, 16, 64), dtype=BF), torch.zeros((2, 16, 64), dtype=BF), 16, 16, False)
    plan = experts16.Plan(4, 1, 2, "cpu")
    with pytest.raises(ValueError, match="CUDA"):
        experts16.gate_up(torch.zeros((4, 16), dtype=BF), ex, plan, torch.zeros((4, 16), dtype=BF), 4)
    with pytest.raises(ValueError, match="CUDA"):
        moe.picked(torch.zeros((4, 16), dtype=BF), ex, torch.zeros((4, 1), dtype=torch.int32), torch.zeros((4, 1)))
    with pytest.raises(ValueError, match="4-bit experts"):
        moe.picked(torch.zeros((4, 16), dtype=BF), SimpleNamespace(), torch.zeros((4, 1), dtype=torch.int32), torch.zeros((4, 1)))
    with pytest.raises(ValueError, match="CUDA"):
        adapters.route(torch.zeros((4,), dtype=torch.int32), adapters.Plan(4, 2, "cpu"))
    ad = adapters.Adapters(2, 8, 16, 16, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        adapters.add(torch.zeros((4, 16), dtype=BF), ad, adapters.Plan(4, 2, "cpu"), torch.zeros((4, 16)))


def test_adapter_slots():
    """Filling, replacing and emptying slots, on the CPU: what the kernel reads."""

    from tensorfold_b200 import adapters

    ad = adapters.Adapters(3, 12, 16, 5, device="cpu")
    assert ad.a.shape == (3, 16, 16) and ad.b.shape == (3, 5, 16) and ad.nbytes() == 3 * (16 * 16 + 5 * 16) * 2 + 12
    a, b = torch.randn(12, 16), torch.randn(5, 12)
    ad.put(1, a, b, 0.5)
    assert torch.equal(ad.a[1, :12], a.to(BF)) and torch.equal(ad.b[1, :, :12], b.to(BF)) and ad.scale.tolist() == [0, 0.5, 0]
    ad.put(1, a[:3], b[:, :3], 2.0)                                    # a smaller rank: nothing of the old one stays
    assert torch.equal(ad.a[1, :3], a[:3].to(BF)) and not ad.a[1, 3:].any() and not ad.b[1, :, 3:].any()
    assert not ad.a[0].any() and not ad.a[2].any()
    ad.clear(1)
    assert not ad.a.any() and not ad.b.any() and not ad.scale.any()
    made = adapters.make(torch.ones(2, 4, 16, dtype=HF), torch.ones(2, 5, 4, dtype=HF), torch.tensor([1.0, 3.0]))
    assert made.dtype == HF and made.a.shape == (2, 8, 16) and made.a.sum() == 128 and made.scale.tolist() == [1, 3]


def test_adapters_that_do_not_fit_are_refused():
    from tensorfold_b200 import adapters

    for args in ((0, 8, 16, 16), (1025, 8, 16, 16), (1, 0, 16, 16), (1, 129, 16, 16), (1, 8, 12, 16), (1, 8, 16, 0)):
        with pytest.raises(ValueError):
            adapters.Adapters(*args, device="cpu")
    with pytest.raises(ValueError, match="bf16 or fp16"):
        adapters.Adapters(1, 8, 16, 16, torch.float32, "cpu")
    ad = adapters.Adapters(2, 8, 16, 6, device="cpu")
    for i, a, b in ((2, (4, 16), (6, 4)), (-1, (4, 16), (6, 4)), (0, (9, 16), (6, 9)), (0, (4, 15), (6, 4)),
                    (0, (4, 16), (6, 5)), (0, (4, 16), (5, 4)), (0, (16,), (6, 1))):
        with pytest.raises(ValueError):
            ad.put(i, torch.zeros(a), torch.zeros(b))
    with pytest.raises(ValueError):
        adapters.make(torch.zeros(2, 4, 16, dtype=BF), torch.zeros(2, 5, 3, dtype=BF))
    with pytest.raises(ValueError, match="one scale"):
        adapters.make(torch.zeros(2, 4, 16, dtype=BF), torch.zeros(2, 5, 4, dtype=BF), torch.ones(3))
    for rows, count in ((0, 1), (1, 0), (1, 1025)):
        with pytest.raises(ValueError):
            adapters.Plan(rows, count, "cpu")
    plan = adapters.Plan(4, 2, "cpu")
    for ids in (torch.zeros((4,)), torch.zeros((5,), dtype=torch.int32), torch.zeros((2, 2), dtype=torch.int32),
                torch.zeros((8,), dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            adapters.route(ids, plan)


@pytest.mark.parametrize("file", ["experts16.cu", "adapters.cu"])
def test_dependent_pointers_are_tied_to_the_wait(file):
    """As ``test_wait_order``: what earlier kernels wrote is read behind the wait (the weights W by bulk copies alone)."""

    found = kernels((CSRC / file).read_text())
    assert any("pdl_wait()" in body for _, _, body in found)
    missing = {name: untied(name, params, body) - ({"W"} if name == "g16_kernel" else set()) for name, params, body in found}
    assert not {n: p for n, p in missing.items() if p}
