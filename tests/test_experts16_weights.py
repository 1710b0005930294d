"""Packed weights of 16-bit experts that are not what the kernel would read by their address: refused by every entry point
before anything is launched (no GPU needed), and on the GPU with the results of the whole weights beside them."""

import pytest
import torch

BF, HF = torch.bfloat16, torch.float16


def experts_of(swiglu=True, device="cpu"):
    from tensorfold_b200 import experts16

    mats = 2 if swiglu else 1                                          # 6 experts, 72 inputs, width 24
    return experts16.Experts16(torch.zeros((6, mats * 32, 128), dtype=BF, device=device),
                               torch.zeros((6, 80, 64), dtype=BF, device=device), 24, 72, swiglu)


def off_by_eight_bytes(t):
    return torch.zeros((t.numel() + 4,), dtype=t.dtype)[4:].view(t.shape)


BAD_UP = {"strided": lambda t: torch.cat([t, t])[::2], "fewer-rows": lambda t: t[:, :-16].contiguous(),
          "fewer-inputs": lambda t: t[..., :64].contiguous(), "flat": lambda t: t.view(6, -1), "fp32": lambda t: t.float(),
          "rows-strided": lambda t: torch.cat([t, t], 2)[..., :128], "unaligned": off_by_eight_bytes}
BAD_DOWN = {"strided": lambda t: torch.cat([t, t])[::2], "shorter": lambda t: t[:5], "longer": lambda t: torch.cat([t, t[:1]]),
            "fewer-rows": lambda t: t[:, :-16].contiguous(), "more-inputs": lambda t: torch.cat([t, t], 2), "fp16": lambda t: t.half(),
            "elsewhere": lambda t: t.to("meta"), "unaligned": off_by_eight_bytes}


@pytest.mark.parametrize("swiglu", [True, False])
@pytest.mark.parametrize("which,kind", [("up", k) for k in BAD_UP] + [("down", k) for k in BAD_DOWN])
def test_weights_that_are_not_packed_as_the_kernel_reads_them(which, kind, swiglu):
    from tensorfold_b200 import experts16, moe

    ex = experts_of(swiglu)
    setattr(ex, which, (BAD_UP if which == "up" else BAD_DOWN)[kind](getattr(ex, which)))
    plan, x, act = experts16.Plan(4, 1, 6, "cpu"), torch.zeros((4, 72), dtype=BF), torch.zeros((4, 24), dtype=BF)
    picks, wts = torch.zeros((4, 1), dtype=torch.int32), torch.zeros((4, 1))
    calls = [lambda: moe.picked(x, ex, picks, wts), lambda: experts16.unpack(ex),
             (lambda: experts16.gate_up(x, ex, plan, act, 4)) if which == "up" else
             (lambda: experts16.down(act, ex, plan, torch.zeros((4, 72)), 4))]
    for call in calls:
        with pytest.raises(ValueError, match=f"{which}: (packed weights|every projection)"):
            call()


def test_whole_weights_pass_up_to_the_device():
    from tensorfold_b200 import experts16, moe

    ex, plan, x = experts_of(), experts16.Plan(4, 1, 6, "cpu"), torch.zeros((4, 72), dtype=BF)
    for call in (lambda: experts16.gate_up(x, ex, plan, x[:, :24], 4), lambda: experts16.down(x[:, :24], ex, plan, x, 4),
                 lambda: moe.picked(x, ex, torch.zeros((4, 1), dtype=torch.int32), torch.zeros((4, 1)))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_a_strided_shard_is_refused_and_its_copy_runs():
    """Every second expert: refused by ``picked``, ``gate_up``, ``down``, ``run`` and ``layer``; made contiguous, the results of a
    layer that was made of those experts."""

    from tensorfold_b200 import experts, experts16, moe

    g = torch.Generator(device="cuda").manual_seed(5)

    def normal(*shape):
        return (torch.randn(shape, generator=g, device="cuda") * 0.1).to(BF)

    up, down = [normal(6, 24, 72), normal(6, 24, 72)], normal(6, 72, 24)
    whole = experts16.make(up, down)
    shard = experts16.Experts16(whole.up[::2], whole.down[::2], 24, 72, True)
    short = experts16.Experts16(whole.up, whole.down[:5], 24, 72, True)
    x, picks = normal(4, 72), torch.tensor([[0, 2], [1, 0], [2, 1], [0, 1]], dtype=torch.int32, device="cuda")
    wts = torch.rand((4, 2), generator=g, device="cuda")
    for ex in (shard, short):
        plan, layer = experts16.Plan(4, 2, ex.count, "cuda"), moe.Routed(normal(ex.count, 72), ex, 2, shared=False)
        experts.route(picks, plan)
        act, y = torch.empty((8, 24), dtype=BF, device="cuda"), torch.empty((8, 72), device="cuda")
        calls = [lambda: moe.picked(x, ex, picks, wts), lambda: moe.run(x, layer), lambda: experts16.down(act, ex, plan, y, 4)]
        if ex is shard:
            calls.append(lambda: experts16.gate_up(x, ex, plan, act, 4))
        for call in calls:
            with pytest.raises(ValueError, match="packed weights"):
                call()
    copy = experts16.Experts16(shard.up.contiguous(), shard.down.contiguous(), 24, 72, True)
    mine = experts16.make([m[::2].contiguous() for m in up], down[::2].contiguous())
    assert torch.equal(moe.picked(x, copy, picks, wts), moe.picked(x, mine, picks, wts))


BAD_BLOCKS = {"down-shorter": lambda ex: setattr(ex, "down", ex.down[:3]), "down-narrow": lambda ex: setattr(ex, "down", ex.down[:, :-1].contiguous()),
              "down-strided": lambda ex: setattr(ex, "down", torch.cat([ex.down, ex.down])[::2]),
              "down-elsewhere": lambda ex: setattr(ex, "down", ex.down.to("meta")), "up-strided": lambda ex: setattr(ex, "up", torch.cat([ex.up, ex.up])[::2]),
              "up-groups": lambda ex: setattr(ex, "dims", 192), "down-type": lambda ex: setattr(ex, "down", ex.down.float())}


@pytest.mark.parametrize("kind", BAD_BLOCKS)
def test_picked_refuses_4_bit_blocks_that_do_not_fit_together(kind):
    from tensorfold_b200 import experts, moe

    ex = experts.Experts(torch.zeros((4, 2, 2, 2, experts.BLOCK), dtype=torch.int32),
                         torch.zeros((4, 4, 1, 1, experts.BLOCK), dtype=torch.int32), 64, 64, 128)
    picks, wts = torch.zeros((4, 1), dtype=torch.int32), torch.zeros((4, 1))
    with pytest.raises(ValueError, match="CUDA"):
        moe.picked(torch.zeros((4, 128), dtype=BF), ex, picks, wts)
    BAD_BLOCKS[kind](ex)
    with pytest.raises(ValueError, match="contiguous int32 blocks"):
        moe.picked(torch.zeros((4, ex.dims), dtype=BF), ex, picks, wts)
