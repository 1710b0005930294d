"""Which kind of experts an entry point takes, said before it sets anything up (no GPU needed)."""

import pytest
import torch

BF = torch.bfloat16


def experts_16_bit():
    from tensorfold_b200 import experts16

    return experts16.Experts16(torch.zeros((2, 32, 64), dtype=BF), torch.zeros((2, 64, 64), dtype=BF), 16, 64, True)


def experts_4_bit():
    from tensorfold_b200 import experts

    return experts.Experts(torch.zeros((2, 2, 1, 2, experts.BLOCK), dtype=torch.int32),
                           torch.zeros((2, 2, 1, 1, experts.BLOCK), dtype=torch.int32), 64, 64, 64)


@pytest.mark.parametrize("step,which", [("CudaBackend", "local"), ("CudaBackend", "shared"), ("GatheredExpertParallel", "local"),
                                        ("PeerExpertParallel", "local"), ("PeerExpertParallel", "shared")])
def test_expert_parallel_steps_refuse_16_bit_experts_before_they_are_set_up(step, which):
    """No window, no buffer, no exchange begun."""

    from tensorfold_b200 import ep

    local, shared = (experts_16_bit(), None) if which == "local" else (experts_4_bit(), experts_16_bit())
    rows = torch.zeros((2, 64), dtype=BF)
    calls = {"CudaBackend": lambda: ep.CudaBackend(rows, local, 1, 2, shared),
             "GatheredExpertParallel": lambda: ep.GatheredExpertParallel(rows, local, 2, 1, 4),
             "PeerExpertParallel": lambda: ep.PeerExpertParallel(rows, local, 2, 1, 4, None, shared)}
    with pytest.raises(ValueError, match="run through experts16"):
        calls[step]()


def test_an_object_with_the_fields_of_4_bit_experts_is_one():
    """A caller's own holder of a layer's blocks passes up to the device check, as ``Experts`` does."""

    from types import SimpleNamespace

    from tensorfold_b200 import experts

    real = experts_4_bit()
    own = SimpleNamespace(**{f: getattr(real, f) for f in ("up", "down", "gs", "width", "dims", "limit", "scale_dtype", "count", "swiglu")})
    plan, x, wts = experts.Plan(4, 1, 2, "cpu"), torch.zeros((4, 64), dtype=BF), torch.zeros((4, 1))
    y, arrive = torch.zeros((4, 64)), torch.zeros((8,), dtype=torch.int32)
    for ex in (real, own):
        for call in (lambda: experts.gate_up(x, ex, plan, x, 4), lambda: experts.down(x, ex, plan, y, 4),
                     lambda: experts.down_combine(x, ex, plan, y, 4, wts, x, arrive)):
            with pytest.raises(ValueError, match="CUDA"):
                call()


@pytest.mark.gpu
def test_an_object_with_the_fields_of_4_bit_experts_runs():
    from types import SimpleNamespace

    from tensorfold_b200 import experts, moe, synthetic

    shape = synthetic.SMALL
    gate, up, down = synthetic.affine_layer(shape, "cuda")
    real = experts.make([gate, up], down, 64)
    own = SimpleNamespace(**{f: getattr(real, f) for f in ("up", "down", "gs", "width", "dims", "limit", "scale_dtype", "count", "swiglu")})
    rows, x = synthetic.router_rows(shape, "cuda"), synthetic.activations(shape, 21, "cuda")
    want = moe.run(x, moe.Routed(rows, real, shape.top_k, shared=False))
    assert torch.equal(moe.run(x, moe.Routed(rows, own, shape.top_k, shared=False)), want)
