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
