"""How many bits of the low-rank row ``adapters.add`` keeps under fp32 rows: whole numbers that need them, exactly."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("rows", [5, 130])
@pytest.mark.parametrize("rank", [8, 32, 40, 100])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_low_rank_rows_of_22_bits_come_out_exactly(dtype, rank, rows):
    """A and x: whole numbers of eight bits, so that A x is exact in fp32 and of up to 22 bits: three parts of a bf16 row hold 24,
    two of fp16 22 (two of bf16, 16, would not).  B: at most two ones a column, base: a whole number below 2^20; all partial
    sums are whole and below 2^24."""

    from tensorfold_b200 import adapters

    g = torch.Generator(device=DEV).manual_seed(rank + rows)

    def bytes_of(*shape):
        sign = torch.randint(0, 2, shape, generator=g, device=DEV) * 2 - 1
        return (sign * torch.randint(128, 256, shape, generator=g, device=DEV)).to(dtype)

    a, x = bytes_of(3, rank, 256), bytes_of(rows, 256)
    b = torch.zeros((3, 72, rank), device=DEV)
    for _ in range(2):
        at = torch.randint(0, rank, (3, 72, 1), generator=g, device=DEV)
        b.scatter_(2, at, (torch.randint(0, 2, at.shape, generator=g, device=DEV) * 2 - 1).float())
    base = torch.randint(-2 ** 19, 2 ** 19, (rows, 72), generator=g, device=DEV).float()
    ids = (torch.arange(rows, device=DEV) % 3).to(torch.int32)
    plan = adapters.Plan(rows, 3, DEV)
    adapters.route(ids, plan)
    low = torch.einsum("mk,mrk->mr", x.double(), a.double()[ids.long()])
    delta = torch.einsum("mr,mnr->mn", low, b.double()[ids.long()])
    assert low.abs().max() < 2 ** 22 and (delta + base).abs().max() < 2 ** 23
    assert ((low.abs() > 2 ** 18) & (low % 2 == 1)).any()
    got = adapters.add(x, adapters.make(a, b.to(dtype)), plan, base)
    assert torch.equal(got.double(), delta + base)
