"""Slots of ``adapters.Adapters``: what a refused call and an emptied slot leave, scales at the ends of fp32."""

import pytest
import torch

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def test_a_refused_put_leaves_the_slot_as_it_was():
    from tensorfold_b200 import adapters

    ad = adapters.make(torch.ones((2, 4, 16), dtype=BF), torch.ones((2, 5, 4), dtype=BF), 2.0)
    for scale in ("two", None, torch.ones(2)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ad.put(1, torch.zeros((3, 16)), torch.zeros((5, 3)), scale)
    assert (ad.a[:, :4] == 1).all() and (ad.b[:, :, :4] == 1).all() and ad.scale.tolist() == [2, 2]


def powers(seed, *shape, least=0, most=2):
    """Plus and minus powers of two."""

    g = torch.Generator(device="cuda").manual_seed(seed)
    sign = torch.randint(0, 2, shape, generator=g, device="cuda") * 2 - 1
    return sign * 2.0 ** torch.randint(least, most + 1, shape, generator=g, device="cuda")


# the parts' layouts: one rank for each build
RANKS = (8, 32, 40, 100)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 130])
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_scales_at_the_ends_of_fp32(dtype, rank, rows):
    """Adapters whose low-rank rows lie at either end of fp32's range: exact, as at its middle.  A x: at most 16 inputs of 1 or
    2^-1 times 2^-2 or 2^-3, a multiple of 2^-4 up to 4, in 7 bits; times B's powers from 2^-14 to 2^-12 the products are
    multiples of 2^-18, their sums of at most 100 ranks below 2^-3, so within 15 bits and exact in any order.  Scaled by 2^125
    the low-rank values stay below 2^128; by 2^-126 the results are multiples of 2^-144, which fp32 holds."""

    from tensorfold_b200 import adapters

    a = powers(1, 2, rank, 64, least=-3, most=-2).to(dtype)
    a[:, :, 16:] = 0
    b, x = powers(2, 2, 48, rank, least=-14, most=-12).to(dtype), powers(3, rows, 64, least=-1, most=0).to(dtype)
    ids = (torch.arange(rows, device="cuda") % 2).to(torch.int32)
    plan = adapters.Plan(rows, 2, "cuda")
    adapters.route(ids, plan)
    low = torch.einsum("mk,mrk->mr", x.double(), a.double()[ids.long()])
    delta = torch.einsum("mr,mnr->mn", low, b.double()[ids.long()])
    assert low.abs().max() <= 4 and delta.abs().max() < 2 ** -3
    base = torch.zeros((rows, 48), device="cuda")
    for power in (0, -60, -101, -115, -126, 60, 101, 116, 125):
        ad = adapters.make(a, b, 2.0 ** power)
        got = adapters.add(x, ad, plan, base)
        assert torch.equal(got.double(), delta * 2.0 ** power), power


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 140])
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_rows_of_empty_slots_are_the_base_whatever_their_inputs(dtype, rank, rows):
    """A slot that was never filled and one that was emptied, under infinities, NaN and the type's largest value (a padded
    batch): the base, rounded; the rows of a filled slot beside them as they are alone."""

    from tensorfold_b200 import adapters

    g = torch.Generator(device="cuda").manual_seed(7)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    ad = adapters.Adapters(3, rank, 72, 40, dtype, "cuda")
    ad.put(0, normal(rank, 72) * 0.1, normal(40, rank))
    ad.put(2, normal(rank, 72) * 0.1, normal(40, rank))
    ad.clear(2)
    ids = (torch.arange(rows, device="cuda") % 3).to(torch.int32)
    plan = adapters.Plan(rows, 3, "cuda")
    adapters.route(ids, plan)
    x, base = normal(rows, 72).to(dtype), normal(rows, 40)
    clean = adapters.add(x, ad, plan, base, dtype=dtype)
    empty = (ids != 0).nonzero()[:, 0]
    for i, value in enumerate((float("inf"), float("-inf"), float("nan"), torch.finfo(dtype).max)):
        x[empty[i::4], i::7] = value
    got = adapters.add(x, ad, plan, base, dtype=dtype)
    assert torch.equal(got[empty], base[empty].to(dtype)) and torch.equal(got[ids == 0], clean[ids == 0])
