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
