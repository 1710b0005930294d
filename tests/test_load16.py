"""``load.routed16`` on checkpoints of another type than bf16: refused by the headers, before a tensor is read (no GPU)."""

import pytest
import torch

BF, HF = torch.bfloat16, torch.float16


def written(path, stacked, bad, dtype):
    """A layer of three experts and a shared one in bf16; the tensor named ``bad`` in ``dtype``."""

    from safetensors.torch import save_file
    from tensorfold_b200 import load

    tensors = {"l.mlp.gate.weight": torch.zeros((3, 64), dtype=BF), "l.mlp.shared_expert_gate.weight": torch.zeros((1, 64), dtype=BF)}
    for proj, shape in (("gate_proj", (16, 64)), ("up_proj", (16, 64)), ("down_proj", (64, 16))):
        if stacked:
            tensors[f"l.mlp.switch_mlp.{proj}.weight"] = torch.zeros((3, *shape), dtype=BF)
        else:
            tensors.update({f"l.mlp.experts.{e}.{proj}.weight": torch.zeros(shape, dtype=BF) for e in range(3)})
        tensors[f"l.mlp.shared_expert.{proj}.weight"] = torch.zeros(shape, dtype=BF)
    for name in tensors:
        if bad in name:
            tensors[name] = tensors[name].to(dtype)
    save_file(tensors, str(path / "model.safetensors"))
    return load.Checkpoint(path)


@pytest.mark.parametrize("dtype,name", [(HF, "F16"), (torch.float32, "F32")])
@pytest.mark.parametrize("stacked,bad", [(True, "switch_mlp"), (True, "switch_mlp.down_proj"), (True, "shared_expert.up_proj"),
                                         (False, "experts."), (False, "experts.2.gate_proj"), (False, "shared_expert.")])
def test_other_types_are_refused_before_anything_is_read(tmp_path, monkeypatch, stacked, bad, dtype, name):
    from tensorfold_b200 import load

    ck = written(tmp_path, stacked, bad, dtype)
    monkeypatch.setattr(load.Checkpoint, "get", lambda *a: pytest.fail("a tensor was read"))
    with pytest.raises(ValueError, match=f"runs in bf16, not {name}"):
        load.routed16(ck, "l.mlp.", 2, "cpu")


@pytest.mark.parametrize("stacked", [True, False])
def test_bf16_is_read(tmp_path, stacked):
    from tensorfold_b200 import load

    with pytest.raises(ValueError, match="CUDA"):                      # packing is the GPU's
        load.routed16(written(tmp_path, stacked, "none", BF), "l.mlp.", 2, "cpu")
