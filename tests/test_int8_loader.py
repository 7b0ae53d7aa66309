"""Which buffers an int8 checkpoint has to fill: those of W8Linear layers, and no other module's that happen to have their names."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from tandem_amd import loader
from tandem_amd.layers import w8


class Scaler(nn.Module):
    """A module whose state is no checkpoint's."""

    def __init__(self) -> None:
        super().__init__()
        self.register_buffer("weight", torch.full((3,), 7.0))
        self.register_buffer("weight_scale", torch.full((2,), 5.0))


def _save(path, tensors):
    from safetensors.torch import save_file

    save_file(tensors, str(path / "model.safetensors"))


def test_other_modules_buffers_are_left_alone(tmp_path):
    model = nn.Module()
    model.proj, model.other, model.dense = w8.W8Linear(32, 6), Scaler(), nn.Linear(4, 2, bias=False)
    tensors = {"proj.weight": torch.randint(-127, 128, (6, 32), dtype=torch.int8), "proj.weight_scale": torch.rand(6, 1),
               "dense.weight": torch.randn(2, 4)}
    assert set(loader.model_tensors(model)) == set(tensors)
    _save(tmp_path, tensors)
    loader.load_weights(model, str(tmp_path))
    assert all(torch.equal(t, tensors[n]) for n, t in loader.model_tensors(model).items())
    assert bool((model.other.weight == 7).all()) and bool((model.other.weight_scale == 5).all())
    _save(tmp_path, {n: t for n, t in tensors.items() if n != "proj.weight_scale"})
    with pytest.raises(RuntimeError, match="weight_scale"):
        loader.load_weights(model, str(tmp_path))


def test_a_layer_that_is_the_model(tmp_path):
    layer = w8.W8Linear(16, 3)
    assert set(loader.model_tensors(layer)) == {"weight", "weight_scale"}


def test_types_are_checked_before_anything_is_copied(tmp_path):
    model = nn.Module()
    model.first, model.proj = nn.Linear(4, 2, bias=False), w8.W8Linear(32, 6)
    _save(tmp_path, {"first.weight": torch.zeros(2, 4), "proj.weight": torch.zeros(6, 32, dtype=torch.uint8), "proj.weight_scale": torch.ones(6, 1)})
    model.proj.weight.fill_(1)
    before = {n: t.clone() for n, t in loader.model_tensors(model).items()}
    with pytest.raises(ValueError, match="proj.weight: int8 tensors expected"):
        loader.load_weights(model, str(tmp_path))
    assert all(torch.equal(t.nan_to_num(), before[n].nan_to_num()) for n, t in loader.model_tensors(model).items())
