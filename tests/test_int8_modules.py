"""Int8Linear and Int8Experts without a GPU: devices, casts and state dicts."""

import pytest
import torch

from viola_amd import nn


def _layers(device):
    return [nn.Int8Linear(40, 24, device=device), nn.Int8Linear(40, 24, False, activation="silu", cache_transpose=True, device=device), nn.Int8Experts(3, 40, 24, device=device)]


def test_empty_on_the_meta_device():
    for meta, source in zip(_layers("meta"), _layers("cpu")):
        for t in source.state_dict().values():
            t.copy_(torch.randint(-127, 128, t.shape))
        layer = torch.nn.Sequential(meta).to_empty(device="cpu")[0]
        assert {name: (t.dtype, t.shape, t.device) for name, t in layer.state_dict().items()} == {name: (t.dtype, t.shape, t.device) for name, t in source.state_dict().items()}
        layer.load_state_dict(source.state_dict())
        assert all(torch.equal(layer.state_dict()[name], t) for name, t in source.state_dict().items())


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to("meta"), lambda m: m.to("meta", torch.half)])
@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_casts_leave_codes_and_scales(cast, device):
    for layer in _layers(device):
        if device == "cpu":
            layer.weight_scale.copy_(torch.rand(layer.weight_scale.shape))
        before = layer.weight_scale.clone()
        cast(layer)
        assert layer.codes.dtype == torch.int8 and layer.weight_scale.dtype == torch.float32 and layer.weight_scale.device == layer.codes.device
        assert layer.weight_scale.is_meta or torch.equal(layer.weight_scale, before)
