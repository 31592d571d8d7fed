"""FP8 Linear and MLP built on the meta device: `to_empty` gives them memory, `load_state_dict` their values."""

import pytest
import torch

from viola_amd import nn


@pytest.mark.parametrize("options", [dict(scaling="current"), dict(scaling="grouped", cache_weight_transpose=True), dict(scaling="mxfp8"), dict(weight_dtype="bf16"), dict(scaling="delayed", bias=False)],
                         ids=lambda o: "-".join(map(str, o.values())))
def test_empty_linear(options):
    meta = nn.Linear(64, 96, device="meta", dtype=torch.bfloat16, **options)
    host = nn.Linear(64, 96, device="cpu", dtype=torch.bfloat16, **options)
    with pytest.raises(NotImplementedError, match="to_empty"):
        meta.to("cpu")
    layer = torch.nn.Sequential(meta).to_empty(device="cpu")[0]
    assert isinstance(layer.weight, torch.nn.Parameter) and layer.weight.requires_grad
    told = lambda m: {name: (t.dtype, t.shape, t.device) for name, t in [*m.named_parameters(), *m.named_buffers()]}  # noqa: E731
    assert told(layer) == told(host)
    host._store.pending = False                                               # (its codes would come on the GPU; any will do here)
    for t in [*host.parameters(), *host.buffers()]:
        t.data = torch.randint(0, 100, t.shape, dtype=torch.uint8).to(t.dtype)
    layer.load_state_dict(host.state_dict())
    assert not layer._store.pending
    for name, t in layer.state_dict().items():
        if isinstance(t, torch.Tensor):
            assert torch.equal(t.float(), host.state_dict()[name].float()), name


def test_empty_mlp_and_back():
    block = nn.MLP(64, 32, device="meta").to_empty(device="cpu")
    assert all(t.device.type == "cpu" for t in [*block.parameters(), *block.buffers()])
    held = block.down.weight
    block.half()
    assert block.down.weight is held and held.dtype == torch.float8_e4m3fn
    block.to("meta")
    assert all(t.is_meta for t in [*block.parameters(), *block.buffers()])
