"""Layers built on the meta device, given memory on the GPU by `to_empty` and values by `load_state_dict`, compute what the layers computed that the values came from."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("options", [dict(scaling="current"), dict(scaling="grouped", cache_weight_transpose=True), dict(scaling="mxfp8"), dict(weight_dtype="bf16")],
                         ids=lambda o: "-".join(map(str, o.values())))
def test_fp8_linear(options):
    from viola_amd import nn
    torch.manual_seed(0)
    source = nn.Linear(64, 96, device="cuda", dtype=torch.bfloat16, **options)
    layer = nn.Linear(64, 96, device="meta", dtype=torch.bfloat16, **options).to_empty(device="cuda")
    layer.load_state_dict(source.state_dict())
    x = torch.randn(40, 64, device="cuda", dtype=torch.bfloat16)
    results = []
    for m in (source, layer):
        leaf = x.clone().requires_grad_()
        y = m(leaf)
        dx, dw = torch.autograd.grad(y, [leaf, m.weight], torch.ones_like(y))
        results.append((y, dx, dw))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cache_transpose", [False, True])
def test_int8_layers(cache_transpose):
    from viola_amd import nn
    torch.manual_seed(1)
    linear = nn.Int8Linear.from_float(torch.nn.Linear(40, 24, device="cuda"), cache_transpose=cache_transpose)
    experts = nn.Int8Experts.from_float(torch.randn(3, 24, 40, device="cuda"), cache_transpose=cache_transpose)
    empty = [nn.Int8Linear(40, 24, cache_transpose=cache_transpose, device="meta"), nn.Int8Experts(3, 40, 24, cache_transpose=cache_transpose, device="meta")]
    offsets = torch.tensor([0, 4, 4, 9], dtype=torch.int32, device="cuda")
    for source, layer, args in zip((linear, experts), empty, ((), (offsets,))):
        layer.to_empty(device="cuda").load_state_dict(source.state_dict())
        assert (layer.weight_t is None) == (not cache_transpose)
        x = torch.randn(10, 40, device="cuda", requires_grad=True)
        a, b = source(x, *args), layer(x, *args)
        assert torch.equal(a, b)
        assert torch.equal(*(torch.autograd.grad(y, x, torch.ones_like(y))[0] for y in (a, b)))
