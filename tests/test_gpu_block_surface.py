"""What autograd, its hooks and the framework's transforms see of the operators around a block."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls():
    """name: (function of a dictionary of tensors that gives tensors, those that have gradients, the others)"""
    from viola_amd import nn
    torch.manual_seed(1)
    cuda = lambda *shape: torch.randn(*shape, device="cuda")  # noqa: E731
    vectors = lambda *names: {k: 1 + 0.3 * cuda(64) for k in names}  # noqa: E731
    x, logits = cuda(4, 6, 64), cuda(4, 6, 8)
    r = nn.route(logits, 2)
    places = {"positions": r.positions, "offsets": r.offsets}
    routing = lambda t: nn.Routing(t["positions"], t["offsets"], t.get("gates"))  # noqa: E731
    return {
        "norm_before": (lambda t: [nn.norm_before(**t)], {"x": x, **vectors("weight", "bias", "scale", "shift")}, {}),
        "norm_after": (lambda t: [nn.norm_after(**t)], {"x": x, "y": cuda(4, 6, 64), **vectors("weight", "bias", "gate")}, {}),
        "norm_between": (lambda t: list(nn.norm_between(**t)),
                         {"x": x, "y": cuda(4, 6, 64), **vectors("after_weight", "after_bias", "weight", "bias", "gate", "scale", "shift")}, {}),
        "route": (lambda t: [nn.route(t["logits"], 2)[i] for i in (2, 5)], {"logits": logits}, {}),
        "balance_loss": (lambda t: [nn.balance_loss(t["logits"], t["experts"])[0]], {"logits": logits}, {"experts": r.experts}),
        "dispatch": (lambda t: [nn.dispatch(t["x"], routing(t))], {"x": x}, places),
        "combine": (lambda t: [nn.combine(t["y"], routing(t))], {"y": cuda(48, 64), "gates": torch.rand(4, 6, 2, device="cuda")}, places),
    }


NAMES = ("norm_before", "norm_after", "norm_between", "route", "balance_loss", "dispatch", "combine")


def _step(name, calls=None):
    """(outputs, gradients) for fixed gradients of the outputs"""
    f, given, others = (calls or _calls())[name]
    given = {k: t.detach().requires_grad_() for k, t in given.items()}
    outputs = f({**given, **others})
    torch.manual_seed(2)
    return outputs, list(torch.autograd.grad(outputs, list(given.values()), [torch.randn_like(t) for t in outputs]))


def _equal(a, b):
    return all(torch.equal(u, v) for u, v in zip([*a[0], *a[1]], [*b[0], *b[1]]))


@pytest.mark.parametrize("name", NAMES)
def test_hooks_see_what_is_saved(name):
    """Moved to the host and back, the saved tensors give the same gradients."""
    calls = _calls()
    first, packed = _step(name, calls), []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (packed.append(t.shape), t.cpu())[1], lambda t: t.cuda()):
        again = _step(name, calls)
    assert packed and _equal(first, again)


@pytest.mark.parametrize("name", NAMES)
def test_checkpointing_gives_the_same(name):
    from torch.utils.checkpoint import checkpoint
    f, given, others = _calls()[name]
    results = []
    for through in (lambda t: f(t), lambda t: checkpoint(f, t, use_reentrant=False)):
        leaves = {k: t.detach().requires_grad_() for k, t in given.items()}
        outputs = through({**leaves, **others})
        results.append((outputs, torch.autograd.grad(outputs, list(leaves.values()), [torch.ones_like(t) for t in outputs])))
    assert _equal(*results)


@pytest.mark.parametrize("name", NAMES)
def test_recording_is_refused(name):
    """A trace must fail, not record this input's output as a constant."""
    from torch.fx.experimental.proxy_tensor import make_fx
    f, given, others = _calls()[name]
    key, x = next(iter(given.items()))
    call = lambda t: f({**given, **others, key: t})[0]  # noqa: E731
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="recorded"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(NotImplementedError):
            make_fx(call)(x)
        assert torch.equal(call(x), f({**given, **others})[0])               # and nothing of it stays


@pytest.mark.parametrize("name", NAMES)
def test_transforms_and_forward_mode_are_refused(name):
    import torch.autograd.forward_ad as forward_ad
    f, given, others = _calls()[name]
    key, x = next(iter(given.items()))
    call = lambda t: f({**given, **others, key: t})[0]  # noqa: E731
    with pytest.raises(NotImplementedError):
        torch.func.grad(lambda t: call(t).sum())(x)
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda t: call(x).sum() * t)(torch.ones(2, device="cuda"))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        call(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("name", NAMES)
def test_modes_that_watch_see_the_same_results(name):
    from torch.utils.flop_counter import FlopCounterMode
    calls = _calls()
    first = _step(name, calls)
    with FlopCounterMode(display=False):
        again = _step(name, calls)
    assert _equal(first, again)


def test_recording_the_grouped_linear_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    from viola_amd import nn
    torch.manual_seed(3)
    experts = nn.GroupedExperts(2, 64, 32, device="cuda").requires_grad_(False)
    x = torch.randn(48, 64, device="cuda").bfloat16()
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="recorded"):
            torch.jit.trace(lambda t: experts(t, [16, 32]), (x,), check_trace=False)
        with pytest.raises(NotImplementedError):
            make_fx(lambda t: experts(t, [16, 32]))(x)
        assert experts(x, [16, 32]).shape == (48, 32)


def test_what_no_gradient_reads_may_change_and_go():
    """The residual stream that norm_after adds to, shifts and biases whose values no gradient needs, gates where the rows have none: changed in place, the gradients
    stay those of the call, and nothing holds their memory."""
    from viola_amd import nn
    torch.manual_seed(4)
    cuda = lambda *shape: torch.randn(*shape, device="cuda")  # noqa: E731
    y, w, gate, d = cuda(64, 256, 512), cuda(512), cuda(512), cuda(64, 256, 512)
    for change in (False, True):
        x, bias, out_bias, shift = cuda(64, 256, 512).requires_grad_(), torch.ones(512, device="cuda"), torch.ones(512, device="cuda"), cuda(64, 1, 512).requires_grad_()
        leaf = [t.detach().requires_grad_() for t in (y, w, gate)]
        before = torch.cuda.memory_allocated()
        stream = x * 1.0
        out = nn.norm_after(stream, leaf[0], leaf[1], gate=leaf[2])
        held = torch.cuda.memory_allocated() - before
        if change:
            stream.data_ptr()
            with torch.no_grad():
                stream.add_(1.0)
        del stream
        # out and the statistics are left
        assert torch.cuda.memory_allocated() - before <= held - x.numel() * 4
        grads = torch.autograd.grad(out, [x, *leaf], d)
        h = nn.norm_before(y, leaf[1], bias, shift=shift)
        plain = nn.norm_after(y, leaf[0], leaf[1], out_bias)
        if change:
            with torch.no_grad():
                for t in (bias, out_bias, shift):
                    t.add_(1.0)
        grads = (*grads, *torch.autograd.grad(h, [leaf[1], shift], d), *torch.autograd.grad(plain, leaf[:2], d))
        if not change:
            first = grads
    assert torch.equal(first[0], d) and all(torch.equal(a, b) for a, b in zip(first[1:], grads[1:]))
    r = nn.route(cuda(50, 8), 2)
    rows, gates = cuda(100, 64), r.gates.clone().requires_grad_()
    out = nn.combine(rows, r._replace(gates=gates))
    expected, = torch.autograd.grad(out, gates, torch.ones_like(out), retain_graph=True)
    with torch.no_grad():
        gates.add_(1.0)
    again, = torch.autograd.grad(out, gates, torch.ones_like(out))
    assert torch.equal(expected, again)


def test_what_a_gradient_reads_may_not_change():
    from viola_amd import nn
    torch.manual_seed(5)
    cuda = lambda *shape: torch.randn(*shape, device="cuda")  # noqa: E731
    given = dict(x=cuda(4, 6, 64), y=cuda(4, 6, 64), after_weight=cuda(64), after_bias=cuda(64), weight=cuda(64), bias=cuda(64), gate=cuda(64), scale=cuda(64))
    for name in given:
        on = {k: t.clone().requires_grad_() for k, t in given.items()}
        out, h = nn.norm_between(**on)
        with torch.no_grad():
            on[name].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            (out.sum() + h.sum()).backward()
    on = {k: t.clone().requires_grad_() for k, t in given.items()}
    out = nn.norm_after(on["x"], on["y"], on["after_weight"], on["after_bias"], gate=on["gate"])
    with torch.no_grad():
        on["after_bias"].add_(1.0)                                           # the gate's gradient reads it
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


@pytest.mark.parametrize("c", [64, 250, 1152, 8200])
@pytest.mark.parametrize("after", ["layer", None])
def test_norm_after_without_its_stream(c, after):
    """The gradients without x's values, in each of the kernels (rows in registers, odd widths, rows beyond them), to the last bit those of a call that kept them:
    the same pass with a gradient of zeros for the h of norm_between."""
    from viola_amd import nn
    torch.manual_seed(6)
    cuda = lambda *shape: torch.randn(*shape, device="cuda")  # noqa: E731
    given = dict(x=cuda(3, 5, c), y=cuda(3, 5, c), after_weight=cuda(c), after_bias=cuda(c), gate=cuda(3, 1, c))
    d = cuda(3, 5, c)
    on = {k: t.clone().requires_grad_() for k, t in given.items()}
    out = nn.norm_after(on["x"], on["y"], on["after_weight"], on["after_bias"], gate=on["gate"], kind=after, residual_scale=0.7)
    with torch.no_grad():
        on["x"].fill_(float("nan"))
    grads = torch.autograd.grad(out, list(on.values()), d)
    on = {k: t.clone().requires_grad_() for k, t in given.items()}
    out, h = nn.norm_between(**on, after=after, residual_scale=0.7)
    expected = torch.autograd.grad([out, h], list(on.values()), [d, torch.zeros_like(h)])
    assert all(torch.equal(a, b) for a, b in zip(grads, expected))
