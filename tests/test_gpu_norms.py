"""nn.norm_before / norm_after / norm_between against the 64-bit formulas (oracle.norms): types, widths, strides, vectors for groups of rows, rows that
are all zero or hold what a type cannot, and which gradients are asked for.

Tolerances. A result of 16 bits is rounded once, by at most 2^-8 (BF16) or 2^-11 (FP16) of each value. In 32 bits a sum of n terms is off by at most n 2^-24
of the sum of their magnitudes; the longest chain of additions here is 64 terms of a row or of a portion and 44 for joining them, and a result is a
few such sums: 2^-16 (1.5e-5) of the 2-norm, for sums over rows of the 2-norm of the terms' magnitudes."""

import itertools

import pytest
import torch

from oracle import norms

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SUMS = 2.0 ** -16


def _close(name, actual, expected, measure=None):
    expected = expected.double().cpu()
    measure = expected if measure is None else measure.double().cpu()
    assert actual.shape == expected.shape, name
    off = (actual.detach().double().cpu() - expected).norm()
    bound = UNIT[actual.dtype] * expected.norm() + SUMS * measure.norm()
    # values too small for the type's full precision: half of FP16's smallest step each
    bound += 2.0 ** -25 * expected.numel() ** 0.5 if actual.dtype == F16 else 0.0
    assert off <= bound, (name, off.item(), bound.item())


def _run(form, given, *, after="rms", before="rms", dtype=None, wanted=None, skip=(), **options):
    """The operator on the GPU (gradients of `wanted`, all by default; outputs in `skip` get no gradient) against the formulas."""
    from viola_amd import nn
    torch.manual_seed(77)
    on = {k: v.cuda() for k, v in given.items()}
    wanted = tuple(given) if wanted is None else wanted
    for k in wanted:
        on[k] = on[k].detach().requires_grad_()
    if form == "before":
        outputs = {"h": nn.norm_before(on["x"], on.get("weight"), on.get("bias"), scale=on.get("scale"), shift=on.get("shift"), kind=before, dtype=dtype, **options)}
    elif form == "after":
        outputs = {"out": nn.norm_after(on["x"], on["y"], on.get("after_weight"), on.get("after_bias"), gate=on.get("gate"), kind=after, **options)}
    else:
        out, h = nn.norm_between(**on, after=after, before=before, **options)
        outputs = {"out": out, "h": h}
    kinds = dict(after=after, before=None if form == "after" else before)
    grads = {k: torch.randn(v.shape).to(v.dtype) for k, v in outputs.items() if k not in skip}
    rows = {k: v for k, v in given.items()}
    expected = norms.norm(**rows, **kinds, **options, **{"d" + k: v for k, v in grads.items()})
    for k, v in outputs.items():
        _close(k, v, expected[k])
    if not wanted:
        return outputs
    result = torch.autograd.grad([outputs[k] for k in grads], [on[k] for k in wanted], [g.cuda() for g in grads.values()], allow_unused=True)
    for k, g in zip(wanted, result):
        if g is None:
            assert "d" + k not in expected or not expected["d" + k].any(), k
            continue
        assert g.dtype == given[k].dtype
        _close("d" + k, g, expected["d" + k], expected["m" + k] if k not in ("x", "y") else None)
    return outputs


def _inputs(form, b, s, c, stream, branch, vectors, *, weights=True, biases=True, gate="group", modulated=True, seed=0):
    torch.manual_seed(seed)
    given = {"x": torch.randn(b, s, c).to(stream)}
    if form != "before":
        given["y"] = (torch.randn(b, s, c) * 0.5 + 0.2).to(branch)
        if weights:
            given["after_weight"] = (1 + 0.2 * torch.randn(c)).to(vectors)
        if biases:
            given["after_bias"] = (0.2 * torch.randn(c)).to(vectors)
        if gate:
            given["gate"] = (0.5 + 0.2 * torch.randn(*((b, 1, c) if gate == "group" else (c,)))).to(vectors)
    if form != "after":
        if weights:
            given["weight"] = (1 + 0.2 * torch.randn(c)).to(vectors)
        if biases:
            given["bias"] = (0.2 * torch.randn(c)).to(vectors)
        if modulated:
            given["scale"], given["shift"] = (0.3 * torch.randn(b, 1, c)).to(vectors), (0.3 * torch.randn(b, 1, c)).to(vectors)
    return given


@pytest.mark.parametrize("form,after,before", [("before", "rms", "rms"), ("before", "rms", "layer"), ("after", "rms", "rms"), ("after", "layer", "rms"), ("after", None, "rms"),
                                               ("between", "rms", "rms"), ("between", "layer", "layer"), ("between", None, "layer"), ("between", "rms", "layer")])
@pytest.mark.parametrize("stream,branch,vectors", [(F32, F32, F32), (BF16, BF16, BF16), (F16, F16, F32), (F32, BF16, F32), (F32, F16, F16), (BF16, F32, F32)])
def test_forms_kinds_and_types(form, after, before, stream, branch, vectors):
    given = _inputs(form, 3, 11, 200, stream, branch, vectors)
    options = {} if form == "before" else dict(residual_scale=0.7, branch_scale=1.5)
    _run(form, given, after=after, before=before, dtype=branch if form == "before" else None, **options)


@pytest.mark.parametrize("c", [1, 7, 8, 64, 72, 255, 512, 520, 768, 1000, 1024, 1152, 2048, 4096, 4104, 5000, 8192, 8200, 16384, 20000])
@pytest.mark.parametrize("stream,branch", [(BF16, BF16), (F32, F32), (F32, BF16)])
def test_widths(c, stream, branch):
    _run("between", _inputs("between", 2, 3, c, stream, branch, F32, seed=c), after="layer", before="rms")


@pytest.mark.parametrize("b,s", [(1, 1), (1, 2), (1, 700), (5, 1), (600, 1), (2, 513), (37, 29), (3, 1030)])
def test_rows_and_groups(b, s):
    _run("between", _inputs("between", b, s, 136, BF16, BF16, BF16, seed=b * s), after="rms", before="layer")
    _run("between", _inputs("between", b, s, 136, BF16, BF16, F32, gate="vector", modulated=False, seed=b * s), after="rms", before="rms")


def test_vectors_of_different_groups_meet():
    torch.manual_seed(5)
    given = _inputs("between", 4, 6, 72, F32, F32, F32, gate="vector", modulated=False)
    given["scale"], given["shift"] = 0.3 * torch.randn(4, 1, 72), 0.3 * torch.randn(4, 6, 72)       # one a sequence, one a token
    _run("between", given)
    given["gate"] = 0.5 + 0.1 * torch.randn(1, 1, 72)
    _run("between", given)


def test_gradients_of_broadcast_vectors_reach_their_source():
    """A gate expanded by the caller, or one row of a wider projection: the gradient comes back summed, in the source's shape."""
    from viola_amd import nn
    torch.manual_seed(6)
    x, y = torch.randn(3, 5, 64, device="cuda"), torch.randn(3, 5, 64, device="cuda")
    d = torch.randn(3, 5, 64, device="cuda")
    for source, view in ((torch.randn(1, 1, 64), lambda g: g.expand(3, 1, 64)), (torch.randn(3, 1, 192), lambda g: g[..., 64:128]), (torch.randn(64), lambda g: g)):
        g = source.cuda().requires_grad_()
        grad, = torch.autograd.grad(nn.norm_after(x, y, gate=view(g)), g, d)
        source_64 = source.double().requires_grad_()
        expected = norms.norm(x, y, gate=view(source_64).detach(), before=None, dout=d)["dgate"]
        expected, = torch.autograd.grad(view(source_64), source_64, expected.view(view(source_64).shape))
        _close("gate", grad, expected, torch.full_like(expected, 15 ** 0.5))


def test_strided_rows():
    """Rows cut out of wider ones, from an odd element on, and rows that have no common distance."""
    torch.manual_seed(7)
    wide = torch.randn(4, 9, 3 * 256).bfloat16()
    given = _inputs("between", 4, 9, 256, BF16, BF16, F32)
    for at in (0, 8, 257):
        given["x"], given["y"] = wide[..., at:at + 256], wide[..., 512:] if at != 257 else wide[..., 511:767]
        _run("between", given)
    given["x"], given["y"] = torch.randn(9, 4, 256).bfloat16().transpose(0, 1), torch.randn(4, 1, 256).bfloat16().expand(4, 9, 256)
    _run("between", given)


@pytest.mark.parametrize("wanted", [("x",), ("y",), ("x", "y"), ("gate",), ("after_weight",), ("after_bias",), ("weight",), ("bias",), ("scale",), ("shift",),
                                    ("gate", "scale"), ("weight", "shift"), ()])
def test_only_the_wanted_gradients(wanted):
    _run("between", _inputs("between", 3, 40, 96, BF16, BF16, F32), wanted=wanted)


@pytest.mark.parametrize("skip", [("out",), ("h",)])
def test_an_output_without_a_gradient(skip):
    _run("between", _inputs("between", 3, 40, 96, F32, F32, F32), skip=skip)


def test_leading_dimensions():
    from viola_amd import nn
    torch.manual_seed(8)
    row = torch.randn(64, device="cuda")
    assert nn.norm_before(row).shape == (64,)
    rows = torch.randn(2, 3, 4, 64, device="cuda")
    assert torch.equal(nn.norm_before(rows)[1, 2, 3], nn.norm_before(rows[1, 2, 3]))
    scale = torch.randn(2, 3, 1, 64, device="cuda")
    _close("h", nn.norm_before(rows, scale=scale), norms.norm(rows, scale=scale)["h"])


def test_between_is_after_then_before_in_32_bits():
    from viola_amd import nn
    torch.manual_seed(9)
    x, y, w, v = torch.randn(50, 1024).cuda(), torch.randn(50, 1024).cuda(), torch.rand(1024).cuda(), torch.rand(1024).cuda()
    out, h = nn.norm_between(x, y, w, weight=v, gate=w)
    assert torch.equal(out, nn.norm_after(x, y, w, gate=w)) and torch.equal(h, nn.norm_before(out, v))


def test_rows_far_from_zero_keep_their_digits():
    """A layer norm of values of 1000 +- 1: the mean is taken out before anything is squared. In 32 bits a value of 1000 is off by 2^-15, and the mean of a row by
    as much, against deviations of one."""
    from viola_amd import nn
    torch.manual_seed(10)
    x = 1000 + torch.randn(16, 1024)
    h = nn.norm_before(x.cuda(), kind="layer")
    expected = norms.norm(x, before="layer")["h"]
    assert (h.double().cpu() - expected).norm() <= 2.0 ** -14 * expected.norm()


def test_zero_rows_and_values_beyond_the_type():
    from viola_amd import nn
    x = torch.zeros(4, 256, device="cuda")
    h = nn.norm_before(x, kind="layer")
    assert torch.equal(h, torch.zeros_like(h)) and torch.equal(nn.norm_before(x), h)
    x = torch.randn(6, 256, device="cuda")
    x[1, 7], x[3, 9], x[5] = float("nan"), float("inf"), 1e30
    h = nn.norm_before(x)
    assert h[[0, 2, 4]].isfinite().all() and h[1].isnan().all() and h[3, 9].isnan() and (h[3].nan_to_num() == 0).all()
    assert (h[5] == 0).all()                                                 # the squares are beyond 32 bits: 1 / infinity
    _close("others", h[[0, 2, 4]], norms.norm(x[[0, 2, 4]])["h"])


def test_no_rows():
    from viola_amd import nn
    x = torch.randn(2, 0, 64, device="cuda", requires_grad=True)
    w, g = torch.ones(64, device="cuda", requires_grad=True), torch.ones(2, 1, 64, device="cuda", requires_grad=True)
    out, h = nn.norm_between(x, x, w, weight=w, gate=g)
    assert out.shape == h.shape == (2, 0, 64)
    dx, dw, dg = torch.autograd.grad([out, h], [x, w, g], [torch.zeros_like(out), torch.zeros_like(h)])
    assert dx.shape == x.shape and (dw == 0).all() and (dg == 0).all() and dg.shape == g.shape


def test_results_do_not_change_from_call_to_call():
    from viola_amd import nn
    given = {k: v.cuda().requires_grad_() for k, v in _inputs("between", 7, 300, 768, BF16, BF16, F32).items()}
    def call():
        out, h = nn.norm_between(**given)
        return (out, h, *torch.autograd.grad([out.float().sum() + h.float().square().sum()], list(given.values())))
    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))


def test_another_stream():
    """The whole pass on a stream of its own, behind inputs made there."""
    from viola_amd import nn
    given = _inputs("between", 4, 64, 512, BF16, BF16, F32)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        on = {k: v.cuda().requires_grad_() for k, v in given.items()}
        out, h = nn.norm_between(**on)
        grads = torch.autograd.grad([out, h], list(on.values()), [torch.ones_like(out), torch.ones_like(h)])
    torch.cuda.current_stream().wait_stream(side)
    expected = norms.norm(**given, dout=torch.ones(out.shape), dh=torch.ones(h.shape))
    _close("h", h, expected["h"])
    for k, g in zip(given, grads):
        _close("d" + k, g, expected["d" + k], expected["m" + k] if k not in ("x", "y") else None)


def test_directional_difference():
    """The gradients of the kernel against differences of the kernel itself, in 32 bits: along a unit direction a step of 2^-7 gives the derivative to
    about 2^-14 (its square) and 2^-24 2^7 of the values."""
    from viola_amd import nn
    torch.manual_seed(11)
    given = {k: v.cuda() for k, v in _inputs("between", 2, 8, 64, F32, F32, F32).items()}
    d_out, d_h = torch.randn(2, 8, 64, device="cuda"), torch.randn(2, 8, 64, device="cuda")

    def loss(values):
        out, h = nn.norm_between(**values, after="layer", before="rms")
        return (out.double() * d_out).sum() + (h.double() * d_h).sum()

    for k in given:
        t = given[k].clone().requires_grad_()
        grad, = torch.autograd.grad(loss({**given, k: t}), t)
        direction = torch.randn_like(t)
        direction /= direction.norm()
        step = 2.0 ** -7
        slope = (loss({**given, k: given[k] + step * direction}) - loss({**given, k: given[k] - step * direction})) / (2 * step)
        along = (grad.double() * direction).sum()
        assert abs(slope - along) <= 2.0 ** -9 * grad.norm(), (k, slope.item(), along.item())


def test_refusals():
    from viola_amd import nn
    x = torch.randn(4, 6, 64, device="cuda")
    v = torch.ones(64, device="cuda")
    for call, match in ((lambda: nn.norm_before(x.double()), "float32, bfloat16 or float16"), (lambda: nn.norm_before(x, v[:63]), "weight has to be of shape"),
                        (lambda: nn.norm_before(x, v.cpu()), "GPU only"), (lambda: nn.norm_before(x, scale=torch.ones(6, 64, device="cuda")), "neither one vector"),
                        (lambda: nn.norm_before(x, scale=torch.ones(1, 6, 64, device="cuda")), "neither one vector"),
                        (lambda: nn.norm_before(x, scale=torch.ones(4, 1, 32, device="cuda")), "has to end in 64"), (lambda: nn.norm_after(x, x[:3]), "one shape"),
                        (lambda: nn.norm_before(x, eps=-1.0), "eps"), (lambda: nn.norm_before(x[..., :0]), "features"),
                        (lambda: nn.norm_before(x, dtype=torch.float8_e4m3fn), "dtype has to be")):
        with pytest.raises(RuntimeError, match=match):
            call()
    t = x.clone().requires_grad_()
    grad, = torch.autograd.grad(nn.norm_before(t).sum(), t, retain_graph=False)
    with pytest.raises(NotImplementedError, match="once only"):
        torch.autograd.grad(nn.norm_before(t).sum(), t, create_graph=True)
    h = nn.norm_before(t * 1.0)
    h.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        h.sum().backward()
    w = v.clone().requires_grad_()
    h = nn.norm_before(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()


def test_offsets_beyond_32_bits():
    """Rows far apart: the last one begins 2^32 elements behind the first."""
    from viola_amd import nn
    pitch = (1 << 32) // 4
    store = torch.empty(pitch * 4 + 128, device="cuda", dtype=BF16)
    x = torch.as_strided(store, (5, 128), (pitch, 1))
    values = torch.randn(5, 128).bfloat16()
    x.copy_(values)
    _close("h", nn.norm_before(x), norms.norm(values)["h"])
    _close("out", nn.norm_after(x, x), norms.norm(values, values, before=None)["out"])
