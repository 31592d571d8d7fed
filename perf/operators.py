"""Performance cases of the operators around a block: norms with gate and residual, and the routing of a mixture of experts.

  norm      nn.norm_before, nn.norm_after, nn.norm_between: the norm that a block reads, the norm, gate and residual sum of
            what it gives, and the two in one pass between two blocks
  route     nn.route: a router's choice, gates, counts and places, with the balance loss
  balance   nn.balance_loss: the balance loss and the counts of choices that are already made
  dispatch  nn.dispatch: the rows of the tokens in the order of the experts
  combine   nn.combine: the sum of the experts' rows of each token under its gates

A training pass is forward and backward and returns the gradients too. `own` says whether `run` makes the framework's calls or
computes the same with elementary operations of torch in 32 bits; `exact` computes it in 64 bits from the formulas.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------- the cases
def _norm(form, sequences, length, width, *, stream="bf16", branch="bf16", after="rms", before="rms", weights=True, bias=False,
          gate="none", modulated=False, residual=1.0, train=True):
    return dict(op="norm", form=form, sequences=sequences, length=length, width=width, stream=stream, branch=branch, after=after,
                before=before, weights=weights, bias=bias, gate=gate, modulated=modulated, residual=residual, train=train)


def _route(sequences, length, experts, top_k, *, dtype="fp32", score="softmax", normalize=True, per_sequence=False, padded=False, train=True):
    return dict(op="route", sequences=sequences, length=length, experts=experts, top_k=top_k, dtype=dtype, score=score,
                normalize=normalize, per_sequence=per_sequence, padded=padded, train=train)


def _balance(sequences, length, experts, top_k, *, dtype="fp32", score="softmax", per_sequence=False, padded=False, train=True):
    return dict(op="balance", sequences=sequences, length=length, experts=experts, top_k=top_k, dtype=dtype, score=score,
                per_sequence=per_sequence, padded=padded, train=train)


def _rows(op, tokens, width, experts, top_k, *, dtype="bf16", padded=False, train=True):
    return dict(op=op, tokens=tokens, width=width, experts=experts, top_k=top_k, dtype=dtype, padded=padded, train=train)


def listed():
    cases = {
        # eight sequences answering with one token each, between two blocks: the smallest call, all latency
        "norm_serve": _norm("between", 8, 1, 1024, gate="vector", train=False),
        # the diffusion transformer's block (width 1152): no norm after, a gate, scale and shift for each image
        "norm_dit": _norm("between", 64, 256, 1152, after=None, before="layer", weights=False, gate="sequence", modulated=True),
        # norms on both sides of every block of a 4096-wide model under a layer scale, a full batch: the largest call
        "norm_sandwich": _norm("between", 8, 2048, 4096, gate="vector"),
        # 50 images of 196 patches and a class token, a 32-bit residual stream read by a 16-bit block
        "norm_ragged": _norm("before", 50, 197, 768, stream="fp32", branch="fp16", before="layer", bias=True),
        # a decoding step of 32 sequences through a router of 128 experts
        "route_serve": _route(32, 1, 128, 8, train=False),
        # the router of a training step over the benchmark's 32768 rows, many small experts
        "route_train": _route(16, 2048, 128, 8),
        # the classic pair of experts out of 16, choices made elsewhere
        "balance_pair": _balance(8, 2048, 16, 2),
        # sigmoid scores, packed sequences of odd length with padding, balanced sequence by sequence
        "balance_sequences": _balance(16, 2047, 256, 8, dtype="bf16", score="sigmoid", per_sequence=True, padded=True),
        # a decoding step's tokens to their two experts
        "dispatch_serve": _rows("dispatch", 32, 4096, 16, 2, train=False),
        # 16384 tokens to two of 16 experts: the 32768 rows of the benchmark's expert layer
        "dispatch_train": _rows("dispatch", 16384, 4096, 16, 2),
        # a ragged batch of images with padding, one expert for each token
        "combine_ragged": _rows("combine", 50 * 197, 768, 8, 1, dtype="fp16", padded=True),
        # back from the benchmark's expert layer (1024 wide), eight experts for each token
        "combine_train": _rows("combine", 16384, 1024, 64, 8),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    """An integer from low to high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """Mostly multiples of 128, some of 8, a few of nothing."""
    unit = rng.choices((128, 8, 1), (70, 20, 10))[0]
    return max(unit, _spread(rng, low, high) // unit * unit)


def _batch(rng, most):
    """(sequences, length): one token each in a quarter of the cases."""
    if rng.random() < .25:
        return _spread(rng, 1, 512), 1
    length = _spread(rng, 16, 4096)
    return _spread(rng, 1, max(1, most // length)), length


def draw(rng):
    most = max(work(case)["bytes"] for case in listed())
    while True:
        op = rng.choices(("norm", "route", "balance", "dispatch", "combine"), (40, 20, 14, 13, 13))[0]
        dtype = rng.choices(("bf16", "fp16", "fp32"), (60, 20, 20))[0]
        if op == "norm":
            sequences, length = _batch(rng, 32768)
            form = rng.choice(("between", "between", "before", "after"))
            weights = rng.random() < .7
            case = _norm(form, sequences, length, _width(rng, 64, 8192), stream="fp32" if rng.random() < .3 else dtype, branch=dtype,
                         after=rng.choice(("rms", "layer", None)) if form == "between" else rng.choice(("rms", "layer")), before=rng.choice(("rms", "layer")),
                         weights=weights, bias=weights and rng.random() < .3, gate=rng.choice(("none", "vector", "sequence")),
                         modulated=rng.random() < .4, residual=rng.choice((1.0, 1.0, 0.7)), train=length > 1 and rng.random() < .8)
        elif op in ("route", "balance"):
            sequences, length = _batch(rng, 65536)
            experts = rng.choice((_spread(rng, 4, 512), 8, 16, 64, 128, 256))
            options = dict(dtype=rng.choice(("fp32", "bf16")), score=rng.choice(("softmax", "sigmoid")), per_sequence=rng.random() < .4, padded=length > 1 and rng.random() < .4,
                           train=length > 1 and rng.random() < .8)
            if op == "route":
                options["normalize"] = rng.random() < .7
            case = (_route if op == "route" else _balance)(sequences, length, experts, rng.randint(1, min(8, experts)), **options)
        else:
            tokens, train = (_spread(rng, 1, 256), False) if rng.random() < .25 else (_spread(rng, 64, 32768), rng.random() < .8)
            experts = rng.choice((8, 16, 64, _spread(rng, 2, 256)))
            case = _rows(op, tokens, _width(rng, 64, 8192), experts, rng.randint(1, min(8, experts)), dtype=dtype, padded=rng.random() < .3, train=train)
        if work(case)["bytes"] <= most:
            return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _normal(generator, shape, scale, dtype, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=generator) * scale + mean).to(_DTYPES[dtype])


def _prepare_norm(case, generator):
    b, s, c = case["sequences"], case["length"], case["width"]
    stream, branch, form = case["stream"], case["branch"], case["form"]
    inputs = {"x": _normal(generator, (b, s, c), 1.0, stream)}
    if form != "before":
        inputs["y"] = _normal(generator, (b, s, c), 0.5, branch)
        if case["weights"] and case["after"]:
            inputs["after_weight"] = _normal(generator, (c,), 0.1, "fp32", 1.0)
            if case["bias"]:
                inputs["after_bias"] = _normal(generator, (c,), 0.1, "fp32")
        if case["gate"] == "vector":
            inputs["gate"] = _normal(generator, (c,), 0.1, "fp32", 0.3)
    if form != "after" and case["weights"]:
        inputs["weight"] = _normal(generator, (c,), 0.1, "fp32", 1.0)
        if case["bias"]:
            inputs["bias"] = _normal(generator, (c,), 0.1, "fp32")
    # what one projection of a sequence's condition gives, cut into its parts
    parts = _normal(generator, (b, 6 * c), 0.3, branch)
    if form != "before" and case["gate"] == "sequence":
        inputs["gate"] = parts[:, None, :c]
    if form != "after" and case["modulated"]:
        inputs["scale"], inputs["shift"] = parts[:, None, c:2 * c], parts[:, None, 2 * c:3 * c]
    grads = {}
    if case["train"]:
        inputs = {key: t.detach().requires_grad_() for key, t in inputs.items()}
        if form != "before":
            grads["out"] = _normal(generator, (b, s, c), 0.01, stream)
        if form != "after":
            grads["h"] = _normal(generator, (b, s, c), 0.01, branch)
    return {"inputs": inputs, "grads": grads}


def _logits(case, generator):
    """A router's logits: some experts are liked more than others."""
    shape = (case["sequences"], case["length"], case["experts"])
    liked = torch.randn(case["experts"], device="cuda", generator=generator) * 0.5
    logits = (torch.randn(shape, device="cuda", generator=generator) * 1.2 + liked).to(_DTYPES[case["dtype"]])
    mask = None
    if case["padded"]:
        lengths = torch.randint(0, case["length"] + 1, (case["sequences"], 1), device="cuda", generator=generator)
        mask = torch.arange(case["length"], device="cuda") < lengths
    return logits, mask


def _prepare_route(case, generator):
    logits, mask = _logits(case, generator)
    state = {"logits": logits.requires_grad_(case["train"]), "mask": mask}
    if case["train"]:
        state["gates_grad"] = _normal(generator, (case["sequences"], case["length"], case["top_k"]), 0.01, "fp32")
        state["loss_grad"] = torch.full((), 0.01, device="cuda")
    return state


def _prepare_balance(case, generator):
    logits, mask = _logits(case, generator)
    # chosen under a bias that the scores do not have, as a router that steers its experts' load does
    steered = logits.float() + torch.randn(case["experts"], device="cuda", generator=generator) * 0.5
    chosen = steered.topk(case["top_k"], dim=-1).indices.to(torch.int32)
    if mask is not None:
        chosen = torch.where(mask[..., None], chosen, -1)
    return {"logits": logits.requires_grad_(case["train"]), "mask": mask, "experts": chosen, "loss_grad": torch.full((), 0.01, device="cuda")}


def _prepare_rows(case, generator):
    t, c, e, k = case["tokens"], case["width"], case["experts"], case["top_k"]
    liked = torch.rand(t, e, device="cuda", generator=generator) + 0.3 * torch.rand(e, device="cuda", generator=generator)
    chosen = liked.topk(k, dim=-1).indices
    if case["padded"]:
        chosen = torch.where(torch.rand(t, 1, device="cuda", generator=generator) < 0.85, chosen, e)
    flat = chosen.flatten()
    order = torch.argsort(flat, stable=True)
    places = torch.empty_like(flat)
    places[order] = torch.arange(t * k, device="cuda")
    counts = torch.bincount(flat, minlength=e + 1)[:e]
    state = {"positions": torch.where(chosen < e, places.view(t, k), -1).to(torch.int32),
             "offsets": torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)}
    if case["op"] == "dispatch":
        state["x"] = _normal(generator, (t, c), 1.0, case["dtype"]).requires_grad_(case["train"])
        if case["train"]:
            state["rows_grad"] = _normal(generator, (t * k, c), 0.01, case["dtype"])
    else:
        gates = torch.sigmoid(torch.randn(t, k, device="cuda", generator=generator))
        state["gates"] = torch.where(chosen < e, gates, 0.0).requires_grad_(case["train"])
        state["y"] = _normal(generator, (t * k, c), 0.5, case["dtype"]).requires_grad_(case["train"])
        if case["train"]:
            state["out_grad"] = _normal(generator, (t, c), 0.01, case["dtype"])
    return state


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    make = {"norm": _prepare_norm, "route": _prepare_route, "balance": _prepare_balance, "dispatch": _prepare_rows, "combine": _prepare_rows}
    return {"case": case, **make[case["op"]](case, generator)}


# --------------------------------------------------------------------------------------------------------- plain forms
def _plain_normed(v, kind, weight, bias):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
    if weight is not None:
        v = v * weight
    return v if bias is None else v + bias


def _plain_norm(state):
    case, i = state["case"], {key: t.float() for key, t in state["inputs"].items()}
    outputs, x = {}, i["x"]
    if case["form"] != "before":
        branch = _plain_normed(i["y"], case["after"], i.get("after_weight"), i.get("after_bias"))
        if "gate" in i:
            branch = branch * i["gate"]
        x = x * case["residual"] + branch
        outputs["out"] = x.to(_DTYPES[case["stream"]])
    if case["form"] != "after":
        h = _plain_normed(x, case["before"], i.get("weight"), i.get("bias"))
        if "scale" in i:
            h = h * (1 + i["scale"]) + i["shift"]
        outputs["h"] = h.to(_DTYPES[case["branch"]])
    return outputs


def _plain_scores(logits, score):
    """Logarithms of scores, up to one number for each row."""
    z = logits.float()
    return z if score == "softmax" else z.clamp(max=0) - torch.log1p(torch.exp(-z.abs()))


def _plain_balance(z, chosen, mask, per_sequence):
    """(loss, counts of all tokens) for chosen [B, S, k], -1 for none."""
    experts = z.shape[-1]
    counted = torch.ones_like(chosen[..., :1], dtype=torch.float32) if mask is None else mask[..., None].float()
    picked = torch.zeros(*z.shape[:-1], experts + 1, device=z.device).scatter_(-1, torch.where(chosen < 0, experts, chosen).long(), 1.0)[..., :experts] * counted
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True) * counted
    axes = (1,) if per_sequence else (0, 1)
    tokens = counted.sum(axes).clamp(min=1)
    loss = (picked.sum(axes) / (tokens * chosen.shape[-1]) * (p.sum(axes) / tokens)).sum(-1) * experts
    return loss.mean(), picked.sum((0, 1)).to(torch.int32)


def _plain_route(state):
    case, logits, mask = state["case"], state["logits"], state["mask"]
    experts, k = case["experts"], case["top_k"]
    with torch.no_grad():
        chosen = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[..., :k].to(torch.int32)
        if mask is not None:
            chosen = torch.where(mask[..., None], chosen, -1)
        there = chosen >= 0
        flat = torch.where(there, chosen, experts).view(-1, k).long()
        picked = torch.zeros(flat.shape[0], experts + 1, device=flat.device, dtype=torch.int32).scatter_(-1, flat, 1)
        counts = picked[:, :experts].sum(0)
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        places = (picked.cumsum(0) - picked + offsets).gather(-1, flat).view(chosen.shape)
        positions = torch.where(there, places, -1).to(torch.int32)
    z = _plain_scores(logits, case["score"])
    index = torch.where(there, chosen, 0).long()
    if case["normalize"]:
        gates = torch.exp((z - z.amax(-1, keepdim=True)).gather(-1, index))
        gates = gates / gates.sum(-1, keepdim=True)
    elif case["score"] == "softmax":
        p = torch.exp(z - z.amax(-1, keepdim=True))
        gates = (p / p.sum(-1, keepdim=True)).gather(-1, index)
    else:
        gates = (1 / (1 + torch.exp(-logits.float()))).gather(-1, index)
    gates = torch.where(there, gates, 0.0)
    loss, _ = _plain_balance(z, chosen, mask, case["per_sequence"])
    return {"gates": gates, "balance": loss, "experts": chosen, "positions": positions, "counts": counts.to(torch.int32), "offsets": offsets.to(torch.int32)}


def _plain_balance_loss(state):
    case = state["case"]
    loss, counts = _plain_balance(_plain_scores(state["logits"], case["score"]), state["experts"], state["mask"], case["per_sequence"])
    return {"balance": loss, "counts": counts}


def _plain_dispatch(state):
    x, positions = state["x"], state["positions"]
    t, k = positions.shape
    # rows without a token stay zero: places that name none go to one more row, which is cut off
    at = torch.where(positions < 0, t * k, positions).flatten().long()
    rows = torch.zeros(t * k + 1, x.shape[1], device=x.device).index_put((at,), x.float().repeat_interleave(k, 0))
    return {"rows": rows[:-1].to(x.dtype)}


def _plain_combine(state):
    y, gates, positions = state["y"], state["gates"], state["positions"]
    there = positions >= 0
    rows = y.float()[torch.where(there, positions, 0).long()]
    return {"out": (torch.where(there, gates, 0.0)[..., None] * rows).sum(1).to(y.dtype)}


_PLAIN = {"norm": _plain_norm, "route": _plain_route, "balance": _plain_balance_loss, "dispatch": _plain_dispatch, "combine": _plain_combine}


# -------------------------------------------------------------------------------------------------- the framework's calls
def _own_norm(state):
    from viola_amd import nn
    case, i = state["case"], state["inputs"]
    after = dict(gate=i.get("gate"), residual_scale=case["residual"])
    before = dict(scale=i.get("scale"), shift=i.get("shift"))
    if case["form"] == "before":
        return {"h": nn.norm_before(i["x"], i.get("weight"), i.get("bias"), kind=case["before"], eps=_EPS, dtype=_DTYPES[case["branch"]], **before)}
    if case["form"] == "after":
        return {"out": nn.norm_after(i["x"], i["y"], i.get("after_weight"), i.get("after_bias"), kind=case["after"], eps=_EPS, **after)}
    out, h = nn.norm_between(i["x"], i["y"], i.get("after_weight"), i.get("after_bias"), i.get("weight"), i.get("bias"), after=case["after"],
                             before=case["before"], eps=_EPS, **after, **before)
    return {"out": out, "h": h}


def _own_route(state):
    from viola_amd import nn
    case = state["case"]
    r = nn.route(state["logits"], case["top_k"], score=case["score"], normalize=case["normalize"], mask=state["mask"], per_sequence=case["per_sequence"])
    return {"gates": r.gates, "balance": r.balance, "experts": r.experts, "positions": r.positions, "counts": r.counts, "offsets": r.offsets}


def _own_balance(state):
    from viola_amd import nn
    case = state["case"]
    loss, counts = nn.balance_loss(state["logits"], state["experts"], score=case["score"], mask=state["mask"], per_sequence=case["per_sequence"])
    return {"balance": loss, "counts": counts}


def _own_dispatch(state):
    from viola_amd import nn
    return {"rows": nn.dispatch(state["x"], nn.Routing(positions=state["positions"], offsets=state["offsets"]))}


def _own_combine(state):
    from viola_amd import nn
    return {"out": nn.combine(state["y"], nn.Routing(positions=state["positions"], offsets=state["offsets"], gates=state["gates"]))}


_OWN = {"norm": _own_norm, "route": _own_route, "balance": _own_balance, "dispatch": _own_dispatch, "combine": _own_combine}


def run(state):
    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        outputs = (_OWN if own else _PLAIN)[case["op"]](state)
    if not case["train"]:
        return outputs
    wanted, given = _gradients(state)
    grads = torch.autograd.grad([outputs[key] for key in given], list(wanted.values()), list(given.values()))
    return {**{key: t.detach() for key, t in outputs.items()}, **{"d" + key: g for key, g in zip(wanted, grads)}}


def _gradients(state):
    """(inputs by name, gradients of the outputs by name) of a training pass."""
    op = state["case"]["op"]
    if op == "norm":
        return state["inputs"], state["grads"]
    if op == "route":
        return {"logits": state["logits"]}, {"gates": state["gates_grad"], "balance": state["loss_grad"]}
    if op == "balance":
        return {"logits": state["logits"]}, {"balance": state["loss_grad"]}
    if op == "dispatch":
        return {"x": state["x"]}, {"rows": state["rows_grad"]}
    return {"y": state["y"], "gates": state["gates"]}, {"out": state["out_grad"]}


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Each input read once and each output written once; a gradient pass has its inputs' gradients and outputs beside them."""
    train = case["train"]
    if case["op"] == "norm":
        n, c, form = case["sequences"] * case["length"], case["width"], case["form"]
        stream, branch = _BYTES[case["stream"]], _BYTES[case["branch"]]
        per = stream + (branch if form != "before" else 0) + (stream if form != "before" else 0) + (branch if form != "after" else 0)
        sides = (form != "before") + (form != "after")
        vectors = case["sequences"] * c * branch * (case["modulated"] * 2 * (form != "after") + (case["gate"] == "sequence") * (form != "before"))
        # the backward pass has as many tensors again: a gradient for each input and each output
        return {"bytes": (n * c * per + vectors + 4 * c * sides) * (2 if train else 1), "flops": n * c * (8 * sides + (20 * sides if train else 0))}
    if case["op"] in ("route", "balance"):
        n, e, k = case["sequences"] * case["length"], case["experts"], case["top_k"]
        choice = n * k * (12 + (4 if train else 0)) if case["op"] == "route" else n * k * 4
        return {"bytes": n * e * _BYTES[case["dtype"]] * (2 if train else 1) + choice + n * case["padded"],
                "flops": n * e * (6 + (8 if train else 0)) + (n * e * k if case["op"] == "route" else 0)}
    t, c, k, size = case["tokens"], case["width"], case["top_k"], _BYTES[case["dtype"]]
    places = t * k * 4
    if case["op"] == "dispatch":
        return {"bytes": t * c * (1 + k) * size * (2 if train else 1) + places, "flops": t * c * k if train else 0}
    return {"bytes": (t * c * (1 + k) * size + places) * (2 if train else 1) + places, "flops": t * c * k * (6 if train else 2)}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _statistics(v, kind):
    """(v's deviation over its size, one over that size)"""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
    r = (((v - mean) ** 2).mean(-1, keepdim=True) + _EPS) ** -0.5
    return (v - mean) * r, r


def _norm_gradient(q, hat, r, kind):
    """The gradient of v from that of its normed values `hat`."""
    q_hat = (q * hat).mean(-1, keepdim=True)
    return r * (q - hat * q_hat - (q.mean(-1, keepdim=True) if kind == "layer" else 0.0))


def _exact_norm(state):
    case, form = state["case"], state["case"]["form"]
    i = {key: t.detach().double() for key, t in state["inputs"].items()}
    x, rho = i["x"], case["residual"]
    result, d = {}, {}
    w_a, b_a, g = i.get("after_weight", 1.0), i.get("after_bias", 0.0), i.get("gate", 1.0)
    w_b, b_b, s, t = i.get("weight", 1.0), i.get("bias", 0.0), i.get("scale", 0.0), i.get("shift", 0.0)
    if form != "before":
        y_hat, y_r = _statistics(i["y"], case["after"]) if case["after"] else (i["y"], 1.0)
        x = rho * x + g * (y_hat * w_a + b_a)
        result["out"] = x
    if form != "after":
        x_hat, x_r = _statistics(x, case["before"])
        result["h"] = (x_hat * w_b + b_b) * (1 + s) + t
    if not case["train"]:
        return result
    grads = {key: v.double() for key, v in state["grads"].items()}
    along = grads.get("out", 0.0)
    if form != "after":
        dh = grads["h"]
        along = along + _norm_gradient(dh * (1 + s) * w_b, x_hat, x_r, case["before"])
        d.update(weight=dh * (1 + s) * x_hat, bias=dh * (1 + s), scale=dh * (x_hat * w_b + b_b), shift=dh)
    d["x"] = along
    if form != "before":
        d["x"] = rho * along
        d["y"] = _norm_gradient(along * g * w_a, y_hat, y_r, case["after"]) if case["after"] else along * g
        d.update(after_weight=along * g * y_hat, after_bias=along * g, gate=along * (y_hat * w_a + b_a))
    return {**result, **{"d" + key: d[key].sum_to_size(v.shape) for key, v in i.items()}}


def _exact_scores(logits, score):
    """(p, gradient of the scores' logarithms, logarithms of the scores)"""
    l = logits.detach().double()
    if score == "softmax":
        return torch.softmax(l, -1), torch.ones_like(l), l
    return torch.sigmoid(l) / torch.sigmoid(l).sum(-1, keepdim=True), torch.sigmoid(-l), -torch.log(1 + torch.exp(-l))


def _exact_balance(state, p, chosen):
    """(loss, counts, gradient of the logarithms of the scores for a loss gradient of one)"""
    case = state["case"]
    b, length, e = p.shape
    mask = state["mask"] if state["mask"] is not None else torch.ones(b, length, dtype=torch.bool, device=p.device)
    picked = torch.zeros_like(p)
    for j in range(case["top_k"]):
        picked += (torch.arange(e, device=p.device) == chosen[..., j:j + 1]) * mask[..., None]
    p = p * mask[..., None]
    parts = b if case["per_sequence"] else 1
    q, c, n = p.view(parts, -1, e), picked.view(parts, -1, e).sum(1), mask.view(parts, -1).sum(1, keepdim=True).clamp(min=1)
    cost = e * c / (case["top_k"] * n * n * parts)
    loss = (cost * q.sum(1)).sum()
    pull = q * (cost[:, None] - (q * cost[:, None]).sum(-1, keepdim=True))
    return loss, c.sum(0), pull.view(p.shape) * mask[..., None]


def _exact_route(state):
    case, logits, k = state["case"], state["logits"], state["case"]["top_k"]
    p, slope, z = _exact_scores(logits, case["score"])
    left, chosen = logits.detach().double().clone(), []
    for _ in range(k):
        best = left.amax(-1, keepdim=True)
        first = torch.where(left == best, torch.arange(case["experts"], device=left.device), case["experts"]).amin(-1, keepdim=True)
        chosen.append(first)
        left.scatter_(-1, first, -math.inf)
    index = torch.cat(chosen, -1)
    there = torch.ones_like(index, dtype=torch.bool) if state["mask"] is None else state["mask"][..., None].expand_as(index)
    loss, counts, pull = _exact_balance(state, p, torch.where(there, index, -1))
    if case["normalize"]:
        gates = torch.softmax(z.gather(-1, index), -1)
    else:
        gates = p.gather(-1, index) if case["score"] == "softmax" else torch.sigmoid(logits.detach().double()).gather(-1, index)
    result = {"gates": gates * there, "balance": loss, "experts": None, "positions": None, "counts": None, "offsets": None}
    if case["train"]:
        dg = state["gates_grad"].double() * there
        dot = (dg * gates).sum(-1, keepdim=True)
        dz = pull * state["loss_grad"].double()
        if case["normalize"]:
            dz.scatter_add_(-1, index, gates * (dg - dot * there))
        else:
            dz.scatter_add_(-1, index, gates * dg)
            if case["score"] == "softmax":
                dz -= p * dot
        result["dlogits"] = dz * slope
    return result


def _exact_balance_loss(state):
    p, slope, _ = _exact_scores(state["logits"], state["case"]["score"])
    loss, _, pull = _exact_balance(state, p, state["experts"])
    result = {"balance": loss, "counts": None}
    if state["case"]["train"]:
        result["dlogits"] = pull * slope * state["loss_grad"].double()
    return result


def _exact_dispatch(state):
    x, positions = state["x"].detach().double(), state["positions"].long()
    t, k = positions.shape
    rows, dx = torch.zeros(t * k, x.shape[1], dtype=torch.float64, device=x.device), torch.zeros_like(x)
    for j in range(k):
        token = (positions[:, j] >= 0).nonzero()[:, 0]
        rows[positions[token, j]] = x[token]
        if state["case"]["train"]:
            dx[token] += state["rows_grad"][positions[token, j]].double()
    return {"rows": rows, "dx": dx} if state["case"]["train"] else {"rows": rows}


def _exact_combine(state):
    y, gates, positions = state["y"].detach(), state["gates"].detach().double(), state["positions"].long()
    t, k = positions.shape
    train = state["case"]["train"]
    out = torch.zeros(t, y.shape[1], dtype=torch.float64, device=y.device)
    dy, dgates = torch.zeros(y.shape, dtype=torch.float64, device=y.device), torch.zeros_like(gates)
    for j in range(k):
        token = (positions[:, j] >= 0).nonzero()[:, 0]
        rows = y[positions[token, j]].double()
        out[token] += gates[token, j, None] * rows
        if train:
            d = state["out_grad"][token].double()
            dy[positions[token, j]] = gates[token, j, None] * d
            dgates[token, j] = (d * rows).sum(-1)
    return {"out": out, "dy": dy, "dgates": dgates} if train else {"out": out}


_EXACT = {"norm": _exact_norm, "route": _exact_route, "balance": _exact_balance_loss, "dispatch": _exact_dispatch, "combine": _exact_combine}


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["op"]](prepare(case, seed))
