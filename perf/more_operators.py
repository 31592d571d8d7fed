"""Performance cases of experts in 8-bit integers and of the router that balances them.

  route    nn.route with a bias on the choice and with groups of experts: choice, gates, places and the balance loss
  linear   nn.int8_linear: the product of 8-bit integers with a scale for each token and each channel, plain or of a gated activation
  experts  nn.int8_grouped_linear: that product for the rows of each expert, whose places the router leaves on the GPU

A training pass is forward and backward and returns the gradients too: of the router's logits, and through the products, whose weights are
fixed, of what goes in and of the bias. `own` says whether `run` makes the framework's calls or computes the same with elementary operations of
torch in 32 bits (choices and roundings to integers, where 32 bits do not settle a border, in 64); `exact` computes it in 64 bits from the formulas.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------------- the cases
def _route(sequences, length, experts, top_k, *, groups=1, top_groups=1, group_top=1, bias=True, dtype="fp32", score="sigmoid", normalize=True,
           per_sequence=False, padded=False, train=True):
    return dict(op="route", sequences=sequences, length=length, experts=experts, top_k=top_k, groups=groups, top_groups=top_groups, group_top=group_top,
                bias=bias, dtype=dtype, score=score, normalize=normalize, per_sequence=per_sequence, padded=padded, train=train)


def _linear(tokens, width, out, *, dtype="bf16", activation="none", bias=False, train=False):
    return dict(op="linear", tokens=tokens, width=width, out=out, dtype=dtype, activation=activation, bias=bias, train=train)


def _experts(rows, experts, width, out, *, dtype="bf16", activation="none", padded=False, train=False):
    return dict(op="experts", rows=rows, experts=experts, width=width, out=out, dtype=dtype, activation=activation, padded=padded, train=train)


def listed():
    cases = {
        # a decoding step of 32 sequences through a router of 256 experts in eight groups, of which four are open to a token
        "route_serve": _route(32, 1, 256, 8, groups=8, top_groups=4, group_top=2, train=False),
        # the router of a training step over 32768 tokens
        "route_train": _route(16, 2048, 256, 8, groups=8, top_groups=4, group_top=2),
        # packed sequences of odd length with padding, softmax scores under a bias, balanced sequence by sequence
        "route_softmax": _route(16, 2047, 64, 6, dtype="bf16", score="softmax", normalize=False, per_sequence=True, padded=True),
        # one token of one sequence through a small layer: the smallest call, all latency
        "linear_token": _linear(1, 1024, 4096),
        # eight sequences answering with one token each, the wide projection of a 4096-wide model: reading its weights
        "linear_serve": _linear(8, 4096, 11008),
        # the benchmark's layer, its weights fixed, with the gradients of what goes in and of its bias
        "linear_train": _linear(8192, 1024, 4096, bias=True, train=True),
        # 50 images of 196 patches and a class token into a head of 1000 classes, of a width that no piece of 16 bytes divides
        "linear_ragged": _linear(50 * 197, 770, 1000, dtype="fp16", bias=True, train=True),
        # a full batch through one branch of the benchmark's gated MLP: the largest product
        "linear_prefill": _linear(16384, 4096, 11008),
        # back from both branches of that MLP, a quarter of the batch
        "linear_down": _linear(4096, 11008, 4096, activation="silu"),
        # a decoding step's 32 tokens at eight of 64 experts each, both branches at once: a few rows an expert, reading all weights
        "experts_serve": _experts(256, 64, 4096, 2048),
        # the benchmark's expert layer, tuned through fixed weights
        "experts_train": _experts(32768, 16, 4096, 1024, train=True),
        # the gated way back from 64 small experts, some rows of the buffer without a token
        "experts_down": _experts(32768, 64, 1024, 1024, activation="silu", padded=True, train=True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, low, high):
    """An integer from low to high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """Mostly multiples of 128, some of 8, a few of nothing."""
    unit = rng.choices((128, 8, 1), (70, 20, 10))[0]
    return max(unit, _spread(rng, low, high) // unit * unit)


def _draw_route(rng):
    length = 1 if rng.random() < .25 else _spread(rng, 16, 4096)
    sequences = _spread(rng, 1, 512) if length == 1 else _spread(rng, 1, max(1, 40000 // length))
    experts = rng.choice((8, 16, 64, 128, 160, 256, 384, 512, _spread(rng, 4, 512)))
    groups = rng.choice([g for g in (1, 1, 2, 4, 8, 16) if experts % g == 0])
    top_groups = rng.randint(1, groups)
    size = experts // groups
    return _route(sequences, length, experts, rng.randint(1, min(8, size * top_groups)), groups=groups, top_groups=top_groups,
                  group_top=rng.randint(1, min(2, size)), bias=groups == 1 or rng.random() < .8, dtype=rng.choice(("fp32", "fp32", "bf16")),
                  score=rng.choice(("sigmoid", "softmax")), normalize=rng.random() < .7, per_sequence=rng.random() < .4,
                  padded=length > 1 and rng.random() < .4, train=length > 1 and rng.random() < .8)


def _draw_product(rng, op):
    activation = rng.choice(("none", "none", "silu", "gelu", "relu"))
    dtype = rng.choices(("bf16", "fp16", "fp32"), (70, 15, 15) if activation == "none" else (80, 20, 0))[0]
    few = rng.random() < .35
    if op == "linear":
        tokens = _spread(rng, 1, 64) if few else _spread(rng, 64, 16384)
        return _linear(tokens, _width(rng, 64, 8192), _width(rng, 64, 8192), dtype=dtype, activation=activation, bias=rng.random() < .5,
                       train=not few and rng.random() < .5)
    experts = rng.choice((2, 8, 16, 64, _spread(rng, 2, 96)))
    rows = _spread(rng, 1, 8 * experts) if few else _spread(rng, 64, 40000)
    return _experts(rows, experts, _width(rng, 64, 4096), _width(rng, 64, 4096), dtype=dtype, activation=activation, padded=rng.random() < .3,
                    train=not few and rng.random() < .5)


def draw(rng):
    most = [max(work(case)[key] for case in listed()) for key in ("bytes", "flops")]
    while True:
        op = rng.choices(("route", "linear", "experts"), (34, 33, 33))[0]
        case = _draw_route(rng) if op == "route" else _draw_product(rng, op)
        if all(work(case)[key] <= limit for key, limit in zip(("bytes", "flops"), most)):
            return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _normal(generator, shape, scale, dtype, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=generator) * scale + mean).to(_DTYPES[dtype])


def _prepare_route(case, generator):
    """A router's logits: some experts are liked more than others, and the bias leans against that."""
    b, s, e = case["sequences"], case["length"], case["experts"]
    liked = torch.randn(e, device="cuda", generator=generator) * 0.5
    logits = (torch.randn((b, s, e), device="cuda", generator=generator) * 1.2 + liked).to(_DTYPES[case["dtype"]])
    state = {"logits": logits.requires_grad_(case["train"]), "mask": None, "bias": None}
    if case["bias"]:
        lean = torch.randn(e, device="cuda", generator=generator) * 0.02 - liked * 0.1
        state["bias"] = lean if case["score"] == "sigmoid" else lean / e
    if case["padded"]:
        lengths = torch.randint(0, s + 1, (b, 1), device="cuda", generator=generator)
        state["mask"] = torch.arange(s, device="cuda") < lengths
    if case["train"]:
        state["gates_grad"] = _normal(generator, (b, s, case["top_k"]), 0.01, "fp32")
        state["loss_grad"] = torch.full((), 0.01, device="cuda")
    return state


def _weights(generator, shape, train):
    """Codes and scales of weights whose channels differ in size; for a training pass their transposed codes, which a program keeps beside them."""
    w = torch.randn(shape, device="cuda", generator=generator) * torch.exp(0.3 * torch.randn((*shape[:-1], 1), device="cuda", generator=generator))
    w *= shape[-1] ** -0.5
    scale = w.abs().amax(-1, keepdim=True) * (1 / 127)
    codes = (w / scale).round().clamp(-127, 127).to(torch.int8)
    return {"weight": codes, "weight_scale": scale.squeeze(-1), "weight_t": codes.transpose(-1, -2).contiguous() if train else None}


def _activations(case, generator, rows):
    """Rows whose sizes differ from token to token, with a few features larger than the rest."""
    cols = case["width"] * (1 if case["activation"] == "none" else 2)
    x = torch.randn((rows, cols), device="cuda", generator=generator) * torch.exp(0.5 * torch.randn((rows, 1), device="cuda", generator=generator))
    x *= 1 + 4 * (torch.rand(cols, device="cuda", generator=generator) < 0.01)
    return x.to(_DTYPES[case["dtype"]]).requires_grad_(case["train"])


def _prepare_linear(case, generator):
    state = _weights(generator, (case["out"], case["width"]), case["train"])
    state["x"] = _activations(case, generator, case["tokens"])
    state["bias"] = _normal(generator, (case["out"],), 0.1, "fp32").requires_grad_(case["train"]) if case["bias"] else None
    if case["train"]:
        state["grad"] = _normal(generator, (case["tokens"], case["out"]), 0.01, case["dtype"])
    return state


def _prepare_experts(case, generator):
    rows, e = case["rows"], case["experts"]
    state = _weights(generator, (e, case["out"], case["width"]), case["train"])
    state["x"] = _activations(case, generator, rows)
    liked = torch.softmax(0.5 * torch.randn(e, device="cuda", generator=generator), 0)
    used = rows - rows // 10 if case["padded"] else rows
    counts = torch.bincount(torch.multinomial(liked, used, replacement=True, generator=generator), minlength=e)
    state["offsets"] = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).to(torch.int32)
    state["room"] = int(counts.max())                                        # what a program that pads to the largest expert plans for
    if case["train"]:
        state["grad"] = _normal(generator, (rows, case["out"]), 0.01, case["dtype"])
    return state


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    make = {"route": _prepare_route, "linear": _prepare_linear, "experts": _prepare_experts}
    return {"case": case, **make[case["op"]](case, generator)}


# --------------------------------------------------------------------------------------------------------- plain forms
def _plain_choice(state):
    """The experts of each token [B, S, k] int32, -1 for none. In 64 bits: a choice between scores next to each other is a whole number."""
    case, l = state["case"], state["logits"].detach().double()
    if case["score"] == "sigmoid":
        c = 1 / (1 + torch.exp(-l))
    else:
        c = torch.exp(l - l.amax(-1, keepdim=True))
        c = c / c.sum(-1, keepdim=True)
    if state["bias"] is not None:
        c = c + state["bias"].double()
    groups = case["groups"]
    if groups > 1:
        by_group = c.unflatten(-1, (groups, -1))
        rank = torch.sort(by_group, dim=-1, descending=True).values[..., :case["group_top"]].sum(-1)
        best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :case["top_groups"]]
        kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, best, True)
        c = torch.where(kept[..., None], by_group, -math.inf).flatten(-2)
    chosen = torch.sort(c, dim=-1, descending=True, stable=True).indices[..., :case["top_k"]].to(torch.int32)
    return chosen if state["mask"] is None else torch.where(state["mask"][..., None], chosen, -1)


def _plain_route(state):
    case, logits, mask = state["case"], state["logits"], state["mask"]
    experts, k = case["experts"], case["top_k"]
    with torch.no_grad():
        chosen = _plain_choice(state)
        there = chosen >= 0
        flat = torch.where(there, chosen, experts).view(-1, k).long()
        picked = torch.zeros(flat.shape[0], experts + 1, device=flat.device, dtype=torch.int32).scatter_(-1, flat, 1)
        counts = picked[:, :experts].sum(0)
        offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
        places = (picked.cumsum(0) - picked + offsets).gather(-1, flat).view(chosen.shape)
        positions = torch.where(there, places, -1).to(torch.int32)
        picked = picked[:, :experts].view(*logits.shape).float()
    z = logits.float()
    if case["score"] == "sigmoid":
        z = z.clamp(max=0) - torch.log1p(torch.exp(-z.abs()))
    u = torch.exp(z - z.amax(-1, keepdim=True))
    p = u / u.sum(-1, keepdim=True)
    index = torch.where(there, chosen, 0).long()
    if case["normalize"]:
        gates = u.gather(-1, index)
        gates = gates / gates.sum(-1, keepdim=True)
    elif case["score"] == "softmax":
        gates = p.gather(-1, index)
    else:
        gates = (1 / (1 + torch.exp(-logits.float()))).gather(-1, index)
    gates = torch.where(there, gates, 0.0)
    counted = torch.ones_like(p[..., :1]) if mask is None else mask[..., None].float()
    axes = (1,) if case["per_sequence"] else (0, 1)
    tokens = counted.sum(axes).clamp(min=1)
    balance = ((picked.sum(axes) / (tokens * k) * ((p * counted).sum(axes) / tokens)).sum(-1) * experts).mean()
    outputs = {"gates": gates, "balance": balance, "experts": chosen, "positions": positions, "counts": counts.to(torch.int32), "offsets": offsets.to(torch.int32)}
    if not case["train"]:
        return outputs
    grad, = torch.autograd.grad([gates, balance], logits, [state["gates_grad"], state["loss_grad"]])
    return {**{key: t.detach() for key, t in outputs.items()}, "dlogits": grad}


def _codes(v):
    """(integers as floats, scales) of the rows of v in 32 bits; the quotients in 64, as a half lies between two integers."""
    scale = (v.abs().amax(-1, keepdim=True).double() / 127).float()
    return torch.where(scale > 0, v.double() / scale.double(), 0.0).round().float(), scale


def _plain_gate(g, activation):
    """(act(g), act'(g)) in 32 bits"""
    if activation == "relu":
        return g.clamp(min=0), (g > 0).float()
    if activation == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = 2 * math.sqrt(2 / math.pi)                                           # gelu as this framework has it: g (1 + tanh y) / 2 = g sigmoid(2 y)
    s = 1 / (1 + torch.exp(-c * g * (1 + 0.044715 * g * g)))
    return g * s, s + g * s * (1 - s) * c * (1 + 3 * 0.044715 * g * g)


def _plain_input(state):
    """What is quantized, in 32 bits, and how its gradient becomes that of x."""
    x, activation = state["x"].detach().float(), state["case"]["activation"]
    if activation == "none":
        return x, lambda d: d
    g, u = x.chunk(2, dim=-1)
    act, slope = _plain_gate(g, activation)
    return act * u, lambda d: torch.cat([d * u * slope, d * act], -1)


def _plain_linear(state):
    case, weight, scale = state["case"], state["weight"].float(), state["weight_scale"]
    dtype = _DTYPES[case["dtype"]]
    v, back = _plain_input(state)
    q, s = _codes(v)
    y = q @ weight.t() * s * scale
    if state["bias"] is not None:
        y = y + state["bias"].detach()
    outputs = {"y": y.to(dtype)}
    if case["train"]:
        dy = state["grad"].float()
        q, s = _codes(dy * scale)
        outputs["dx"] = back(q @ weight * s).to(dtype)
        if state["bias"] is not None:
            outputs["dbias"] = dy.sum(0)
    return outputs


def _plain_experts(state):
    case, weight, scale, offsets, room = state["case"], state["weight"].float(), state["weight_scale"], state["offsets"].long(), state["room"]
    dtype, rows, experts = _DTYPES[case["dtype"]], case["rows"], case["experts"]
    # every expert's rows padded to the largest one's, rows without an expert in one more that stays zero
    row = torch.arange(rows, device=offsets.device)
    expert = torch.searchsorted(offsets[1:], row, right=True)
    there = expert < experts
    expert = torch.where(there, expert, 0)
    at = torch.where(there, expert * room + row - offsets[expert], experts * room)

    def product(q, w):
        """q [rows, k], w [experts, n, k] -> [rows, n]"""
        padded = torch.zeros(experts * room + 1, q.shape[1], device=q.device).index_copy_(0, at, q * there[:, None])
        out = torch.bmm(w, padded[:-1].view(experts, room, -1).transpose(1, 2).contiguous()).transpose(1, 2).reshape(experts * room, -1)
        return torch.cat([out, out.new_zeros(1, out.shape[1])])[at]

    v, back = _plain_input(state)
    q, s = _codes(v)
    outputs = {"y": torch.where(there[:, None], product(q, weight) * s * scale[expert], 0.0).to(dtype)}
    if case["train"]:
        q, s = _codes(state["grad"].float() * scale[expert])
        outputs["dx"] = torch.where(there[:, None], back(product(q, weight.transpose(1, 2).contiguous()) * s), 0.0).to(dtype)
    return outputs


_PLAIN = {"route": _plain_route, "linear": _plain_linear, "experts": _plain_experts}


# -------------------------------------------------------------------------------------------------- the framework's calls
def _own_route(state):
    from viola_amd import nn
    case = state["case"]
    r = nn.route(state["logits"], case["top_k"], score=case["score"], normalize=case["normalize"], mask=state["mask"], per_sequence=case["per_sequence"],
                 bias=state["bias"], groups=case["groups"], top_groups=case["top_groups"], group_top=case["group_top"])
    outputs = {"gates": r.gates, "balance": r.balance, "experts": r.experts, "positions": r.positions, "counts": r.counts, "offsets": r.offsets}
    if not case["train"]:
        return outputs
    grad, = torch.autograd.grad([r.gates, r.balance], state["logits"], [state["gates_grad"], state["loss_grad"]])
    return {**{key: t.detach() for key, t in outputs.items()}, "dlogits": grad}


def _own_product(state):
    from viola_amd import nn
    case = state["case"]
    options = dict(activation=None if case["activation"] == "none" else case["activation"], weight_t=state["weight_t"])
    if case["op"] == "linear":
        y = nn.int8_linear(state["x"], state["weight"], state["weight_scale"], state["bias"], **options)
    else:
        y = nn.int8_grouped_linear(state["x"], state["weight"], state["weight_scale"], state["offsets"], **options)
    if not case["train"]:
        return {"y": y}
    wanted = {"dx": state["x"]}
    if state.get("bias") is not None:
        wanted["dbias"] = state["bias"]
    return {"y": y.detach(), **dict(zip(wanted, torch.autograd.grad(y, list(wanted.values()), state["grad"])))}


def run(state):
    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        if own:
            return _own_route(state) if case["op"] == "route" else _own_product(state)
        return _PLAIN[case["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Each input read once and each output written once; a gradient pass has its inputs' gradients and outputs beside them."""
    train = case["train"]
    if case["op"] == "route":
        n, e, k = case["sequences"] * case["length"], case["experts"], case["top_k"]
        return {"bytes": n * e * _BYTES[case["dtype"]] * (2 if train else 1) + n * k * (16 if train else 12) + n * case["padded"] + 4 * e * case["bias"],
                "flops": n * e * (8 + (8 if train else 0)) + n * e * k}
    m = case["tokens"] if case["op"] == "linear" else case["rows"]
    k, n, size, gated = case["width"], case["out"], _BYTES[case["dtype"]], case["activation"] != "none"
    experts = 1 if case["op"] == "linear" else min(case["experts"], m)       # weights that can be read at all
    cols = k * (2 if gated else 1)
    return {"bytes": (m * (cols + n) * size + experts * (n * k + 4 * n)) * (2 if train else 1) + (m * cols * size if train and gated else 0),
            "flops": 2 * m * n * k * (2 if train else 1)}


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_route(state):
    case, k, mask = state["case"], state["case"]["top_k"], state["mask"]
    l = state["logits"].detach().double()
    b, length, e = l.shape
    sigmoid = case["score"] == "sigmoid"
    s = torch.sigmoid(l) if sigmoid else torch.softmax(l, -1)
    c = s if state["bias"] is None else s + state["bias"].double()
    if case["groups"] > 1:
        rank = c.view(b, length, case["groups"], -1).topk(case["group_top"], -1).values.sum(-1)
        # a group is kept where fewer than top_groups are before it, of its rank those of a lower index
        before = (rank[..., None, :] > rank[..., None]) | ((rank[..., None, :] == rank[..., None]) & torch.ones(rank.shape[-1:] * 2, device=l.device, dtype=torch.bool).tril(-1))
        c = torch.where((before.sum(-1) < case["top_groups"]).repeat_interleave(e // case["groups"], -1), c, -math.inf)
    index = torch.argsort(c, dim=-1, descending=True, stable=True)[..., :k]
    there = (torch.ones(b, length, device=l.device, dtype=torch.bool) if mask is None else mask)[..., None]
    p = s / s.sum(-1, keepdim=True) * there
    picked = torch.zeros_like(p).scatter_(-1, index, 1.0) * there
    parts = b if case["per_sequence"] else 1
    tokens = there.view(parts, -1).sum(-1, keepdim=True).clamp(min=1)
    cost = e * picked.view(parts, -1, e).sum(1) / (k * tokens * tokens * parts)
    z = torch.log(s)
    if case["normalize"]:
        gates = torch.softmax(z.gather(-1, index), -1)
    else:
        gates = s.gather(-1, index)
    result = {"gates": gates * there, "balance": (cost * p.view(parts, -1, e).sum(1)).sum(), "experts": None, "positions": None, "counts": None, "offsets": None}
    if case["train"]:
        q = p.view(parts, -1, e)
        dz = (q * (cost[:, None] - (q * cost[:, None]).sum(-1, keepdim=True))).view(p.shape) * state["loss_grad"].double()
        dg = state["gates_grad"].double() * there
        dot = (dg * gates).sum(-1, keepdim=True)
        dz.scatter_add_(-1, index, gates * (dg - dot) if case["normalize"] else gates * dg)
        if not case["normalize"] and not sigmoid:
            dz -= p * dot
        result["dlogits"] = dz * torch.sigmoid(-l) if sigmoid else dz
    return result


def _exact_codes(v):
    """Integers and scales: scales are 32-bit numbers by definition."""
    scale = (v.abs().max(-1, keepdim=True).values / 127.0).to(torch.float32).double()
    return torch.nan_to_num(torch.round(v / scale)), scale


def _exact_gate(g, kind):
    if kind == "relu":
        return torch.relu(g), torch.heaviside(g, torch.zeros_like(g))
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g)
    y = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
    half = (1 + torch.tanh(y)) / 2
    return g * half, half + g / 2 / torch.cosh(y) ** 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g ** 2)


def _exact_rows(x, dy, weight, scale, bias, activation):
    """(y, dx, dbias) of the rows of one weight"""
    w, sw, x = weight.double(), scale.double(), x.double()
    h = x
    if activation != "none":
        g, u = torch.tensor_split(x, 2, dim=-1)
        act, slope = _exact_gate(g, activation)
        h = act * u
    q, s = _exact_codes(h)
    y = torch.matmul(q, w.t()) * s * sw
    if bias is not None:
        y += bias.double()
    if dy is None:
        return y, None, None
    q, s = _exact_codes(dy.double() * sw)
    dh = torch.matmul(q, w) * s
    return y, dh if activation == "none" else torch.cat([slope * dh * u, act * dh], -1), dy.double().sum(0)


def _exact_linear(state):
    bias = state["bias"]
    y, dx, dbias = _exact_rows(state["x"].detach(), state.get("grad"), state["weight"], state["weight_scale"], bias, state["case"]["activation"])
    return {"y": y, **({"dx": dx} if dx is not None else {}), **({"dbias": dbias} if dx is not None and bias is not None else {})}


def _exact_experts(state):
    case, x = state["case"], state["x"].detach()
    result = {"y": torch.zeros(case["rows"], case["out"], dtype=torch.float64, device=x.device)}
    if case["train"]:
        result["dx"] = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    bounds = state["offsets"].tolist()
    for e, (begin, end) in enumerate(zip(bounds, bounds[1:])):
        if begin == end:
            continue
        grad = state["grad"][begin:end] if case["train"] else None
        y, dx, _ = _exact_rows(x[begin:end], grad, state["weight"][e], state["weight_scale"][e], None, case["activation"])
        result["y"][begin:end] = y
        if case["train"]:
            result["dx"][begin:end] = dx
    return result


_EXACT = {"route": _exact_route, "linear": _exact_linear, "experts": _exact_experts}


def exact(case, seed):
    with torch.no_grad():
        return _EXACT[case["op"]](prepare(case, seed))
