"""Routing of a mixture of experts in 64 bits, with the gradients written out. The reference has no such operators: these are the formulas that
the entry points declare (parity unpinned); tests/test_block_operators.py holds the gradients to central differences and the rest to brute force.
"""

import math

import torch


def choose(logits, top_k, mask=None):
    """[..., top_k] indices of the largest logits: ties to the lowest, NaN above all, -inf never, -1 for none. Row by row."""
    flat = logits.detach().double().cpu().reshape(-1, logits.shape[-1])
    counted = torch.ones(flat.shape[0], dtype=torch.bool) if mask is None else mask.cpu().reshape(-1)
    chosen = torch.full((flat.shape[0], top_k), -1)
    for t, row in enumerate(flat.tolist()):
        if not counted[t]:
            continue
        order = sorted((e for e in range(len(row)) if row[e] != -math.inf), key=lambda e: (0 if row[e] != row[e] else 1, -row[e] if row[e] == row[e] else 0, e))
        for j, e in enumerate(order[:top_k]):
            chosen[t, j] = e
    return chosen.reshape(*logits.shape[:-1], top_k)


def places(chosen, experts):
    """(positions, counts, offsets): choices numbered expert by expert, within one by token."""
    flat = chosen.reshape(-1, chosen.shape[-1]).tolist()
    rows = [[] for _ in range(experts)]
    for t, row in enumerate(flat):
        for j, e in enumerate(row):
            if e >= 0:
                rows[e].append((t, j))
    positions = torch.full((len(flat), chosen.shape[-1]), -1)
    at, offsets = 0, [0]
    for list_ in rows:
        for t, j in list_:
            positions[t, j] = at
            at += 1
        offsets.append(at)
    return positions.reshape(chosen.shape), torch.tensor([len(r) for r in rows]), torch.tensor(offsets)


def probabilities(logits, score):
    """(p, logarithms of the scores, their slope in the logits); rows without a finite logit are NaN"""
    l = logits.detach().double().cpu()
    if score == "softmax":
        return torch.softmax(l, -1), l, torch.ones_like(l)
    z = torch.nn.functional.logsigmoid(l)
    return torch.softmax(z, -1), z, torch.sigmoid(-l)


def counted_tokens(logits, mask):
    counted = ~(logits.detach().double().cpu() == -math.inf).all(-1)
    return counted if mask is None else counted & mask.cpu()


def gates(logits, chosen, score, normalize, scale=1.0):
    p, z, _ = probabilities(logits, score)
    there = chosen >= 0
    index = chosen.clamp(min=0)
    if normalize:
        value = torch.softmax(torch.where(there, z.gather(-1, index), -math.inf), -1)
    else:
        value = (p if score == "softmax" else torch.sigmoid(logits.detach().double().cpu())).gather(-1, index)
    return torch.where(there, scale * value, 0.0)


def balance(logits, chosen, score, mask=None, per_sequence=False):
    """(loss, counts, costs [sequences, experts]: the loss's gradient in each probability)"""
    p, _, _ = probabilities(logits, score)
    experts, k = logits.shape[-1], chosen.shape[-1]
    counted = counted_tokens(logits, mask)
    sequences = math.prod(logits.shape[:-2]) if per_sequence else 1
    p = torch.where(counted[..., None], p, 0.0).reshape(sequences, -1, experts)
    picked = torch.zeros_like(p)
    flat, seen = chosen.cpu().long().reshape(sequences, -1, k), counted.reshape(sequences, -1, 1)
    for j in range(k):
        e = flat[..., j:j + 1]
        picked += ((torch.arange(experts) == e) & seen).double()
    n = counted.reshape(sequences, -1).sum(-1, keepdim=True).double().clamp(min=1)
    cost = experts * picked.sum(1) / (n * n * k * sequences)
    return (cost * p.sum(1)).sum(), picked.sum((0, 1)), cost


def gradient(logits, chosen, score, mask=None, per_sequence=False, *, dloss=0.0, dgates=None, normalize=True, scale=1.0):
    """The logits' gradient of dloss * balance + sum(dgates * gates)."""
    p, _, slope = probabilities(logits, score)
    counted = counted_tokens(logits, mask)[..., None]
    p = torch.where(counted, p, 0.0)
    _, _, cost = balance(logits, chosen, score, mask, per_sequence)
    cost = cost.repeat_interleave(math.prod(logits.shape[:-1]) // cost.shape[0], 0).reshape(p.shape)
    dz = dloss * p * (cost - (p * cost).sum(-1, keepdim=True))
    if dgates is not None:
        there = chosen >= 0
        dg = torch.where(there, dgates.detach().double().cpu(), 0.0)
        g = gates(logits, chosen, score, normalize, 1.0)
        dz_g = torch.zeros(*p.shape[:-1], p.shape[-1] + 1, dtype=torch.float64)
        index = torch.where(there, chosen, p.shape[-1])
        mean = (g * dg).sum(-1, keepdim=True)
        dz_g.scatter_add_(-1, index, scale * g * (dg - mean) if normalize else scale * g * dg)
        dz_g = dz_g[..., :-1]
        if not normalize and score == "softmax":
            dz_g = dz_g - scale * p * mean
        dz = dz + dz_g
    return torch.where(counted, dz * slope, 0.0)


def dispatch(x, positions, rows):
    out = torch.zeros(rows, x.shape[-1], dtype=torch.float64)
    for t, row in enumerate(positions.reshape(-1, positions.shape[-1]).tolist()):
        for r in row:
            if 0 <= r < rows:
                out[r] = x.reshape(-1, x.shape[-1])[t].double().cpu()
    return out


def combine(y, positions, gates=None):
    flat = positions.reshape(-1, positions.shape[-1])
    out = torch.zeros(flat.shape[0], y.shape[-1], dtype=torch.float64)
    y = y.detach().double().cpu()
    g = torch.ones(flat.shape) if gates is None else gates.detach().double().cpu().reshape(flat.shape)
    for t, row in enumerate(flat.tolist()):
        for j, r in enumerate(row):
            if 0 <= r < y.shape[0]:
                out[t] += g[t, j].double() * y[r]
    return out.reshape(*positions.shape[:-1], y.shape[-1])


def combine_gradient(dout, y, positions, gates=None):
    """(dy, dgates)"""
    flat = positions.reshape(-1, positions.shape[-1])
    d = dout.detach().double().cpu().reshape(flat.shape[0], -1)
    y = y.detach().double().cpu()
    g = torch.ones(flat.shape) if gates is None else gates.detach().double().cpu().reshape(flat.shape)
    dy, dg = torch.zeros_like(y), torch.zeros(flat.shape, dtype=torch.float64)
    for t, row in enumerate(flat.tolist()):
        for j, r in enumerate(row):
            if 0 <= r < y.shape[0]:
                dy[r] = g[t, j].double() * d[t]
                dg[t, j] = (d[t] * y[r]).sum()
    return dy, dg.reshape(positions.shape)


def steered_scores(logits, score, bias=None):
    """c = s + bias in 64 bits, -inf where an expert is never chosen; None for a row whose choice is by the logits alone"""
    l = logits.detach().double().cpu().reshape(-1, logits.shape[-1])
    rows = []
    for row in l:
        if bool(torch.isnan(row).any()) or (score == "softmax" and bool((row == math.inf).any())):
            rows.append(None)
            continue
        s = torch.sigmoid(row) if score == "sigmoid" else torch.softmax(row, -1)
        c = s if bias is None else s + bias.detach().double().cpu()
        rows.append([-math.inf if row[e] == -math.inf or c[e] != c[e] else c[e].item() for e in range(len(row))])
    return rows


def choose_steered(logits, top_k, score, mask=None, bias=None, groups=1, top_groups=1, group_top=1):
    """`choose` by s + bias among the experts of the top_groups runs whose group_top largest add up to most. Row by row."""
    by_logits = choose(logits, top_k, mask).reshape(-1, top_k)
    counted = (torch.ones(by_logits.shape[0], dtype=torch.bool) if mask is None else mask.cpu().reshape(-1))
    flat = logits.detach().double().cpu().reshape(-1, logits.shape[-1]).tolist()
    size = logits.shape[-1] // groups
    chosen = torch.full_like(by_logits, -1)
    for t, c in enumerate(steered_scores(logits, score, bias)):
        if not counted[t]:
            continue
        if c is None:
            chosen[t] = by_logits[t]
            continue
        ranks = []
        for g in range(groups):
            best = sorted((v for v in c[g * size:(g + 1) * size] if v > -math.inf), reverse=True)[:group_top]
            ranks.append(sum(best) if best else -math.inf)
        kept = sorted(range(groups), key=lambda g: (-ranks[g], g))[:top_groups]
        value = c if bias is not None else flat[t]
        order = sorted((e for e in range(len(c)) if e // size in kept and c[e] > -math.inf), key=lambda e: (-value[e], e))
        for j, e in enumerate(order[:top_k]):
            chosen[t, j] = e
    return chosen.reshape(*logits.shape[:-1], top_k)
