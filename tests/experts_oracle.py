"""The operators around a layer's experts by their definitions, in 64 bits, element by element where that is short."""

from __future__ import annotations

import math

import torch


def gate(logits, topk, score, renormalize, scale=1.0):
    """(weights, idx) of [tokens, experts] logits, from the definition."""
    weights = torch.zeros(logits.shape[0], topk, dtype=torch.float64)
    idx = torch.full((logits.shape[0], topk), -1)
    for t, row in enumerate(logits.double().cpu().tolist()):
        order = sorted(range(len(row)), key=lambda e: (0 if math.isnan(row[e]) else 1, -row[e] if not math.isnan(row[e]) else 0, e))
        chosen = [e for e in order[:topk] if row[e] != -math.inf]
        x = torch.tensor(row, dtype=torch.float64)
        if not chosen:
            continue
        s = torch.softmax(x, 0) if score == "softmax" else torch.sigmoid(x)
        if renormalize:  # in logarithms: the scores of a row may all be too small for a number
            log = x if score == "softmax" else torch.nn.functional.logsigmoid(x)
            w = torch.softmax(log[chosen], 0)
        else:
            w = s[chosen]
        weights[t, : len(chosen)] = scale * w
        idx[t, : len(chosen)] = torch.tensor(chosen)
    return weights, idx


def gate_gradient(logits, idx, dweights, score, renormalize, scale=1.0):
    """The logits' gradient by automatic differentiation of the definition on the choice made."""
    out = torch.zeros(logits.shape, dtype=torch.float64)
    for t in range(logits.shape[0]):
        chosen = [e for e in idx[t].tolist() if e >= 0]
        if not chosen:
            continue
        x = logits[t].double().cpu().requires_grad_()
        if renormalize:
            w = torch.softmax((x if score == "softmax" else torch.nn.functional.logsigmoid(x))[chosen], 0)
        else:
            w = (torch.softmax(x, 0) if score == "softmax" else torch.sigmoid(x))[chosen]
        d = dweights[t, : len(chosen)].double().cpu()
        out[t] = torch.autograd.grad((scale * w * d).sum(), x)[0]
    return out


def order(idx, n_experts):
    """(counts, place, source) by going through the choices once per expert."""
    flat = idx.reshape(-1).tolist()
    place, source, counts = [-1] * len(flat), [], []
    for e in range(n_experts):
        mine = [p for p, v in enumerate(flat) if v == e]
        counts.append(len(mine))
        for p in mine:
            place[p] = len(source)
            source.append(p)
    source += [-1] * (len(flat) - len(source))
    as_int = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return as_int(counts), as_int(place).view(idx.shape), as_int(source)


def take(x, place):
    """Rows of the choices, zeros behind the last, in x's type."""
    rows = torch.zeros(place.numel(), x.shape[1], dtype=x.dtype)
    token, k = (place >= 0).nonzero(as_tuple=True)
    rows[place[token, k].long()] = x[token]
    return rows


def combine(rows, place, weights=None):
    """(out, sum of magnitudes) in 64 bits."""
    out = torch.zeros(place.shape[0], rows.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    for k in range(place.shape[1]):
        token = (place[:, k] >= 0).nonzero().squeeze(1)
        y = rows[place[token, k].long()].double()
        if weights is not None:
            y = y * weights[token, k : k + 1].double()
        out[token] += y
        size[token] += y.abs()
    return out, size


def combine_gradients(dout, rows, place, weights):
    """(drows, dweights, sums of magnitudes of dweights) in 64 bits."""
    drows = torch.zeros(rows.shape, dtype=torch.float64)
    dweights = torch.zeros(place.shape, dtype=torch.float64)
    size = torch.zeros_like(dweights)
    for k in range(place.shape[1]):
        token = (place[:, k] >= 0).nonzero().squeeze(1)
        at = place[token, k].long()
        d, y = dout[token].double(), rows[at].double()
        drows[at] = d * weights[token, k : k + 1].double()
        dweights[token, k] = (d * y).sum(1)
        size[token, k] = (d * y).abs().sum(1)
    return drows, dweights, size


def half_step(dtype):
    """A rounding's largest error relative to the value."""
    return torch.finfo(dtype).eps / 2
