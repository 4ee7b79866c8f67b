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


# ---------------------------------------------------------------------------------- the product with an epilogue
def parts_of(m, rows):
    if rows is None:
        return [(None, slice(0, m))]
    parts, at = [], 0
    for e, n in enumerate(rows.tolist()):
        end = min(m, at + max(n, 0))
        parts.append((e, slice(at, end)))
        at = end
    return parts


def act(z, activation):
    if activation is None:
        return z
    if activation == "relu":
        return torch.relu(z)
    if activation == "gelu":
        return torch.nn.functional.gelu(z)
    if activation == "silu":
        return torch.nn.functional.silu(z)
    z = z.view(z.shape[0], -1, 2, 128)
    return (torch.nn.functional.silu(z[:, :, 0]) * z[:, :, 1]).reshape(z.shape[0], -1)


def product(a, b, bias, activation, residual, rows, dout=None, dtype=torch.bfloat16, out_dtype=torch.bfloat16):
    """Values in 64 bits and bounds of the error of a computation with sums in 32 bits, in a dict of (value, bound).

    Sums of n products in 32 bits are off by at most (n / 16 + 32) * 2^-23 of the sum of magnitudes (matrix instructions add 16 products at
    a time to 24 bits or more, the result of each addition once more).  An activation's slope is at most 1.13, a gated one's the
    other factor; its own evaluation is good to 2^-18.  Results are rounded once.  For the gradients z was rounded to the output's type
    (the slope's slope is at most 1 for all activations), and dz to the operands'."""
    e_out, e = half_step(out_dtype), half_step(dtype)
    tiny = 2.0**-23 if torch.float16 in (dtype, out_dtype) else 2.0**-120  # steps of numbers below the smallest normal one
    a64, b64 = a.double(), b.double()
    m, k, n = a.shape[0], a.shape[1], b.shape[-2]
    sums = lambda terms: (terms / 16 + 32) * 2.0**-23  # noqa: E731
    z, z_err = a64.new_zeros(m, n), a64.new_zeros(m, n)
    for g, part in parts_of(m, rows):
        at = slice(None) if g is None else g
        z[part] = a64[part] @ b64[at].T
        z_err[part] = sums(k) * (a64[part].abs() @ b64[at].abs().T)
        if bias is not None:
            z[part] += bias[at].double()
    z_err += 2.0**-23 * z.abs()
    taken = torch.zeros(m, 1, dtype=torch.bool, device=a.device)
    for _, part in parts_of(m, rows):
        taken[part] = True
    z.requires_grad_()
    y = torch.where(taken, act(z, activation), torch.zeros((), dtype=torch.float64, device=a.device))
    if activation == "swiglu":
        gate, up = z.detach().view(m, -1, 2, 128).unbind(2)
        ge, ue = z_err.view(m, -1, 2, 128).unbind(2)
        silu = torch.nn.functional.silu(gate).abs()
        y_err = (1.13 * ge * (up.abs() + ue) + (silu + 1.13 * ge) * ue).reshape(m, -1)
    else:
        y_err = 1.13 * z_err
    out = y.detach() + (residual.double() if residual is not None else 0)
    y_err = y_err + 2.0**-18 * y.detach().abs() + 2.0**-23 * out.abs()
    result = {"out": (out, y_err * (1 + e_out) + e_out * out.abs() + tiny)}
    if dout is None:
        return result
    (dz,) = torch.autograd.grad(y, z, dout.double())
    z = z.detach()
    # dz: the slope's error from the rounded z, its evaluation, and the rounding to the operands' type
    dz_err = e * dz.abs() + tiny
    if activation is not None:
        step = z_err + e_out * z.abs() + tiny  # error of the z that was kept
        if activation == "swiglu":
            d = dout.double().view(m, -1, 1, 128)
            gate, up = z.view(m, -1, 2, 128).unbind(2)
            s_gate, s_up = step.view(m, -1, 2, 128).unbind(2)
            d = d.squeeze(2).abs()
            to_gate = d * ((up.abs() + s_up) * s_gate + 1.13 * s_up + 2.0**-16 * (up.abs() + 1) * (gate.abs() + 1))
            to_up = d * (1.13 * s_gate + 2.0**-16 * gate.abs())
            dz_err = dz_err + torch.stack((to_gate, to_up), 2).reshape(m, -1)
        elif activation == "relu":  # a sum on the other side of zero has the whole gradient
            dz_err = dz_err + torch.where(z.abs() <= step, dout.double().abs(), torch.zeros_like(z))
        else:
            dz_err = dz_err + dout.double().abs() * (step + 2.0**-16 * (z.abs() + 1))
    da, da_err = torch.zeros_like(a64), torch.zeros_like(a64)
    db, db_err = torch.zeros_like(b64), torch.zeros_like(b64)
    dbias, dbias_err = b64.new_zeros(b.shape[:-1]), b64.new_zeros(b.shape[:-1])
    for g, part in parts_of(m, rows):
        at, count = slice(None) if g is None else g, part.stop - part.start
        da[part], da_err[part] = dz[part] @ b64[at], dz_err[part] @ b64[at].abs() + sums(n) * (dz[part].abs() @ b64[at].abs())
        db[at] = dz[part].T @ a64[part]
        db_err[at] = dz_err[part].T @ a64[part].abs() + sums(count) * (dz[part].abs().T @ a64[part].abs())
        dbias[at] = dz[part].sum(0)
        dbias_err[at] = (dz_err[part] + count * 2.0**-24 * dz[part].abs()).sum(0)
    result["da"] = da, da_err * (1 + e) + e * da.abs() + tiny
    result["db"] = db, db_err * (1 + e) + e * db.abs() + tiny
    if bias is not None:
        e_bias = half_step(bias.dtype)
        result["dbias"] = dbias, dbias_err * (1 + e_bias) + e_bias * dbias.abs() + tiny
    if residual is not None:
        result["dresidual"] = dout.double(), torch.zeros_like(out)
    return result
