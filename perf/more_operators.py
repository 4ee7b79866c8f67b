"""Performance cases of the operators around and inside a mixture-of-experts layer in 16 and 32 bits, for training and serving.

Four kinds of work, all through the public entry points of ``lplb_b200.ops``:

* ``gate``     ``gate_topk``: a router's logits to the chosen experts and their weights, and the logits' gradient
* ``sort``     ``expert_order`` and ``take_rows``: tokens sorted by expert, and the gradient of the tokens
* ``combine``  ``combine_rows``: the experts' rows back to their tokens, weighted, and the gradients of rows and weights
* ``matmul``   ``matmul``: a product with bias, activation and residual in its epilogue, of one matrix or of the sorted rows of many
               experts, and the gradients of everything that went in

With ``own`` false the same operators run in elementary torch operations in 32 bits.
"""

import math

import torch

own = False

BLOCK = 128  # gate rows in front of their up rows in the weights of a "swiglu" product


def listed():
    return [
        # the router's choice in a decode step of a few sequences
        dict(name="gate_decode", kind="gate", tokens=16, experts=256, topk=8, dtype="float32", score="sigmoid", renormalize=True,
             padded=False, grad=False),
        # the same over a training batch of the headline workload (256 experts), with the logits' gradient
        dict(name="gate_train", kind="gate", tokens=8192, experts=256, topk=8, dtype="float32", score="softmax", renormalize=False,
             padded=False, grad=True),
        # a decode step: 64 tokens to the 48 physical experts of the layer benchmark
        dict(name="sort_decode", kind="sort", tokens=64, topk=8, experts=48, hidden=7168, dtype="bfloat16", padded=False, grad=False),
        # a ragged batch with padded tokens, rows that are no whole number of sectors
        dict(name="sort_ragged", kind="sort", tokens=1001, topk=6, experts=160, hidden=2065, dtype="float32", padded=True, grad=True),
        # a training batch of the layer benchmark: 256 + 16 physical experts
        dict(name="sort_train", kind="sort", tokens=8192, topk=8, experts=272, hidden=7168, dtype="bfloat16", padded=False, grad=True),
        # the way back in a decode step
        dict(name="combine_decode", kind="combine", tokens=64, topk=8, experts=48, hidden=7168, dtype="bfloat16", padded=False,
             grad=False),
        # the way back in training, with the gradients of the experts' rows and of the weights
        dict(name="combine_train", kind="combine", tokens=8192, topk=8, experts=272, hidden=7168, dtype="bfloat16", padded=False,
             grad=True),
        # down projection of one token onto the residual stream
        dict(name="matmul_token", kind="matmul", experts=0, rows=1, n=7168, k=2048, dtype="bfloat16", out="bfloat16", bias=False,
             activation=None, residual=True, spare=False, grad=False),
        # gate and up projection of a decode batch with the activation
        dict(name="matmul_decode", kind="matmul", experts=0, rows=64, n=4096, k=7168, dtype="bfloat16", out="bfloat16", bias=False,
             activation="swiglu", residual=False, spare=False, grad=False),
        # odd sizes of a model in half precision, everything in the epilogue, result in 32 bits, with all gradients
        dict(name="matmul_ragged", kind="matmul", experts=0, rows=1001, n=4100, k=2064, dtype="float16", out="float32", bias=True,
             activation="gelu", residual=True, spare=False, grad=True),
        # a dense projection of a prefill batch (tensor bound)
        dict(name="matmul_prefill", kind="matmul", experts=0, rows=8192, n=4096, k=7168, dtype="bfloat16", out="bfloat16", bias=True,
             activation="silu", residual=False, spare=False, grad=False),
        # the first product of 32 experts in training: the sorted rows of a batch, some experts nearly idle
        dict(name="matmul_experts", kind="matmul", experts=32, rows=16384, n=4096, k=7168, dtype="bfloat16", out="bfloat16", bias=False,
             activation="swiglu", residual=False, spare=False, grad=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["gate", "sort", "combine", "matmul", "matmul", "matmul"])
    topk = rng.choice([1, 2, 4, 6, 8])
    if kind == "gate":
        return dict(kind=kind, tokens=_spread(rng, 1, 8192), experts=rng.randint(topk, 256), topk=topk,
                    dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]), score=rng.choice(["softmax", "sigmoid"]),
                    renormalize=rng.random() < 0.5, padded=rng.random() < 0.3, grad=rng.random() < 0.6)
    if kind != "matmul":
        hidden = rng.choice([_spread(rng, 65, 3500), 8 * _spread(rng, 16, 896)])
        return dict(kind=kind, tokens=_spread(rng, 1, 8192), topk=topk, experts=_spread(rng, 8, 272), hidden=hidden,
                    dtype=rng.choice(["bfloat16", "float16", "float32" if hidden <= 3500 else "bfloat16"]),
                    padded=rng.random() < 0.3, grad=rng.random() < 0.6)
    experts = rng.choice([0, 0, 0, rng.randint(2, 32)])
    activation = rng.choice([None, None, "silu", "gelu", "relu", "swiglu", "swiglu"])
    n = 256 * _spread(rng, 1, 16) if activation == "swiglu" else rng.choice([_spread(rng, 33, 4096), 8 * _spread(rng, 8, 512)])
    return dict(kind=kind, experts=experts, rows=_spread(rng, max(1, experts), 8192), n=n, k=8 * _spread(rng, 16, 896),
                dtype=rng.choice(["bfloat16", "bfloat16", "float16"]), out=rng.choice(["same", "same", "float32"]),
                bias=rng.random() < 0.5, activation=activation, residual=rng.random() < 0.4,
                spare=experts > 0 and rng.random() < 0.3, grad=rng.random() < 0.6)


def _out_type(case):
    return getattr(torch, case["dtype"] if case["out"] == "same" else case["out"])


def _out_cols(case):
    return case["n"] // 2 if case["activation"] == "swiglu" else case["n"]


# ---------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _logits(g, tokens, experts):
    """N(0, 1) plus a preference per expert: the skew that a balancer meets."""
    return _normal(g, tokens, experts) + _normal(g, experts)


def _chosen(g, case):
    idx = _logits(g, case["tokens"], case["experts"]).topk(case["topk"], dim=-1).indices
    if case["padded"]:
        idx[torch.rand(case["tokens"], device="cuda", generator=g) < 0.2] = -1
    return idx


def _sorted_by_expert(idx, experts):
    """Rows of every expert, the row of every pair of token and choice, the pair of every row; -1 where there is none."""
    flat = idx.flatten()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    key, pair = torch.sort(key, stable=True)
    at = torch.arange(len(flat), device=flat.device)
    there = key < experts
    counts = torch.bincount(key, minlength=experts + 1)[:experts].int()
    place = torch.empty_like(flat)
    place[pair] = torch.where(there, at, -1)
    return counts, place.view(idx.shape).int(), torch.where(there, pair, -1).int()


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    if case["kind"] == "gate":
        dtype = getattr(torch, case["dtype"])
        x = _logits(g, case["tokens"], case["experts"])
        if case["padded"]:  # experts that are out of service, slots without a token
            x[:, torch.rand(case["experts"], device="cuda", generator=g) < 0.1] = -math.inf
            x[torch.rand(case["tokens"], device="cuda", generator=g) < 0.2] = -math.inf
        state["logits"] = x.to(dtype)
        state["dweights"] = _normal(g, case["tokens"], case["topk"])
        return state
    if case["kind"] in ("sort", "combine"):
        t, k, h = case["tokens"], case["topk"], case["hidden"]
        dtype = getattr(torch, case["dtype"])
        state["idx"] = _chosen(g, case)
        if case["kind"] == "sort":
            state["x"] = _normal(g, t, h).to(dtype)
            state["drows"] = _normal(g, t * k, h).to(dtype) if case["grad"] else None
            return state
        state["counts"], state["place"], state["source"] = _sorted_by_expert(state["idx"], case["experts"])
        state["rows"] = _normal(g, t * k, h).to(dtype)
        state["weights"] = torch.softmax(_normal(g, t, k), -1)
        state["dout"] = _normal(g, t, h).to(dtype) if case["grad"] else None
        return state
    m, n, k, e = case["rows"], case["n"], case["k"], max(1, case["experts"])
    dtype, out = getattr(torch, case["dtype"]), _out_type(case)
    state["a"] = _normal(g, m, k).to(dtype)
    state["b"] = torch.stack([(_normal(g, n, k) * k**-0.5).to(dtype) for _ in range(e)])
    state["bias"] = _normal(g, e, n).to(dtype) if case["bias"] else None
    state["residual"] = _normal(g, m, _out_cols(case)).to(out) if case["residual"] else None
    state["dout"] = _normal(g, m, _out_cols(case)).to(out) if case["grad"] else None
    state["group"] = None
    if case["experts"]:
        # rows of every expert: a gate's skewed choice, the last expert idle; in a padded batch some rows are nobody's
        popular = torch.softmax(_normal(g, e), 0)
        popular[-1] = 0
        taken = m - m // 8 if case["spare"] else m
        chosen = torch.multinomial(popular, taken, replacement=True, generator=g)
        state["group"] = torch.bincount(chosen, minlength=e).int()
    else:
        state["b"] = state["b"][0]
        state["bias"] = state["bias"][0] if case["bias"] else None
    return state


# ---------------------------------------------------------------------------------- one pass


def run(state):
    return {"gate": _gate, "sort": _sort, "combine": _combine, "matmul": _matmul}[state["kind"]](state)


def _named(**outputs):
    return {name: v for name, v in outputs.items() if v is not None}


def _leaf(t, grad):
    """The tensor as a user's parameter or activation: a leaf of this pass's graph."""
    return None if t is None else t.detach().requires_grad_() if grad else t


def _gate(s):
    if own:
        from lplb_b200 import ops

        x = _leaf(s["logits"], s["grad"])
        weights, idx = ops.gate_topk(x, s["topk"], score=s["score"], renormalize=s["renormalize"])
        dlogits = torch.autograd.grad(weights, x, s["dweights"])[0] if s["grad"] else None
        return _named(weights=weights.detach(), idx=idx, dlogits=dlogits)
    x = s["logits"].float()
    top, idx = torch.sort(x, dim=-1, descending=True, stable=True)
    top, idx = top[:, : s["topk"]], idx[:, : s["topk"]]
    there = top > -math.inf
    idx = torch.where(there, idx, -1)
    most = torch.where(there[:, :1], x.amax(-1, keepdim=True), 0.0)
    if s["score"] == "softmax":
        p = torch.exp(x - most)
        if not s["renormalize"]:
            p = p / p.sum(-1, keepdim=True)
    else:
        # sigmoids, or sigmoids over that of the largest logit's negative part, which a renormalisation takes out again
        p = torch.exp(x.clamp_max(0) - (most.clamp_max(0) if s["renormalize"] else 0)) / (1 + torch.exp(-x.abs()))
    w = torch.where(there, p.gather(1, idx.clamp_min(0)), 0.0)
    if s["renormalize"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(there, w / total, 0.0)
    if not s["grad"]:
        return {"weights": w, "idx": idx}
    d = torch.where(there, s["dweights"], 0.0)
    along = (d * w).sum(-1, keepdim=True)
    if s["score"] == "softmax":
        each = w * (d - along) if s["renormalize"] else w * d
        dx = torch.zeros_like(x) if s["renormalize"] else -torch.where(there[:, :1], p, 0.0) * along
    else:
        slope = 1 - 1 / (1 + torch.exp(-top))  # of log(sigmoid)
        each = torch.where(there, w * ((d - along) if s["renormalize"] else d) * slope, 0.0)
        dx = torch.zeros_like(x)
    dx.scatter_add_(1, idx.clamp_min(0), torch.where(there, each, 0.0))
    return {"weights": w, "idx": idx, "dlogits": dx.to(s["logits"].dtype)}


def _sort(s):
    if own:
        from lplb_b200 import ops

        x = _leaf(s["x"], s["grad"])
        order = ops.expert_order(s["idx"], s["experts"])
        rows = ops.take_rows(x, order)
        dx = torch.autograd.grad(rows, x, s["drows"])[0] if s["grad"] else None
        return _named(counts=order.counts, place=order.place, source=order.source, rows=rows.detach(), dx=dx)
    counts, place, source = _sorted_by_expert(s["idx"], s["experts"])
    rows = s["x"][source.clamp_min(0).long() // s["topk"]]
    rows[source < 0] = 0
    dx = None
    if s["grad"]:
        total = torch.zeros(s["x"].shape, device=rows.device)
        for k in range(s["topk"]):
            at = place[:, k].long()
            total += torch.where((at >= 0).unsqueeze(1), s["drows"][at.clamp_min(0)].float(), 0.0)
        dx = total.to(s["x"].dtype)
    return _named(counts=counts, place=place, source=source, rows=rows, dx=dx)


def _combine(s):
    if own:
        from lplb_b200 import ops

        rows, weights = _leaf(s["rows"], s["grad"]), _leaf(s["weights"], s["grad"])
        out = ops.combine_rows(rows, ops.ExpertOrder(s["counts"], s["place"], s["source"]), weights)
        drows, dweights = torch.autograd.grad(out, (rows, weights), s["dout"]) if s["grad"] else (None, None)
        return _named(out=out.detach(), drows=drows, dweights=dweights)
    place, w = s["place"].long(), s["weights"]
    out = torch.zeros(s["tokens"], s["hidden"], device=w.device)
    drows = torch.zeros_like(s["rows"]) if s["grad"] else None
    dweights = torch.zeros_like(w) if s["grad"] else None
    for k in range(s["topk"]):
        there = (place[:, k] >= 0).unsqueeze(1)
        at = place[:, k].clamp_min(0)
        y = torch.where(there, s["rows"][at].float(), 0.0)
        out += y * w[:, k : k + 1]
        if s["grad"]:
            dout = s["dout"].float()
            dweights[:, k] = (dout * y).sum(-1)
            token = there.squeeze(1).nonzero().squeeze(1)
            drows[at[token]] = (dout[token] * w[token, k : k + 1]).to(drows.dtype)
    return _named(out=out.to(s["rows"].dtype), drows=drows, dweights=dweights)


def _activate(z, activation):
    """The activation's values, and a function that takes a gradient of them to one of `z`."""
    if activation is None:
        return z, lambda d: d
    if activation == "relu":
        return z.clamp_min(0), lambda d: torch.where(z > 0, d, 0.0)
    if activation == "gelu":
        share = 0.5 * (1 + torch.erf(z * 2**-0.5))
        return z * share, lambda d: d * (share + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5)
    if activation == "silu":
        share = 1 / (1 + torch.exp(-z))
        return z * share, lambda d: d * share * (1 + z * (1 - share))
    both = z.unflatten(-1, (-1, 2, BLOCK))
    gate, up = both[..., 0, :], both[..., 1, :]
    share = 1 / (1 + torch.exp(-gate))

    def back(d):
        d = d.unflatten(-1, (-1, BLOCK))
        return torch.stack((d * up * share * (1 + gate * (1 - share)), d * gate * share), -2).flatten(-3)

    return (gate * share * up).flatten(-2), back


def _matmul(s):
    out_type = _out_type(s)
    if own:
        from lplb_b200 import ops

        a, b, bias, residual = (_leaf(s[name], s["grad"]) for name in ("a", "b", "bias", "residual"))
        out = ops.matmul(a, b, bias=bias, activation=s["activation"], residual=residual, rows=s["group"], out_dtype=out_type)
        if not s["grad"]:
            return {"out": out}
        leaves = _named(da=a, db=b, dbias=bias, dresidual=residual)
        return {"out": out.detach(), **dict(zip(leaves, torch.autograd.grad(out, tuple(leaves.values()), s["dout"])))}
    if s["group"] is None:
        parts = [(slice(0, s["rows"]), ...)]
    else:
        ends = s["group"].cumsum(0).tolist()
        parts = [(slice(end - n, end), e) for e, (n, end) in enumerate(zip(s["group"].tolist(), ends))]
    out = torch.zeros(s["rows"], _out_cols(s), device=s["a"].device)
    da, db = torch.zeros_like(s["a"]), torch.zeros_like(s["b"])
    dbias = torch.zeros_like(s["bias"]) if s["bias"] is not None else None
    for rows, e in parts:
        a, b = s["a"][rows].float(), s["b"][e].float()
        z = a @ b.T
        if s["bias"] is not None:
            z = z + s["bias"][e].float()
        out[rows], back = _activate(z, s["activation"])
        if s["grad"]:
            dz = back(s["dout"][rows].float())
            da[rows] = (dz @ b).to(da.dtype)
            db[e] = (dz.T @ a).to(db.dtype)
            if dbias is not None:
                dbias[e] = dz.sum(0).to(dbias.dtype)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    if not s["grad"]:
        return {"out": out.to(out_type)}
    dresidual = s["dout"].clone() if s["residual"] is not None else None
    return _named(out=out.to(out_type), da=da, db=db, dbias=dbias, dresidual=dresidual)


# ---------------------------------------------------------------------------------- what a pass cannot do without


def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    if case["kind"] == "gate":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        n = t * e * _size(case["dtype"])
        # the gradient reads the logits or what was kept of them, and the weights' gradient
        return {"bytes": n * (3 if case["grad"] else 1) + t * k * (16 if case["grad"] else 12),
                "flops": t * e * (10 if case["grad"] else 5)}
    if case["kind"] != "matmul":
        t, k, h, size = case["tokens"], case["topk"], case["hidden"], _size(case["dtype"])
        way = (t + t * k) * h * size  # tokens on one side, rows on the other
        if case["kind"] == "sort":
            return {"bytes": way * (2 if case["grad"] else 1) + t * k * 16, "flops": t * k * h * (1 if case["grad"] else 0)}
        back = (t + 2 * t * k) * h * size
        return {"bytes": way + (back if case["grad"] else 0) + t * k * 12, "flops": t * k * h * (5 if case["grad"] else 2)}
    m, n, k, e = case["rows"], case["n"], case["k"], max(1, case["experts"])
    cols, size, out = _out_cols(case), _size(case["dtype"]), _out_type(case).itemsize
    used = max(1, min(m, e - 1)) if case["experts"] else 1
    moved = (m * k + used * n * k) * size + m * cols * out * (2 if case["residual"] else 1)
    moved += e * n * size if case["bias"] else 0
    if case["grad"]:
        # dout and the operands again, da, db and the bias's gradient
        moved += m * cols * out + 2 * (m * k + e * n * k) * size + (e * n * size if case["bias"] else 0)
    return {"bytes": moved, "flops": 2 * m * n * k * (3 if case["grad"] else 1)}


# ---------------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"gate": _exact_gate, "sort": _exact_sort, "combine": _exact_combine, "matmul": _exact_matmul}[case["kind"]](s)


def _exact_gate(s):
    x = s["logits"].double()
    tokens, experts = x.shape
    number = torch.arange(experts, device=x.device)
    weights = x.new_zeros(tokens, s["topk"])
    idx = torch.full((tokens, s["topk"]), -1, device=x.device)
    dlogits = torch.zeros_like(x)
    for t0 in range(0, tokens, 512):
        part = x[t0 : t0 + 512]
        # an expert's rank: how many come before it, larger ones and equal ones of a lower number
        mine, other = part.unsqueeze(2), part.unsqueeze(1)
        rank = ((other > mine) | ((other == mine) & (number < number.unsqueeze(1)))).sum(2)
        chosen = (rank < s["topk"]) & (part > -math.inf)
        alive = (part > -math.inf).any(1)
        if s["score"] == "softmax":
            score = torch.zeros_like(part)
            score[alive] = torch.softmax(part[alive], 1)
        else:
            score = torch.sigmoid(part)
        w = score * chosen
        if s["renormalize"]:
            w[alive] = w[alive] / w[alive].sum(1, keepdim=True)
        d = torch.zeros_like(part)
        row, col = chosen.nonzero(as_tuple=True)
        weights[t0 + row, rank[row, col]] = w[row, col]
        idx[t0 + row, rank[row, col]] = col
        d[row, col] = s["dweights"].double()[t0 + row, rank[row, col]]
        # gradient of the scores, then through the score's own derivative
        if s["renormalize"]:
            total = (score * chosen).sum(1, keepdim=True)
            total[~alive] = 1
            d = chosen * (d - (d * w).sum(1, keepdim=True)) / total
        if s["score"] == "softmax":
            dlogits[t0 : t0 + 512] = score * (d - (d * score).sum(1, keepdim=True))
        else:
            dlogits[t0 : t0 + 512] = d * score * (1 - score)
    return {"weights": weights, "idx": idx, **({"dlogits": dlogits} if s["grad"] else {})}


def _order_by_counting(idx, experts):
    flat = idx.flatten()
    counts = torch.stack([(flat == e).sum() for e in range(experts)])
    place, source, at = torch.full_like(flat, -1), torch.full_like(flat, -1), 0
    for e, n in enumerate(counts.tolist()):
        pairs = (flat == e).nonzero().squeeze(1)
        place[pairs] = torch.arange(at, at + n, device=flat.device)
        source[at : at + n] = pairs
        at += n
    return counts.int(), place.view(idx.shape).int(), source.int()


def _exact_sort(s):
    counts, place, source = _order_by_counting(s["idx"], s["experts"])
    taken = (source >= 0).nonzero().squeeze(1)
    token = source[taken] // s["topk"]
    rows = torch.zeros(source.numel(), s["hidden"], dtype=s["x"].dtype, device=source.device)
    rows[taken] = s["x"][token]  # copies
    out = {"counts": counts, "place": place, "source": source, "rows": rows}
    if s["grad"]:
        out["dx"] = torch.zeros(s["x"].shape, dtype=torch.float64, device=source.device)
        for at in range(0, len(taken), 8192):  # a part at a time: rows in 64 bits are large
            out["dx"].index_add_(0, token[at : at + 8192], s["drows"][taken[at : at + 8192]].double())
    return out


def _exact_combine(s):
    _, place, source = _order_by_counting(s["idx"], s["experts"])
    taken = (source >= 0).nonzero().squeeze(1)
    pair = source[taken]
    token, w = pair // s["topk"], s["weights"].double().flatten()[pair].unsqueeze(1)
    out = torch.zeros(s["tokens"], s["hidden"], dtype=torch.float64, device=w.device)
    out.index_add_(0, token, s["rows"][taken].double() * w)
    if not s["grad"]:
        return {"out": out}
    drows = torch.zeros(s["rows"].shape, dtype=torch.float64, device=w.device)
    dweights = torch.zeros(place.numel(), dtype=torch.float64, device=w.device)
    for at in range(0, len(taken), 8192):  # a part at a time: rows in 64 bits are large
        part = slice(at, at + 8192)
        d = s["dout"][token[part]].double()
        drows[taken[part]] = d * w[part]
        dweights[pair[part]] = torch.linalg.vecdot(d, s["rows"][taken[part]].double())
    return {"out": out, "drows": drows, "dweights": dweights.view(place.shape)}


def _exact_matmul(s):
    def activated(z):
        if s["activation"] == "relu":
            return torch.nn.functional.relu(z)
        if s["activation"] == "gelu":
            return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
        if s["activation"] == "silu":
            return z * torch.sigmoid(z)
        if s["activation"] == "swiglu":
            z = z.view(z.shape[0], -1, 2, BLOCK)
            return (z[:, :, 0] * torch.sigmoid(z[:, :, 0]) * z[:, :, 1]).reshape(z.shape[0], -1)
        return z.clone()

    grouped = s["group"] is not None
    m, cols, device = s["rows"], _out_cols(s), s["a"].device
    out = torch.zeros(m, cols, dtype=torch.float64, device=device)
    grads = _named(da=s["a"], db=s["b"], dbias=s["bias"]) if s["grad"] else {}
    grads = {name: torch.zeros(v.shape, dtype=torch.float64, device=device) for name, v in grads.items()}
    at = 0
    for e, n in enumerate(s["group"].tolist() if grouped else [m]):
        b = s["b"][e] if grouped else s["b"]
        bias = None if s["bias"] is None else (s["bias"][e] if grouped else s["bias"]).double()
        step = 4096  # rows at a time
        for r in range(at, at + n, step):
            part = slice(r, min(r + step, at + n))
            a = s["a"][part].double()
            z = a @ b.double().T
            z = z if bias is None else z + bias
            with torch.enable_grad():
                z.requires_grad_(s["grad"])
                y = activated(z)
            out[part] = y.detach()
            if s["grad"]:
                (dz,) = torch.autograd.grad(y, z, s["dout"][part].double())
                grads["da"][part] = dz @ b.double()
                (grads["db"][e] if grouped else grads["db"]).add_(dz.T @ a)
                if bias is not None:
                    (grads["dbias"][e] if grouped else grads["dbias"]).add_(dz.sum(0))
        at += n
    if s["residual"] is not None:
        out += s["residual"].double()
        if s["grad"]:
            grads["dresidual"] = s["dout"].double()
    return {"out": out, **grads}
