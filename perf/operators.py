"""Performance cases of the 8-bit serving operators and of the MoE layer for a few tokens.

Three kinds of work, all through the public entry points of ``lplb_b200.ops``:

* ``norm``    ``rms_norm_fp8``: the residual's addition, the root-mean-square norm and an e4m3 output with a
              power-of-two scale for every block of 128
* ``matmul``  ``matmul_fp8``: the product of such rows with weights that have a scale for every block of 128 x 128,
              for one matrix or for the rows of many experts
* ``few``     ``moe_few_tokens``: a whole SwiGLU mixture-of-experts layer for up to 64 tokens

With ``own`` false the same operators run in elementary torch operations in 32 bits.
"""

import torch

own = False

BLOCK = 128


def listed():
    return [
        # the norm in front of the layer in a decode step of a few sequences
        dict(name="norm_decode", kind="norm", tokens=4, hidden=7168, dtype="bfloat16", residual=True),
        # a ragged batch of a model in half precision whose rows end inside a block, first norm (no residual yet)
        dict(name="norm_ragged", kind="norm", tokens=1000, hidden=2064, dtype="float16", residual=False),
        # the same norm over a whole prefill batch of the layer benchmark
        dict(name="norm_prefill", kind="norm", tokens=8192, hidden=7168, dtype="bfloat16", residual=True),
        # down projection of one token
        dict(name="matmul_token", kind="matmul", experts=0, rows=1, n=7168, k=2048, out="bfloat16"),
        # gate and up projection of a decode batch
        dict(name="matmul_decode", kind="matmul", experts=0, rows=64, n=4096, k=7168, out="bfloat16"),
        # odd sizes and a result in 32 bits
        dict(name="matmul_ragged", kind="matmul", experts=0, rows=1001, n=4100, k=2064, out="float32"),
        # a dense projection of a prefill batch (tensor bound)
        dict(name="matmul_prefill", kind="matmul", experts=0, rows=8192, n=4096, k=7168, out="bfloat16"),
        # the first product of 32 experts in prefill, some of them nearly idle
        dict(name="matmul_experts", kind="matmul", experts=32, rows=16384, n=4096, k=7168, out="bfloat16"),
        # one sequence decoding: 8 of 48 physical experts, weights in 8 bits
        dict(name="few_token", kind="few", tokens=1, topk=8, experts=48, hidden=7168, inter=2048, fp8=True, x8=True,
             padded=False),
        # a small model's decode step with padded slots, hidden states not quantised yet
        dict(name="few_small", kind="few", tokens=12, topk=4, experts=32, hidden=1024, inter=512, fp8=True, x8=False,
             padded=True),
        # a few sequences on the layer's bf16 weights
        dict(name="few_bf16", kind="few", tokens=16, topk=8, experts=48, hidden=7168, inter=2048, fp8=False, x8=False,
             padded=False),
        # the largest batch: every expert is active
        dict(name="few_decode", kind="few", tokens=64, topk=8, experts=48, hidden=7168, inter=2048, fp8=True, x8=True,
             padded=False),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["norm", "matmul", "matmul", "few", "few"])
    if kind == "norm":
        return dict(kind="norm", tokens=_spread(rng, 1, 8192), hidden=16 * rng.randint(16, 448),
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), residual=rng.random() < 0.7)
    if kind == "matmul":
        experts = rng.choice([0, 0, 0, rng.randint(2, 32)])
        return dict(kind="matmul", experts=experts, rows=_spread(rng, max(1, experts), 8192), n=_spread(rng, 100, 4096),
                    k=16 * _spread(rng, 16, 448), out=rng.choice(["bfloat16", "bfloat16", "float32"]))
    fp8 = rng.random() < 0.6
    return dict(kind="few", tokens=_spread(rng, 1, 64), topk=rng.choice([1, 2, 4, 6, 8]), experts=rng.randint(8, 48),
                hidden=256 * rng.randint(2, 28), inter=128 * rng.randint(1, 16), fp8=fp8, x8=fp8 and rng.random() < 0.6,
                padded=rng.random() < 0.3)


# ---------------------------------------------------------------------------------- values in 8 bits


def _scale_of(amax):
    """Biased exponent of the smallest power of two s with amax / s <= 448 = 1.75 * 2^8."""
    bits = amax.float().contiguous().view(torch.int32)
    return (((bits + 0x1FFFFF) >> 23) - 8).clamp_min(1)


def _power(exponent):
    return (exponent.int() << 23).view(torch.float32)


def _blocks(x):
    """[..., K] -> [..., blocks, 128], the last block filled up with zeros."""
    k = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))


def _quantise(x):
    """Rows in 8 bits: values and scales of [..., K]."""
    b = _blocks(x.float())
    e = _scale_of(torch.where(b.isfinite(), b.abs(), 0.0).amax(-1))
    q = (b * _power(254 - e).unsqueeze(-1)).flatten(-2)[..., : x.shape[-1]].to(torch.float8_e4m3fn)
    return q.contiguous(), e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _quantise_weight(w):
    """[N, K] weights, one scale for every block of 128 x 128."""
    n, k = w.shape
    b = torch.nn.functional.pad(w.float(), (0, -k % BLOCK, 0, -n % BLOCK))
    b = b.unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK))
    e = _scale_of(b.abs().amax((1, 3)))
    q = (b * _power(254 - e)[:, None, :, None]).flatten(2).flatten(0, 1)[:n, :k].to(torch.float8_e4m3fn)
    return q.contiguous(), e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _rows_in_32(q, scale):
    s = _power(scale.view(torch.uint8))
    return q.float() * s.repeat_interleave(BLOCK, -1)[..., : q.shape[-1]]


def _weight_in_32(q, scale):
    s = _power(scale.view(torch.uint8))
    s = s.repeat_interleave(BLOCK, -1)[..., : q.shape[-1]]
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., : q.shape[-2], :]


# ---------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _hidden_states(g, tokens, hidden):
    """N(0, 1) with a few channels that are larger, as residual streams have them."""
    channel = torch.exp(torch.randn(hidden, device="cuda", generator=g))
    return torch.randn(tokens, hidden, device="cuda", generator=g) * channel


def prepare(case, seed):
    g = _generator(seed)
    state = dict(case)
    if case["kind"] == "norm":
        dtype = getattr(torch, case["dtype"])
        state["x"] = _hidden_states(g, case["tokens"], case["hidden"]).to(dtype)
        state["r"] = _hidden_states(g, case["tokens"], case["hidden"]).to(dtype) if case["residual"] else None
        state["w"] = (1 + 0.2 * torch.randn(case["hidden"], device="cuda", generator=g)).to(dtype)
    elif case["kind"] == "matmul":
        state["a"], state["a_scale"] = _quantise(_hidden_states(g, case["rows"], case["k"]))
        made = [
            _quantise_weight(torch.randn(case["n"], case["k"], device="cuda", generator=g) * case["k"] ** -0.5)
            for _ in range(max(1, case["experts"]))
        ]
        state["b"] = torch.stack([q for q, _ in made])
        state["b_scale"] = torch.stack([s.view(torch.uint8) for _, s in made]).view(torch.float8_e8m0fnu)
        state["group"] = None
        if case["experts"]:
            # rows of every expert: a gate's skewed choice, the last expert idle where there are several rows each
            popular = torch.softmax(torch.randn(case["experts"], device="cuda", generator=g), 0)
            popular[-1] = 0
            chosen = torch.multinomial(popular, case["rows"], replacement=True, generator=g)
            state["group"] = torch.bincount(chosen, minlength=case["experts"]).int()
            state["most"] = int(state["group"].max())
        else:
            state["b"], state["b_scale"] = state["b"][0], state["b_scale"][0]
    else:
        t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
        x = torch.randn(t, h, device="cuda", generator=g).bfloat16()
        state["x"], state["x_scale"] = _quantise(x) if case["x8"] else (x, None)
        w13, w2 = [], []
        for _ in range(e):
            # 128 gate rows, the 128 matching up rows, and so on
            up = (torch.randn(2 * i, h, device="cuda", generator=g) * h**-0.5).bfloat16()
            down = (torch.randn(h, i, device="cuda", generator=g) * i**-0.5).bfloat16()
            w13.append(_quantise_weight(up) if case["fp8"] else (up, None))
            w2.append(_quantise_weight(down) if case["fp8"] else (down, None))
        state["w13"], state["w2"] = torch.stack([q for q, _ in w13]), torch.stack([q for q, _ in w2])
        for name, made in (("w13_scale", w13), ("w2_scale", w2)):
            state[name] = (
                torch.stack([s.view(torch.uint8) for _, s in made]).view(torch.float8_e8m0fnu) if case["fp8"] else None
            )
        logits = torch.randn(t, e, device="cuda", generator=g) + torch.randn(e, device="cuda", generator=g)
        state["gate"], state["idx"] = torch.softmax(logits, -1).topk(case["topk"], dim=-1)
        if case["padded"]:
            state["idx"][torch.rand(t, device="cuda", generator=g) < 0.2] = -1
    return state


# ---------------------------------------------------------------------------------- one pass


def run(state):
    return {"norm": _norm, "matmul": _matmul, "few": _few}[state["kind"]](state)


def _norm(s):
    if own:
        from lplb_b200 import ops

        q, scale, h = ops.rms_norm_fp8(s["x"], s["w"], s["r"], eps=1e-6)
        return {"q": q, "scale": scale, "h": h} if s["residual"] else {"q": q, "scale": scale}
    h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
    f = h.float()
    n = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + 1e-6) * s["w"].float()
    q, scale = _quantise(n)
    return {"q": q, "scale": scale, "h": h} if s["residual"] else {"q": q, "scale": scale}


def _matmul(s):
    out = getattr(torch, s["out"])
    if own:
        from lplb_b200 import ops

        return ops.matmul_fp8(s["a"], s["a_scale"], s["b"], s["b_scale"], rows=s["group"], out_dtype=out)
    a, b = _rows_in_32(s["a"], s["a_scale"]), _weight_in_32(s["b"], s["b_scale"])
    if s["group"] is None:
        return (a @ b.T).to(out)
    ends = s["group"].long().cumsum(0)
    each = torch.arange(s["rows"], device=a.device)
    expert = (each.unsqueeze(1) >= ends.unsqueeze(0)).sum(1)
    place = each - (ends - s["group"])[expert]
    padded = a.new_zeros(s["experts"], s["most"], s["k"])
    padded[expert, place] = a
    return torch.bmm(padded, b.transpose(1, 2))[expert, place].to(out)


def _few(s):
    if own:
        from lplb_b200 import ops

        return ops.moe_few_tokens(s["x"], s["idx"], s["gate"], s["w13"], s["w2"], x_scale=s["x_scale"],
                                  w13_scale=s["w13_scale"], w2_scale=s["w2_scale"])
    active = torch.unique(s["idx"])
    active = active[active >= 0]
    if s["fp8"]:
        x = _rows_in_32(s["x"], s["x_scale"]) if s["x8"] else _rows_in_32(*_quantise(s["x"]))
        w13 = _weight_in_32(s["w13"].view(torch.uint8)[active].view(torch.float8_e4m3fn),
                            s["w13_scale"].view(torch.uint8)[active])
        w2 = _weight_in_32(s["w2"].view(torch.uint8)[active].view(torch.float8_e4m3fn),
                           s["w2_scale"].view(torch.uint8)[active])
    else:
        x, w13, w2 = s["x"].float(), s["w13"][active].float(), s["w2"][active].float()
    both = torch.matmul(x, w13.transpose(1, 2)).unflatten(-1, (-1, 2, BLOCK))
    gate, up = both[..., 0, :].flatten(-2), both[..., 1, :].flatten(-2)
    act = gate / (1 + torch.exp(-gate)) * up
    act = _rows_in_32(*_quantise(act)) if s["fp8"] else act.bfloat16().float()
    y = torch.bmm(act, w2.transpose(1, 2))
    hit = s["idx"].unsqueeze(0) == active.view(-1, 1, 1)
    share = torch.where(hit, s["gate"], 0.0).sum(-1)
    return torch.where(hit.any(-1).unsqueeze(-1), y * share.unsqueeze(-1), 0.0).sum(0).bfloat16()


# ---------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["kind"] == "norm":
        n, size = case["tokens"] * case["hidden"], 4 if case["dtype"] == "float32" else 2
        moved = n * (size * (3 if case["residual"] else 1) + 1 + 1 / BLOCK) + case["hidden"] * size
        return {"bytes": moved, "flops": 6 * n}
    if case["kind"] == "matmul":
        m, n, k = case["rows"], case["n"], case["k"]
        used = max(1, min(m, case["experts"] - 1)) if case["experts"] else 1
        return {"bytes": m * k + used * n * k + m * n * (2 if case["out"] == "bfloat16" else 4), "flops": 2 * m * n * k}
    t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
    # experts that a gate without a preference reaches
    reached = e * (1 - (1 - case["topk"] / e) ** t)
    return {"bytes": reached * 3 * h * i * (1 if case["fp8"] else 2) + t * h * (3 if case["x8"] else 4),
            "flops": 2 * t * case["topk"] * 3 * h * i}


# ---------------------------------------------------------------------------------- the definition in 64 bits


def _in_64(q, scale, rows_per_scale):
    """The values that 8-bit numbers and their scales stand for."""
    v = q.to(torch.float64)
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=v.device), scale.view(torch.uint8).double() - 127)
    row = torch.arange(v.shape[-2], device=v.device) // rows_per_scale
    col = torch.arange(v.shape[-1], device=v.device) // BLOCK
    return v * s[..., row, :][..., col]


def _to_8_bits(v):
    """Values rounded to e4m3 with the scale of their block, and the scales; `v` is [rows, K] in 64 bits."""
    rows, k = v.shape
    blocks = -(-k // BLOCK)
    full = v.new_zeros(rows, blocks * BLOCK)
    full[:, :k] = v
    full = full.view(rows, blocks, BLOCK)
    top = full.abs().max(-1).values / 448
    mantissa, exponent = torch.frexp(top)
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent).double().clamp_min(-126)
    exponent = torch.where(top == 0, torch.full_like(exponent, -126), exponent)
    scale = torch.exp2(exponent)
    u = full / scale.unsqueeze(-1)
    digit = (torch.frexp(u)[1] - 1).clamp_min(-6)  # floor(log2 |u|), subnormals below 2^-6
    step = torch.exp2(digit.double() - 3)
    q = torch.round(u / step) * step
    return q.view(rows, -1)[:, :k], scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = (h + s["r"].double()).to(s["x"].dtype).double()  # the sum is a result of the type, and its norm is taken
        n = h / torch.sqrt(h.square().sum(-1, keepdim=True) / case["hidden"] + 1e-6) * s["w"].double()
        q, scale = _to_8_bits(n)
        return {"q": q, "scale": scale, "h": h} if case["residual"] else {"q": q, "scale": scale}
    if case["kind"] == "matmul":
        a = _in_64(s["a"], s["a_scale"], 1)
        if not case["experts"]:
            return a @ _in_64(s["b"], s["b_scale"], BLOCK).T
        parts, at = [], 0
        for e, n in enumerate(s["group"].tolist()):
            parts.append(a[at : at + n] @ _in_64(s["b"][e], s["b_scale"][e], BLOCK).T)
            at += n
        return torch.cat(parts)
    if case["fp8"]:
        x = _in_64(s["x"], s["x_scale"], 1) if case["x8"] else None
        if x is None:
            q, scale = _to_8_bits(s["x"].double())
            x = q * scale.repeat_interleave(BLOCK, 1)[:, : case["hidden"]]
    else:
        x = s["x"].double()
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        token, place = (s["idx"] == e).nonzero(as_tuple=True)
        if not len(token):
            continue
        if case["fp8"]:
            w13, w2 = _in_64(s["w13"][e], s["w13_scale"][e], BLOCK), _in_64(s["w2"][e], s["w2_scale"][e], BLOCK)
        else:
            w13, w2 = s["w13"][e].double(), s["w2"][e].double()
        w13 = w13.view(case["inter"] // BLOCK, 2, BLOCK, case["hidden"])
        gate = x[token] @ w13[:, 0].reshape(case["inter"], -1).T
        up = x[token] @ w13[:, 1].reshape(case["inter"], -1).T
        act = gate * torch.sigmoid(gate) * up
        if case["fp8"]:
            q, scale = _to_8_bits(act)
            act = q * scale.repeat_interleave(BLOCK, 1)[:, : case["inter"]]
        else:
            act = act.to(torch.bfloat16).double()  # the activations are held in the weights' type
        out.index_add_(0, token, act @ w2.T * s["gate"][token, place].double().unsqueeze(1))
    return out
