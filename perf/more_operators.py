"""The operators of 8-bit experts as workloads: INT8 products and their gradients, routing, and the exchange of tokens.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes a case's inputs
on the GPU, ``run(state)`` is one pass and ``work(case)`` what a pass cannot do without. With ``own`` true ``run`` calls
``piper_offload_b200.int8`` and ``piper_offload_b200.routing``; with ``own`` false it computes the same operators from
elementary torch operations. ``exact(case, seed)`` is the definition in 64 bits.

Operators
  linear         tokens, quantised to 8 bits each by its own scale, times an INT8 weight with a scale (and, where
                 ``weight`` is "zero", a zero point) for each row, or one scale for all of it ("tensor"), or in
                 LLM.int8's storage ("bnb8": codes times a row's largest magnitude over 127)
  grouped        the same with a weight per expert and the tokens sorted by expert
  grad           the gradient of ``linear`` with respect to the tokens (the weight is frozen)
  grouped_grad   the gradient of ``grouped`` with respect to the tokens
  route          each token's experts from a router's logits: softmax or sigmoid scores, a bias for balance, the best
                 groups of experts, the best experts in them, renormalised weights, and the order by expert; with
                 ``grad`` the weights' gradient down to the logits too
  exchange       every token's row copied to its experts' places, and the experts' rows added up by the router's
                 weights; with ``grad`` all gradients of both
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
EXACT_FLOPS = 1.2e14  # a 64-bit product above this takes too long


# ----------------------------------------------------------------------------------------------- cases
def _product_case(name, op, tokens, rows, cols, *, weight="rows", experts=0, skew=0.0, empty_every=0, tail=0, dtype="bfloat16"):
    case = {"op": op, "tokens": tokens, "rows": rows, "cols": cols, "weight": weight, "experts": experts, "skew": skew,
            "empty_every": empty_every, "tail": tail, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def _route_case(name, op, tokens, experts, top_k, *, hidden=0, scoring="softmax", bias=False, groups=1, top_groups=1,
                group_score="max", renormalize=True, scale=1.0, masked=0.0, grad=False, dtype="bfloat16"):
    case = {"op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden, "scoring": scoring, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_score": group_score, "renormalize": renormalize, "scale": scale,
            "masked": masked, "grad": grad, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one token of decoding through a Llama-3-8B-shaped gate projection
        _product_case("linear 1 token", "linear", 1, 14336, 4096),
        # a short ragged prompt in fp16 through an asymmetric weight whose rows start on odd addresses
        _product_case("linear 333 odd zero points", "linear", 333, 1000, 2081, weight="zero", dtype="float16"),
        # a long prompt through the gate projection
        _product_case("linear 4096 tokens", "linear", 4096, 14336, 4096),
        # a decoding step over a layer of experts, two of which get nothing
        _product_case("grouped 16 rows 8 experts", "grouped", 16, 14336, 4096, experts=8, skew=0.5, empty_every=4),
        # a prompt over many small experts, uneven, the last rows being padding of a fixed-capacity buffer
        _product_case("grouped 4096 rows 32 experts", "grouped", 4096, 2048, 2048, experts=32, skew=0.6, empty_every=8, tail=96),
        # training adapters over a frozen Llama-3-8B-shaped projection
        _product_case("grad 2048 tokens", "grad", 2048, 14336, 4096),
        # the same over experts
        _product_case("grouped grad 2048 rows 16 experts", "grouped_grad", 2048, 2048, 2048, experts=16, skew=0.6, empty_every=8),
        # a decoding batch over a few experts: a call's own cost
        _route_case("route 64 tokens 8 experts", "route", 64, 8, 2, dtype="float32"),
        # a padded batch of odd sizes, trained, weights not renormalised
        _route_case("route 777 tokens 60 experts", "route", 777, 60, 4, renormalize=False, masked=0.15, grad=True),
        # a training batch over many experts in groups, balanced by a bias
        _route_case("route 16384 tokens 256 experts", "route", 16384, 256, 8, scoring="sigmoid", bias=True, groups=8, top_groups=4,
                    group_score="top2", scale=2.5, grad=True, dtype="float32"),
        # a decoding batch's rows to their experts and back
        _route_case("exchange 24 tokens", "exchange", 24, 8, 2, hidden=4096),
        # a training batch's, with the gradients
        _route_case("exchange 8192 tokens top 8", "exchange", 8192, 64, 8, hidden=2048, grad=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: sizes spread over the listed ones' ranges, most of them no multiple of a tile."""
    op = rng.choice(["linear", "linear", "grouped", "grouped", "grad", "grouped_grad", "route", "route", "exchange", "exchange"])
    if op in ("route", "exchange"):
        top_k = rng.choice([1, 2, 3, 4, 6, 8])
        groups, top_groups, experts = 1, 1, _log_int(rng, 8, 256)
        scoring, bias = rng.choice(["softmax", "sigmoid"]), rng.random() < 0.4
        if rng.random() < 0.4:
            groups = rng.choice([2, 4, 8])
            top_groups = rng.randint(1, groups)
            experts = groups * max(_log_int(rng, 2, 32), -(-top_k // top_groups), 2)
        kw = {"scoring": scoring, "bias": bias, "groups": groups, "top_groups": top_groups, "group_score": rng.choice(["max", "top2"]),
              "renormalize": rng.random() < 0.7, "scale": rng.choice([1.0, 1.0, 2.5]), "masked": rng.choice([0.0, 0.0, 0.2]),
              "grad": rng.random() < 0.6, "dtype": rng.choice(["bfloat16", "float16", "float32"])}
        if op == "route":
            return _route_case(None, op, _log_int(rng, 1, 16384), experts, top_k, **kw)
        hidden = _log_int(rng, 64, 4096)
        tokens = min(_log_int(rng, 1, 8192), 8192 * 8 * 2048 * 2 // (top_k * hidden * DTYPES[kw["dtype"]].itemsize))
        return _route_case(None, op, tokens, experts, top_k, hidden=hidden, **kw)
    weight = rng.choice(["rows", "rows", "zero", "tensor", "bnb8"])
    dtype = "float16" if weight == "bnb8" else rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op in ("linear", "grad"):
        rows, cols = _log_int(rng, 128, 14336), _log_int(rng, 128, 8192)
        tokens = _log_int(rng, 1, 4096) if op == "linear" else _log_int(rng, 16, 2048)
        return _product_case(None, op, min(tokens, 4096 * 14336 * 4096 // (rows * cols)), rows, cols, weight=weight,
                             dtype="bfloat16" if op == "grad" and dtype == "float32" else dtype)
    return _product_case(None, op, _log_int(rng, 8, 4096), _log_int(rng, 256, 2816), _log_int(rng, 256, 2816),
                         weight="rows" if weight in ("tensor", "bnb8") else weight, experts=_log_int(rng, 4, 48),
                         skew=round(rng.uniform(0.0, 0.8), 2), empty_every=rng.choice([0, 0, 3, 5, 8]), tail=rng.choice([0, 0, 5]),
                         dtype=rng.choice(["bfloat16", "float16"]))


def _sizes(case):
    """Rows of each expert: a power law in an order of its own, some experts empty, ``tail`` rows left over."""
    experts, rows = case["experts"], max(0, case["tokens"] - case["tail"])
    every = case["empty_every"]
    weight = [0.0 if every and i % every == every - 1 else (1.0 + (i * 7) % experts) ** -case["skew"] for i in range(experts)]
    total, at, sizes, taken = sum(weight), 0.0, [], 0
    for w in weight:
        at += w
        end = int(round(rows * at / total))
        sizes.append(end - taken)
        taken = end
    return sizes


def work(case):
    tokens, wide = case["tokens"], DTYPES[case["dtype"]].itemsize
    if case["op"] == "route":
        chosen = tokens * case["top_k"]
        once = tokens * case["experts"] * wide
        # logits, weights and experts, places and sources; backward: the logits again, the weights' gradient, the logits'
        return {"bytes": once + chosen * 16 + (2 * once + chosen * 12 if case["grad"] else 0),
                "flops": 10.0 * tokens * case["experts"]}
    if case["op"] == "exchange":
        row = case["hidden"] * wide
        copies = tokens * case["top_k"]
        there, back = (tokens + copies) * row, (copies + tokens) * row
        # backward: the copies' gradients added up; the result's gradient, the rows and their gradients
        grads = (copies + tokens) * row + (tokens + 2 * copies) * row
        return {"bytes": there + back + (grads if case["grad"] else 0) + copies * 8,
                "flops": 2.0 * copies * case["hidden"] * (4 if case["grad"] else 1)}
    rows, cols = case["rows"], case["cols"]
    used, weights = tokens, 1
    if case["experts"]:
        sizes = _sizes(case)
        used, weights = sum(sizes), sum(n > 0 for n in sizes)
    into, out = (rows, cols) if "grad" in case["op"] else (cols, rows)
    return {"bytes": weights * rows * (cols + 2) + (used * into + tokens * out) * wide, "flops": 2.0 * used * rows * cols}


# ---------------------------------------------------------------------------------------------- inputs
def _prepare_product(case, state, generator):
    e, rows, cols, tokens = max(1, case["experts"]), case["rows"], case["cols"], case["tokens"]
    w = torch.randn((e, rows, cols), generator=generator, device="cuda") * 0.02
    kind, state["zero"] = case["weight"], None
    if kind == "zero":
        # rows off zero, as asymmetric weights are
        w += 0.01 * torch.randn((e, rows, 1), generator=generator, device="cuda")
        low, high = w.amin(-1, keepdim=True).clamp(max=0.0), w.amax(-1, keepdim=True).clamp(min=0.0)
        scale = (high - low) / 255
        state["zero"] = (-128 - torch.round(low / scale)).clamp(-128, 127).to(torch.int8)
        codes = (torch.round(w / scale) + state["zero"].float()).clamp(-128, 127)
    else:
        top = w.abs().amax((1, 2), keepdim=True) if kind == "tensor" else w.abs().amax(-1, keepdim=True)
        scale = (top / 127).to(torch.bfloat16).float() if kind != "bnb8" else top / 127
        codes = torch.round(w / scale).clamp(-127, 127)
        # LLM.int8 keeps a row's largest magnitude
        scale = top.reshape(rows) if kind == "bnb8" else scale.to(torch.bfloat16)
    state.update(codes=codes.to(torch.int8), scale=scale)
    if not case["experts"]:
        state["codes"] = state["codes"][0]
        state["scale"] = scale if kind == "bnb8" else scale[0]
        state["zero"] = None if state["zero"] is None else state["zero"][0]
    dtype = DTYPES[case["dtype"]]
    if "grad" in case["op"]:
        state["x"] = (torch.randn((tokens, rows), generator=generator, device="cuda") * 1e-3).to(dtype)
    else:
        # activations after a norm: unit scale, with a few channels far larger
        x = torch.randn((tokens, cols), generator=generator, device="cuda")
        x *= torch.where(torch.rand(cols, generator=generator, device="cuda") < 0.005, 20.0, 1.0)
        state["x"] = x.to(dtype)
    if case["experts"]:
        sizes = _sizes(case)
        state["ends"] = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
        state["capacity"] = max(1, max(sizes))


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    state = {"case": case}
    if case["op"] not in ("route", "exchange"):
        _prepare_product(case, state, generator)
        return state

    def normal(*shape, dtype=DTYPES[case["dtype"]]):
        return torch.randn(shape, generator=generator, device="cuda").to(dtype)

    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    # some experts are liked more than others
    logits = (1.5 * normal(tokens, experts, dtype=torch.float32) + 0.5 * normal(experts, dtype=torch.float32)).to(DTYPES[case["dtype"]])
    state["bias"] = 0.05 * normal(experts, dtype=torch.float32) if case["bias"] else None
    state["mask"] = torch.rand(tokens, generator=generator, device="cuda") >= case["masked"] if case["masked"] else None
    if case["op"] == "route":
        state["logits"] = logits.requires_grad_(case["grad"])
        state["gradient"] = normal(tokens, top_k, dtype=torch.float32)
        return state
    state["logits"] = logits
    state.update(_plain_route(state))
    del state["logits"]
    hidden = case["hidden"]
    state["x"], state["y"] = normal(tokens, hidden), normal(tokens * top_k, hidden)
    state["x_gradient"], state["y_gradient"] = normal(tokens * top_k, hidden), normal(tokens, hidden)
    for name in ("x", "y", "weights") if case["grad"] else ():
        state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------------------- the framework
def _own_weight(state):
    from piper_offload_b200 import weights as W

    case = state["case"]
    if case["weight"] == "bnb8":
        return W.Bnb8Weight(state["codes"], state["scale"])
    if case["experts"]:
        return W.Int8Experts(state["codes"], state["scale"], (1, case["cols"]), zero_point=state["zero"])
    block = (case["rows"], case["cols"]) if case["weight"] == "tensor" else (1, case["cols"])
    return W.Int8Weight(state["codes"], state["scale"], block, zero_point=state["zero"])


def _own(state):
    from piper_offload_b200 import int8, routing

    case = state["case"]
    if case["op"] == "route":
        r = routing.route_tokens(state["logits"], case["top_k"], scoring=case["scoring"], bias=state["bias"], groups=case["groups"],
                                 top_groups=case["top_groups"], group_score=case["group_score"], renormalize=case["renormalize"],
                                 scale=case["scale"], mask=state["mask"])
        out = {"weights": r.weights, "experts": r.experts, "ends": r.ends, "rows": r.rows, "source": r.source}
        if case["grad"]:
            (out["gradient"],) = torch.autograd.grad(r.weights, state["logits"], state["gradient"])
        return out
    if case["op"] == "exchange":
        r = routing.Routing(state["weights"], state["experts"], state["ends"], state["rows"], state["source"])
        sent = routing.dispatch_tokens(state["x"], r)
        back = routing.combine_tokens(state["y"], r)
        if not case["grad"]:
            return sent, back
        return sent, back, *torch.autograd.grad(sent, state["x"], state["x_gradient"]), *torch.autograd.grad(
            back, (state["y"], state["weights"]), state["y_gradient"])
    weight = _own_weight(state)
    if case["op"] == "linear":
        return int8.linear_int8(state["x"], weight)
    if case["op"] == "grouped":
        return int8.grouped_linear_int8(state["x"], weight, state["ends"])
    if case["op"] == "grad":
        return int8.linear_int8_grad_input(state["x"], weight)
    return int8.grouped_linear_int8_grad_input(state["x"], weight, state["ends"])


# ---------------------------------------------------------------------------------------- the plain form
def _quantized(x):
    """The codes of each row (whole numbers in fp32) and its scale. Codes next to a border of two are found in 64 bits."""
    top = x.double().abs().amax(-1, keepdim=True)
    codes = torch.round(x.double() * 127 / torch.where(top == 0, torch.ones_like(top), top))
    return codes.float(), top.float() / 127


def _row_scales(state):
    """The scale of each row of the weight (E, rows, 1), fp32."""
    case = state["case"]
    scale = state["scale"].float().reshape(max(1, case["experts"]), -1, 1)
    return (scale / 127 if case["weight"] == "bnb8" else scale).expand(-1, case["rows"], 1)


def _centred(state):
    """The weight's codes less their zero points (E, rows, cols), fp32."""
    codes = state["codes"].float().reshape(max(1, state["case"]["experts"]), state["case"]["rows"], -1)
    return codes if state["zero"] is None else codes - state["zero"].float().reshape(codes.shape[0], -1, 1)


def _places(state):
    """Each row's expert, its place in the expert's group, and whether it belongs to one."""
    ends = state["ends"].long()
    row = torch.arange(state["x"].shape[0], device="cuda")
    expert = torch.searchsorted(ends, row, right=True)
    inside = expert < ends.numel()
    expert = expert.clamp(max=ends.numel() - 1)
    start = torch.cat((ends.new_zeros(1), ends[:-1]))
    return expert, (row - start[expert]).clamp(0, state["capacity"] - 1), inside


def _product(x, w, state, grad):
    """x by each expert's w over the last axis (over w's rows for a gradient)."""
    if not state["case"]["experts"]:
        return x @ (w[0] if grad else w[0].T)
    expert, place, inside = _places(state)
    padded = x.new_zeros((w.shape[0], state["capacity"], x.shape[1]))
    padded.index_put_((expert, place), x * inside[:, None], accumulate=True)
    y = torch.bmm(padded, w if grad else w.transpose(1, 2))[expert, place]
    return torch.where(inside[:, None], y, torch.zeros_like(y))


def _scores(logits, scoring):
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _best(values, count):
    """The places of the ``count`` largest along the last axis, the largest first, equal ones by their index."""
    return torch.sort(values, dim=-1, descending=True, stable=True).indices[..., :count]


def _chosen(state):
    """Each token's experts. Scores next to one another are told apart in 64 bits; without a bias the logits' order is theirs."""
    case, logits = state["case"], state["logits"].detach().double()
    tokens, experts = logits.shape
    score = _scores(logits, case["scoring"])
    choice = logits if state["bias"] is None else score + state["bias"].double()
    if case["groups"] > 1:
        per = experts // case["groups"]
        by_group = choice.view(tokens, case["groups"], per)
        if case["group_score"] == "max":
            group = by_group.amax(-1)
        else:
            score = score if state["bias"] is None else choice
            group = torch.sort(score.view(tokens, case["groups"], per), dim=-1, descending=True).values[..., :2].sum(-1)
        kept = torch.zeros_like(group, dtype=torch.bool).scatter_(1, _best(group, case["top_groups"]), True)
        choice = torch.where(kept[..., None].expand(-1, -1, per).reshape(tokens, experts), choice, -math.inf)
    return _best(choice, case["top_k"])


def _plain_weights(logits, chosen, state):
    case = state["case"]
    weight = _scores(logits.float(), case["scoring"]).gather(1, chosen)
    if case["renormalize"]:
        weight = weight / weight.sum(-1, keepdim=True)
    weight = weight * case["scale"]
    return weight if state["mask"] is None else torch.where(state["mask"][:, None], weight, torch.zeros_like(weight))


def _order(chosen, state):
    """(experts, ends, rows, source): the choices in the order of their experts, and within one of their tokens."""
    experts, (tokens, top_k) = state["case"]["experts"], chosen.shape
    flat = chosen if state["mask"] is None else torch.where(state["mask"][:, None], chosen, experts)
    flat = flat.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    ends = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(0).cumsum(0)
    place = torch.empty_like(order)
    place[order] = torch.arange(flat.numel(), device=flat.device)
    inside = torch.arange(flat.numel(), device=flat.device) < ends[-1]
    return (torch.where(flat < experts, flat, -1).view(tokens, top_k).int(), ends.int(),
            torch.where(flat < experts, place, -1).view(tokens, top_k).int(), torch.where(inside, order, -1).int())


def _plain_route(state):
    chosen = _chosen(state)
    experts, ends, rows, source = _order(chosen, state)
    return {"weights": _plain_weights(state["logits"].detach(), chosen, state), "experts": experts, "ends": ends, "rows": rows,
            "source": source}


def _plain_route_gradient(state, chosen):
    """The logits' gradient: through the scale, the renormalisation, the scores."""
    case, logits = state["case"], state["logits"].detach().float()
    g = state["gradient"] * case["scale"]
    if state["mask"] is not None:
        g = torch.where(state["mask"][:, None], g, torch.zeros_like(g))
    score = _scores(logits, case["scoring"])
    picked = score.gather(1, chosen)
    if case["renormalize"]:
        total = picked.sum(-1, keepdim=True)
        g = (g - (g * picked / total).sum(-1, keepdim=True)) / total
    spread = torch.zeros_like(logits).scatter(1, chosen, g)
    if case["scoring"] == "sigmoid":
        d = spread * score * (1 - score)
    else:
        d = score * (spread - (spread * score).sum(-1, keepdim=True))
    return d.to(state["logits"].dtype)


def _plain_exchange(state):
    x, y, rows, source = state["x"].detach(), state["y"].detach(), state["rows"].long(), state["source"].long()
    top_k, sent_to = rows.shape[1], (rows >= 0)[..., None]
    inside = (source >= 0)[:, None]
    token = source.clamp(min=0) // top_k
    sent = torch.where(inside, x[token], torch.zeros_like(x[:1]))
    weights = state["weights"].detach()[..., None]
    mine = torch.where(sent_to, y[rows.clamp(min=0)].float(), torch.zeros((), device="cuda"))
    back = (mine * weights).sum(1).to(y.dtype)
    if not state["case"]["grad"]:
        return sent, back
    x_grad = torch.where(sent_to, state["x_gradient"][rows.clamp(min=0)].float(), torch.zeros((), device="cuda")).sum(1).to(x.dtype)
    g = state["y_gradient"].float()
    y_grad = torch.where(inside, g[token] * weights.reshape(-1, 1)[source.clamp(min=0)], torch.zeros((), device="cuda")).to(y.dtype)
    return sent, back, x_grad, y_grad, (mine * g[:, None]).sum(-1)


def _plain(state):
    case = state["case"]
    if case["op"] == "route":
        out = _plain_route(state)
        if case["grad"]:
            out["gradient"] = _plain_route_gradient(state, _chosen(state))
        return out
    if case["op"] == "exchange":
        return _plain_exchange(state)
    x = state["x"]
    if "grad" in case["op"]:
        return _product(x.float(), _centred(state) * _row_scales(state), state, True).to(x.dtype)
    codes, scale = _quantized(x)
    y = _product(codes, _centred(state), state, False)
    row_scales = _row_scales(state)[..., 0]
    return (y * scale * (row_scales if not case["experts"] else row_scales[_places(state)[0]])).to(x.dtype)


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------- the definition in 64 bits
def _exact_product(case, state):
    w = state["codes"].double()
    if state["zero"] is not None:
        w = w - state["zero"].double()
    w = w * (state["scale"].double().reshape(-1, 1) / 127 if case["weight"] == "bnb8" else state["scale"].double())
    x, grad = state["x"].double(), "grad" in case["op"]
    if not grad:
        unit = x.abs().max(dim=1, keepdim=True).values / 127
        # 127 x is held exactly, and so are the borders: half-way codes go to the even one
        whole = torch.floor(x.abs() * 127 / (unit * 127))
        over = 2 * (x.abs() * 127) - (2 * whole + 1) * (unit * 127)
        whole = whole + ((over > 0) | ((over == 0) & (whole % 2 == 1))).double()
        x = torch.sign(x) * whole * unit
    if not case["experts"]:
        return x @ (w if grad else w.T)
    y, at = x.new_zeros((x.shape[0], w.shape[2 if grad else 1])), 0
    for e, n in enumerate(_sizes(case)):
        y[at:at + n] = x[at:at + n] @ (w[e] if grad else w[e].T)
        at += n
    return y


def _exact_route(case, state):
    """Experts found one at a time, the weights' derivatives through the logarithms of scores."""
    logits = state["logits"].detach().double()
    tokens, experts = logits.shape
    score = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else torch.softmax(logits, 1)
    choice = logits.clone() if state["bias"] is None else score + state["bias"].double()
    if case["groups"] > 1:
        value = choice if case["group_score"] == "max" or state["bias"] is not None else score
        value = value.reshape(tokens * case["groups"], -1)
        first, at = value.max(dim=1)
        if case["group_score"] == "top2":
            first = first + value.scatter(1, at[:, None], -math.inf).max(dim=1).values
        order = first.view(tokens, -1)
        dropped = torch.ones_like(order, dtype=torch.bool)
        for _ in range(case["top_groups"]):
            at = order.max(dim=1).indices
            dropped[torch.arange(tokens), at] = False
            order = order.scatter(1, at[:, None], -math.inf)
        choice[dropped.repeat_interleave(experts // case["groups"], dim=1)] = -math.inf
    chosen = []
    for _ in range(case["top_k"]):
        best = choice.max(dim=1, keepdim=True).values
        at = (choice == best).int().argmax(dim=1, keepdim=True)
        chosen.append(at)
        choice = choice.scatter(1, at, -math.inf)
    chosen = torch.cat(chosen, 1)
    picked = score.gather(1, chosen)
    weights = picked / picked.sum(1, keepdim=True) if case["renormalize"] else picked
    weights = weights * case["scale"]
    if state["mask"] is not None:
        weights = weights * state["mask"][:, None].double()
    out = {"weights": weights, "experts": None, "ends": None, "rows": None, "source": None}
    if case["grad"]:
        # d weight_j = weight_j d log(weight_j); d log(sigmoid) = 1 - sigmoid, d log(softmax_e) = [e] - softmax
        g = state["gradient"].double() * weights
        if case["renormalize"]:
            share = picked / picked.sum(1, keepdim=True)
            g = g - g.sum(1, keepdim=True) * share
        if case["scoring"] == "sigmoid":
            out["gradient"] = torch.zeros_like(logits).scatter(1, chosen, g * (1 - picked))
        else:
            out["gradient"] = torch.zeros_like(logits).scatter(1, chosen, g) - g.sum(1, keepdim=True) * score
    return out


def _exact_exchange(case, state):
    top_k, hidden = case["top_k"], case["hidden"]
    flat, weights = state["rows"].reshape(-1).long(), state["weights"].detach().double().reshape(-1, 1)
    used = torch.nonzero(flat >= 0).reshape(-1)
    at, token = flat[used], used // top_k

    def zeros(n):
        return torch.zeros((n, hidden), dtype=torch.float64, device="cuda")

    x, y = state["x"].detach().double(), state["y"].detach().double()
    sent = zeros(flat.numel())
    sent[at] = x[token]
    back = zeros(x.shape[0]).index_add_(0, token, y[at] * weights[used])
    if not case["grad"]:
        return sent, back
    x_grad = zeros(x.shape[0]).index_add_(0, token, state["x_gradient"].double()[at])
    g, y_grad = state["y_gradient"].double(), zeros(flat.numel())
    y_grad[at] = g[token] * weights[used]
    w_grad = torch.zeros(flat.numel(), dtype=torch.float64, device="cuda")
    w_grad[used] = (y[at] * g[token]).sum(1)
    return sent, back, x_grad, y_grad, w_grad.view(-1, top_k)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, state)
    if case["op"] == "exchange":
        return _exact_exchange(case, state)
    return _exact_product(case, state) if work(case)["flops"] <= EXACT_FLOPS else None
