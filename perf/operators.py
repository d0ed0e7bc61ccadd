"""The 4-bit floating-point operators as workloads: quantisation, products and gradients.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes a case's inputs
on the GPU, ``run(state)`` is one pass and ``work(case)`` what a pass cannot do without. With ``own`` true ``run`` calls
``piper_offload_b200.fp4``; with ``own`` false it computes the same operators from elementary torch operations in 32
bits. ``exact(case, seed)`` is the definition in 64 bits.

Operators
  quantize       a dense matrix to MXFP4 (32 values share a power of two) or NVFP4 (16 values share an e4m3 scale, with
                 an fp32 scale over all of it when ``levels`` is 2), returned as the values the codes stand for
  linear         tokens times a packed weight, the tokens quantised to the weight's format on the way
  grouped        the same with a weight per expert and the tokens sorted by expert
  grad           the gradient of ``linear`` with respect to the tokens (the weight is frozen)
  grouped_grad   the gradient of ``grouped`` with respect to the tokens
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
EXACT_FLOPS = 1.2e14  # a 64-bit product above this takes too long


# ----------------------------------------------------------------------------------------------- cases
def _case(name, op, fmt, tokens, rows, cols, *, experts=0, skew=0.0, empty_every=0, tail=0, levels=1, act_scale=False,
          swizzled=True, mode="floor", dtype="bfloat16"):
    case = {"op": op, "format": fmt, "tokens": tokens, "rows": rows, "cols": cols, "experts": experts, "skew": skew,
            "empty_every": empty_every, "tail": tail, "levels": levels, "act_scale": act_scale, "swizzled": swizzled,
            "mode": mode, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a small projection with ragged sides, as an adapter's or router's weight: a call's own cost
        _case("quantize small odd", "quantize", "nvfp4", 0, 70, 208, levels=2, swizzled=False),
        # an MLP weight of the DiT-shaped stack made ready for merging
        _case("quantize mx 12288x3072", "quantize", "mxfp4", 0, 12288, 3072, mode="rceil"),
        # a Llama-3-8B-shaped down projection from an fp32 checkpoint, two-level
        _case("quantize nv 4096x14336 fp32", "quantize", "nvfp4", 0, 4096, 14336, levels=2, dtype="float32"),
        # one token of decoding through the gate projection
        _case("linear nv 1 token", "linear", "nvfp4", 1, 14336, 4096, levels=2),
        # a batch of decoding sequences through an attention projection, scales as plain rows
        _case("linear mx 24 tokens", "linear", "mxfp4", 24, 4096, 4096, swizzled=False),
        # a short ragged prompt and an odd output width
        _case("linear mx 333 odd", "linear", "mxfp4", 333, 1000, 2080, mode="even"),
        # a long prompt through the gate projection, activations with a calibrated second-level scale
        _case("linear nv 4096 tokens", "linear", "nvfp4", 4096, 14336, 4096, levels=2, act_scale=True),
        # a decoding step over a layer of experts, two of which get nothing
        _case("grouped nv 16 rows 8 experts", "grouped", "nvfp4", 16, 14336, 4096, experts=8, skew=0.5, empty_every=4,
              levels=2),
        # a prompt over many small experts, uneven, the last rows being padding of a fixed-capacity buffer
        _case("grouped mx 4096 rows 32 experts", "grouped", "mxfp4", 4096, 2048, 2048, experts=32, skew=0.6,
              empty_every=8, tail=96),
        # a middling batch with sizes that fill no tile
        _case("grouped nv 777 rows 12 experts", "grouped", "nvfp4", 777, 1040, 1072, experts=12, skew=0.3),
        # training adapters over a frozen Llama-3-8B-shaped projection
        _case("grad nv 2048 tokens", "grad", "nvfp4", 2048, 14336, 4096, levels=2),
        # the same over experts
        _case("grouped grad mx 2048 rows 16 experts", "grouped_grad", "mxfp4", 2048, 2048, 2048, experts=16, skew=0.6,
              empty_every=8),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: sizes spread over the listed ones' ranges, most of them no multiple of a tile."""
    op = rng.choice(["quantize", "linear", "linear", "grouped", "grouped", "grad", "grouped_grad"])
    fmt = rng.choice(["mxfp4", "nvfp4"])
    block = BLOCK[fmt]
    levels = rng.choice([1, 2]) if fmt == "nvfp4" else 1
    mode = rng.choice(["floor", "rceil", "ceil", "even"]) if fmt == "mxfp4" else "floor"
    swizzled = rng.random() < 0.6
    kw = {"levels": levels, "mode": mode, "swizzled": swizzled}
    if op == "quantize":
        return _case(None, op, fmt, 0, _log_int(rng, 64, 8192), block * _log_int(rng, 4, 8192 // block),
                     dtype=rng.choice(["bfloat16", "float32"]), **kw)
    if op in ("linear", "grad"):
        rows, cols = _log_int(rng, 128, 14336), block * _log_int(rng, 128 // block, 8192 // block)
        tokens = _log_int(rng, 1, 4096) if op == "linear" else _log_int(rng, 16, 2048)
        tokens = min(tokens, 4096 * 14336 * 4096 // (rows * cols))
        return _case(None, op, fmt, tokens, rows, cols,
                     act_scale=op == "linear" and levels == 2 and rng.random() < 0.5, **kw)
    experts = _log_int(rng, 4, 48)
    return _case(None, op, fmt, _log_int(rng, 8, 4096), _log_int(rng, 256, 2816), block * _log_int(rng, 256 // block, 2816 // block),
                 experts=experts, skew=round(rng.uniform(0.0, 0.8), 2), empty_every=rng.choice([0, 0, 3, 5, 8]),
                 tail=rng.choice([0, 0, 5]), **kw)


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
    rows, cols, tokens, block = case["rows"], case["cols"], case["tokens"], BLOCK[case["format"]]
    packed = rows * cols / 2 + rows * cols / block
    wide = DTYPES[case["dtype"]].itemsize
    if case["op"] == "quantize":
        return {"bytes": 2 * rows * cols * wide + packed, "flops": 0}  # the matrix, its codes and the values they stand for
    used, weights = tokens, 1
    if case["experts"]:
        sizes = _sizes(case)
        used, weights = sum(sizes), sum(n > 0 for n in sizes)
    return {"bytes": weights * packed + (used * (cols if "grad" not in case["op"] else rows) + tokens *
                                         (rows if "grad" not in case["op"] else cols)) * wide,
            "flops": 2.0 * used * rows * cols}


# ---------------------------------------------------------------------------------------------- inputs
def _swizzle(scale, padding):
    """Row-major block scales (E, R, C) in tiles of 128 rows x 4 scales: byte (r % 32) * 16 + (r / 32) * 4 + c of a tile."""
    e, r, c = scale.shape
    rp, cp = -(-r // 128) * 128, -(-c // 4) * 4
    full = torch.full((e, rp, cp), padding, dtype=torch.uint8, device=scale.device)
    full[:, :r, :c] = scale
    return full.view(e, rp // 128, 4, 32, cp // 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(e, rp // 4, cp * 4).contiguous()


def _weight(case, generator):
    """Packed codes, scale bytes and second-level scales of normal weights (E, rows, cols)."""
    e, rows, cols, fmt = max(1, case["experts"]), case["rows"], case["cols"], case["format"]
    block = BLOCK[fmt]
    codes, scales, second = [], [], []
    for _ in range(e):
        w = torch.randn((rows, cols // block, block), generator=generator, device="cuda") * 0.02
        top = w.abs().amax(-1, keepdim=True)
        if fmt == "mxfp4":
            exponent = torch.frexp(top).exponent - 3
            byte, unit = (exponent + 127).clamp(0, 254).to(torch.uint8), torch.exp2(exponent.float())
        else:
            g = w.abs().max() / 2688 if case["levels"] == 2 else torch.ones((), device="cuda")
            second.append(g.reshape(1))
            # without a second level the small weights need a larger unit to keep their bits
            w, top = (w, top) if case["levels"] == 2 else (w * 64, top * 64)
            e4m3 = (top / 6 / g).clamp(0.015625, 448.0).to(torch.float8_e4m3fn)
            byte, unit = e4m3.view(torch.uint8), e4m3.float() * g
        m = (w / unit).clamp(-6, 6)
        magnitude = m.abs()
        step = torch.where(magnitude < 2, 0.5, torch.where(magnitude < 4, 1.0, 2.0))
        q = torch.round(magnitude / step) * step
        code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8) | (m < 0).to(torch.uint8) * 8
        code = code.view(rows, cols)
        codes.append(code[:, 0::2] | code[:, 1::2] << 4)
        scales.append(byte.view(rows, cols // block))
    scale = torch.stack(scales)
    if case["swizzled"]:
        scale = _swizzle(scale, 0)
    return torch.stack(codes).contiguous(), scale, torch.cat(second) if case["levels"] == 2 else None


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    dtype, state = DTYPES[case["dtype"]], {"case": case}
    rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
    if case["op"] == "quantize":
        state["dense"] = (torch.randn((rows, cols), generator=generator, device="cuda") * 0.02).to(dtype)
        if case["levels"] == 1 and case["format"] == "nvfp4":
            state["dense"] *= 64
        return state
    codes, scale, second = _weight(case, generator)
    if not case["experts"]:
        codes, scale = codes[0], scale[0]
    state.update(codes=codes, second=second)
    state["scale"] = scale.view(torch.float8_e4m3fn) if case["format"] == "nvfp4" else scale
    if "grad" in case["op"]:
        state["x"] = (torch.randn((tokens, rows), generator=generator, device="cuda") * 1e-3).to(dtype)
    else:
        # activations after a norm: unit scale, with a few channels far larger
        x = torch.randn((tokens, cols), generator=generator, device="cuda")
        x *= torch.where(torch.rand(cols, generator=generator, device="cuda") < 0.005, 20.0, 1.0)
        state["x"] = x.to(dtype)
    # calibration saw a largest activation of about 80
    amax = 70 + 20 * torch.rand(1, generator=generator, device="cuda")
    state["act_scale"] = amax / 2688 if case["act_scale"] else None
    if case["experts"]:
        sizes = _sizes(case)
        state["ends"] = torch.tensor(sizes, device="cuda").cumsum(0).to(torch.int32)
        state["capacity"] = max(1, max(sizes))
    return state


# ---------------------------------------------------------------------------------------- the framework
def _own_weight(state):
    from piper_offload_b200 import weights as W

    case = state["case"]
    kw = {"per_tensor_scale": state["second"]} if case["format"] == "nvfp4" else {
        "elem_dtype": torch.float4_e2m1fn_x2, "act_quant_kwargs": W.MXActQuantKwargs(W.MXScalingMode(case["mode"]))}
    kind = {"mxfp4": (W.MXWeight, W.MXExperts), "nvfp4": (W.NVFP4Weight, W.NVFP4Experts)}[case["format"]]
    return kind[case["experts"] > 0](state["codes"], state["scale"], is_swizzled_scales=case["swizzled"], **kw)


def _own(state):
    from piper_offload_b200 import fp4

    case = state["case"]
    if case["op"] == "quantize":
        if case["format"] == "mxfp4":
            packed = fp4.quantize_mxfp4(state["dense"], scaling_mode=case["mode"], swizzled=case["swizzled"])
        else:
            packed = fp4.quantize_nvfp4(state["dense"], two_level=case["levels"] == 2, swizzled=case["swizzled"])
        return fp4.dequantize_fp4(packed)
    weight = _own_weight(state)
    if case["op"] == "linear":
        return fp4.linear_fp4(state["x"], weight, act_per_tensor_scale=state["act_scale"])
    if case["op"] == "grouped":
        return fp4.grouped_linear_fp4(state["x"], weight, state["ends"], act_per_tensor_scale=state["act_scale"])
    if case["op"] == "grad":
        return fp4.linear_fp4_grad_input(state["x"], weight)
    return fp4.grouped_linear_fp4_grad_input(state["x"], weight, state["ends"])


# ---------------------------------------------------------------------------------------- the plain form
def _round_e2m1(v):
    m = v.abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return torch.copysign(torch.round(m / step) * step, v)


def _quantized(x, case, g):
    """The fp32 values (without the second-level scale ``g``) that x stands for after quantisation."""
    block = BLOCK[case["format"]]
    b = x.float().view(x.shape[0], -1, block)
    top = b.abs().amax(-1, keepdim=True)
    six = torch.full_like(top, 6.0)
    if case["format"] == "mxfp4":
        mode = case["mode"]
        bits = (top / six if mode == "rceil" else top).view(torch.int32)
        if mode == "even":
            bits = bits + (1 << 21)
        exponent = (bits >> 23) + ((bits & 0x7FFFFF) != 0).int() * (mode in ("ceil", "rceil"))
        exponent = (exponent - (0 if mode == "rceil" else 2)).clamp(0, 254)
        unit = torch.where(exponent == 0, torch.full_like(exponent, 1 << 22), exponent << 23).view(torch.float32)
        return (_round_e2m1((b / unit).clamp(-6, 6)) * unit).view(x.shape)
    s = top / six
    if g is not None:
        s = s / g
    unit = s.clamp(0.015625, 448.0).to(torch.float8_e4m3fn).float()
    v = b / unit if g is None else b * (torch.ones_like(g) / g / unit)
    return (_round_e2m1(v.clamp(-6, 6)) * unit).view(x.shape)


def _block_scales(state):
    """The weight's block scales as fp32, row-major (E, rows, blocks)."""
    case = state["case"]
    rows, blocks = case["rows"], case["cols"] // BLOCK[case["format"]]
    byte = state["scale"].view(torch.uint8)
    byte = byte.view(max(1, case["experts"]), *byte.shape[-2:])
    if case["swizzled"]:
        e, rt, ct = byte.shape[0], -(-rows // 128), -(-blocks // 4)
        byte = byte.view(e, rt, ct, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(e, rt * 128, ct * 4)[:, :rows, :blocks]
    if case["format"] == "nvfp4":
        return byte.contiguous().view(torch.float8_e4m3fn).float()
    return torch.exp2(byte.float() - 127)


def _values(state, dtype=torch.float32):
    """The weight's values without the second-level scales, (E, rows, cols)."""
    case = state["case"]
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda", dtype=dtype)
    codes = state["codes"].view(max(1, case["experts"]), case["rows"], -1)
    v = torch.stack((grid[(codes & 15).int()], grid[(codes >> 4).int()]), dim=-1)
    scales = _block_scales(state).to(dtype)
    return (v.view(*scales.shape, -1) * scales[..., None]).view(*scales.shape[:2], case["cols"])


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
    """x by each expert's w over the last axis (over w's rows for a gradient), in x's type."""
    if not state["case"]["experts"]:
        return x @ (w[0] if grad else w[0].T)
    expert, place, inside = _places(state)
    padded = x.new_zeros((w.shape[0], state["capacity"], x.shape[1]))
    padded.index_put_((expert, place), x * inside[:, None], accumulate=True)
    y = torch.bmm(padded, w if grad else w.transpose(1, 2))[expert, place]
    return torch.where(inside[:, None], y, torch.zeros_like(y))


def _second(state, rows):
    """The second-level scale of each row of the output, or None."""
    if state["second"] is None:
        return None
    if not state["case"]["experts"]:
        return state["second"]
    return state["second"][_places(state)[0]][:, None]


def _plain(state):
    case = state["case"]
    if case["op"] == "quantize":
        x = state["dense"]
        g = (x.float().abs().max() / torch.full((), 2688.0, device="cuda")).clamp_min(2.0 ** -23) if case["levels"] == 2 else None
        v = _quantized(x, case, g)
        return (v if g is None else v * g).to(x.dtype)
    x, w = state["x"], _values(state)
    if "grad" in case["op"]:
        y = _product(x.float(), w, state, True)
    else:
        y = _product(_quantized(x, case, state["act_scale"]), w, state, False)
        if state["act_scale"] is not None:
            y = y * state["act_scale"]
    second = _second(state, x.shape[0])
    return (y if second is None else y * second).to(x.dtype)


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------- the definition in 64 bits
def _exact_quantized(x, case, g):
    block = BLOCK[case["format"]]
    b = x.double().reshape(-1, block)
    top = b.abs().max(dim=1).values
    if case["format"] == "mxfp4":
        mantissa, exponent = torch.frexp(top)  # top = mantissa * 2**exponent, mantissa in [0.5, 1)
        if case["mode"] == "rceil":
            mantissa, exponent = torch.frexp(top / 6)
            power = exponent - (mantissa == 0.5).int()
        else:
            power = exponent - 3
            if case["mode"] == "ceil":
                power = power + (mantissa > 0.5).int()
            elif case["mode"] == "even":
                power = power + (mantissa >= 0.875).int()
        unit = torch.ldexp(torch.ones_like(top), power.clamp(-127, 127))
    else:
        unit = (top / 6 / (1 if g is None else g.double())).clamp(0.015625, 448.0)
        # e4m3: 3 mantissa bits from 2**-6 up
        quantum = torch.exp2(torch.floor(torch.log2(unit)) - 3)
        unit = torch.round(unit / quantum) * quantum
    whole = unit if g is None else unit * g.double()
    v = (b / whole[:, None]).clamp(-6, 6)
    m = v.abs()
    # the midpoints between neighbours go to the neighbour with the even code
    out = torch.zeros_like(m)
    for low, value, closed in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True),
                               (2.5, 3.0, False), (3.5, 4.0, True), (5.0, 6.0, False)):
        out = torch.where((m >= low) if closed else (m > low), torch.full_like(m, value), out)
    return (torch.where(v < 0, -out, out) * whole[:, None]).view(x.shape)


def exact(case, seed):
    if work(case)["flops"] > EXACT_FLOPS:
        return None
    state = prepare(case, seed)
    if case["op"] == "quantize":
        x = state["dense"]
        g = (x.double().abs().max() / 2688).clamp_min(2.0 ** -23) if case["levels"] == 2 else None
        return _exact_quantized(x, case, g)
    grad = "grad" in case["op"]
    x = state["x"].double() if grad else _exact_quantized(state["x"], case, state["act_scale"])
    w = _values(state, torch.float64)
    if state["second"] is not None:
        w = w * state["second"].double()[:, None, None]
    if not case["experts"]:
        return x @ (w[0] if grad else w[0].T)
    y, at = x.new_zeros((x.shape[0], w.shape[2 if grad else 1])), 0
    for e, n in enumerate(_sizes(case)):
        y[at:at + n] = x[at:at + n] @ (w[e] if grad else w[e].T)
        at += n
    return y
