"""Measured cases of the 8-bit integer operators and of routing: quantisation with a scale for each token or channel, the
product of two such operands, the choice of experts with its plan, and the experts' two products on that plan.

An i8 operand is `rows` rows of k codes -127..127, k padded with zeros to kp, a multiple of 128, and an fp32 scale for
each row: codes [rows, kp], scales [rows]; a code stands for code x scale. The scale is the row's largest magnitude / 127,
rounded to fp32; a code is the exact quotient x / scale rounded to the nearest integer, ties to the even one.

A plan says which expert takes which token: a pair is token x top_k + place, order[slot] a pair, slots sorted by expert
and within it by pair, expert e's from offsets[e] to offsets[e + 1].

Sizes are those of the shipped MLP graphs and of the benchmark's GEMMs (512 x 2048, 4096 x 14336), of the
mixture-of-experts cases measured beside these, and odd ones between them."""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}
MOST_ELEMENTS = 4096 * 14336              # of a quantised tensor
MOST_MULTIPLY_ADDS = 4096 * 4096 * 14336  # of a product
MOST_EXPERT_WEIGHTS = 64 * 2048 * 2048    # of one of the experts' products
MOST_SLOTS = 2048 * 8                     # tokens x experts of each


def listed():
    return [
        # One token's activations before a layer: latency only.
        {"name": "quantize_one_row", "op": "quantize", "form": "rows", "type": "bf16", "rows": 1, "k": 4096, "pad": 0},
        # The hidden activations of the benchmark's MLP block.
        {"name": "quantize_8192_rows", "op": "quantize", "form": "rows", "type": "f32", "rows": 8192, "k": 2048, "pad": 0},
        # A layer's weights at load, odd sizes, a view of wider rows, stored [k, n] as the matmuls take B.
        {"name": "quantize_columns_odd", "op": "quantize", "form": "columns", "type": "f16", "rows": 2047, "k": 1001,
         "pad": 7},
        # One token through the benchmark's FFN: the weights' bytes.
        {"name": "i8_one_row", "op": "product", "m": 1, "n": 14336, "k": 4096, "out": "bf16", "bias": False, "act": "none"},
        # A prompt through a layer whose sizes no tile divides, with bias and activation.
        {"name": "i8_ragged", "op": "product", "m": 1000, "n": 1001, "k": 1023, "out": "f32", "bias": True, "act": "gelu"},
        # The FFN shape of the benchmark.
        {"name": "i8_ffn", "op": "product", "m": 4096, "n": 14336, "k": 4096, "out": "bf16", "bias": False, "act": "none"},
        # One token of a decoding step: latency only.
        {"name": "route_one_token", "op": "route", "type": "f32", "tokens": 1, "experts": 64, "top_k": 8,
         "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_best": 1, "normalize": True, "scale": 1.0},
        # A long prompt, groups of experts and a bias that keeps them evenly used.
        {"name": "route_8192_tokens", "op": "route", "type": "bf16", "tokens": 8192, "experts": 256, "top_k": 8,
         "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "group_best": 2, "normalize": True, "scale": 2.5},
        # One token of a decoding step: its eight experts' weights.
        {"name": "up_one_token", "op": "up", "type": "bf16", "tokens": 1, "d": 2048, "h": 1024, "experts": 64, "top_k": 8,
         "bias": False, "act": "swiglu"},
        # A prompt on the same experts.
        {"name": "up_2048_tokens", "op": "up", "type": "bf16", "tokens": 2048, "d": 2048, "h": 1024, "experts": 64,
         "top_k": 8, "bias": False, "act": "swiglu"},
        # A serving batch at the shipped MLP block's width, an odd one inside, biases, fp32 result.
        {"name": "down_16_tokens", "op": "down", "type": "f32", "tokens": 16, "d": 512, "h": 2047, "experts": 8, "top_k": 2,
         "bias": True},
        # The prompt's way back.
        {"name": "down_2048_tokens", "op": "down", "type": "bf16", "tokens": 2048, "d": 2048, "h": 1024, "experts": 64,
         "top_k": 8, "bias": False},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, even over its logarithm: as it falls, or a multiple of 8 or of 64."""
    hi = max(lo, hi)
    n = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    step = rng.choice((1, 1, 8, 64))
    return max(lo, min(hi, (n + step - 1) // step * step))


def draw(rng):
    op = rng.choice(("quantize", "product", "route", "up", "down"))
    if op == "quantize":
        k = _size(rng, 32, 14336)
        return {"op": op, "form": rng.choice(("rows", "columns")), "type": rng.choice(sorted(TYPES)),
                "rows": _size(rng, 1, min(8192, MOST_ELEMENTS // 4 // k)), "k": k, "pad": rng.choice((0, 0, 1, 8, 24))}
    if op == "product":
        k = _size(rng, 64, 8192)
        n = _size(rng, 64, min(14336, MOST_ELEMENTS // k))
        # Rows from one token on; half of them the few of a decoding step.
        most = min(4096, MOST_MULTIPLY_ADDS // (n * k)) if rng.random() < 0.5 else 64
        act = rng.choice(("none", "none", "relu", "gelu", "swiglu"))
        return {"op": op, "m": _size(rng, 1, most), "n": max(1, n // 2) if act == "swiglu" else n, "k": k,
                "out": rng.choice(sorted(TYPES)), "bias": rng.random() < 0.5, "act": act}
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        each = rng.choice((4, 7, 8, 16, 31, 32, 48) if groups > 1 else (4, 8, 16, 31, 60, 64, 128, 256, 384))
        top_groups = rng.randint(1, groups)
        return {"op": op, "type": rng.choice(sorted(TYPES)), "tokens": _size(rng, 1, 16384), "experts": groups * each,
                "top_k": rng.randint(1, min(8, top_groups * each)), "score": rng.choice(("softmax", "sigmoid")),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "group_best": rng.choice((1, 2)),
                "normalize": rng.random() < 0.7, "scale": rng.choice((1.0, 1.0, 2.5))}
    experts = rng.choice((4, 8, 16, 31, 64, 128))
    top_k = rng.randint(1, min(8, experts))
    d = _size(rng, 256, 4096)
    act = rng.choice(("relu", "gelu", "swiglu")) if op == "up" else "none"
    mats = 2 if act == "swiglu" else 1
    h = _size(rng, 128, min(4096, MOST_EXPERT_WEIGHTS // (mats * d * experts)))
    tokens = _size(rng, 1, min(4096, MOST_SLOTS // top_k) if rng.random() < 0.5 else 64)
    case = {"op": op, "type": rng.choice(sorted(TYPES)), "tokens": tokens, "d": d, "h": h, "experts": experts,
            "top_k": top_k, "bias": rng.random() < 0.5}
    return {**case, "act": act} if op == "up" else case


# ---------------------------------------------------------------- the operators in elementary operations


def _padded(k):
    return (k + 127) // 128 * 128


def _quantize(x):
    """Rows [..., k] to (whole fp32 codes [..., k], fp32 scales [..., 1]); finite inputs. In 64 bits, where a quotient
    next to a half stays on its side of it."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / 127.0).float()
    code = torch.round(x / torch.where(scale > 0, scale, 1.0).double())
    return torch.where(scale > 0, code, 0.0).clamp(-127, 127).float(), scale


def _operand(x):
    """The operand of rows [..., k]: codes [..., kp] and scales [...]."""
    code, scale = _quantize(x)
    code = torch.nn.functional.pad(code, (0, _padded(x.shape[-1]) - x.shape[-1]))
    return code.to(torch.int8).contiguous(), scale.squeeze(-1).contiguous()


def _act(u, act):
    if act == "relu":
        return torch.relu(u)
    if act == "gelu":
        return 0.5 * u * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (u + 0.044715 * u * u * u)))
    if act == "swiglu":
        gate, up = u.chunk(2, -1)
        return gate * torch.sigmoid(gate) * up
    return u


def _plan(chosen, experts):
    """order and offsets of chosen [tokens, top_k]."""
    expert, order = torch.sort(chosen.reshape(-1), stable=True)
    offsets = torch.searchsorted(expert, torch.arange(experts + 1, device=DEVICE, dtype=expert.dtype))
    return order.int(), offsets.int()


def _largest(keys, count):
    """The places of the `count` largest along the last axis, ties to the lowest place."""
    return torch.sort(keys, dim=-1, descending=True, stable=True)[1][..., :count]


def _route(case, logits, bias):
    """In 64 bits, where two scores next to each other keep their order."""
    l = logits.double()
    score = torch.softmax(l, -1) if case["score"] == "softmax" else torch.sigmoid(l)
    # One score by itself is as large as its logit.
    key = score + bias.double() if bias is not None else score if case["group_best"] > 1 and case["groups"] > 1 else l
    if case["groups"] > 1:
        by_group = key.reshape(len(key), case["groups"], -1)
        best = torch.sort(by_group, -1, descending=True)[0][..., :case["group_best"]].sum(-1)
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(-1, _largest(best, case["top_groups"]), True)
        key = torch.where(kept.unsqueeze(-1), by_group, -math.inf).reshape(key.shape)
    chosen = _largest(key, case["top_k"])
    gate = torch.gather(score, -1, chosen)
    if case["normalize"]:
        gate = gate / gate.sum(-1, keepdim=True)
    order, offsets = _plan(chosen, case["experts"])
    return {"chosen": chosen.int(), "gates": (gate * case["scale"]).float(), "order": order, "offsets": offsets}


def _experts(state, a, scales, rows, act):
    """act(A W^T + b) of each slot in fp32; a: fp32 codes and scales of the rows that the slots take. Experts' slots side
    by side, padded to the most that one has."""
    offsets, (codes, weight_scales) = state["offsets"].long(), state["w"]
    slots = torch.arange(rows, device=DEVICE)
    expert = torch.searchsorted(offsets, slots, right=True) - 1
    place = slots - offsets[expert]
    side = torch.zeros(len(codes), state["most"], a.shape[-1], device=DEVICE)
    side[expert, place] = a
    out = torch.bmm(side, codes.float().transpose(1, 2).contiguous())[expert, place]
    out = out * scales.unsqueeze(-1) * weight_scales[expert]
    if state["b"] is not None:
        out = out + state["b"][expert]
    return _act(out, act)


# ---------------------------------------------------------------- inputs


def _normal(gen, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(0.0, std, generator=gen)


def _activations(gen, shape):
    """Normal values with channels of different strength, as activations have them."""
    return _normal(gen, shape) * torch.exp(0.5 * _normal(gen, shape[-1:]))


def _logits(gen, tokens, experts):
    """Some experts are more popular than others."""
    return _normal(gen, [tokens, experts], 1.5) + _normal(gen, [experts], 0.5)


def _weights(gen, experts, rows, k):
    """Experts' weights, a few experts at a time: fp32 ones of all would be large."""
    parts = [_operand(_normal(gen, [min(16, experts - e), rows, k], k ** -0.5)) for e in range(0, experts, 16)]
    return tuple(torch.cat(t) for t in zip(*parts))


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]
    if op == "quantize":
        shape = [case["rows"], case["k"]] if case["form"] == "rows" else [case["k"], case["rows"]]
        wide = _activations(gen, [shape[0], shape[1] + case["pad"]]).to(TYPES[case["type"]])
        return {"x": wide[:, :shape[1]]}
    if op == "product":
        rows = 2 * case["n"] if case["act"] == "swiglu" else case["n"]
        return {"a": _operand(_activations(gen, [case["m"], case["k"]])),
                "b": _operand(_normal(gen, [rows, case["k"]], case["k"] ** -0.5)),
                "bias": _normal(gen, [rows], 0.1) if case["bias"] else None}
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    logits = _logits(gen, tokens, experts)
    if op == "route":
        return {"logits": logits.to(TYPES[case["type"]]), "bias": _normal(gen, [experts], 0.1) if case["bias"] else None}
    chosen = _largest(logits, top_k)
    order, offsets = _plan(chosen, experts)
    t = {"order": order, "offsets": offsets, "most": int(offsets.diff().max())}
    if op == "up":
        rows, k = case["h"] * (2 if case["act"] == "swiglu" else 1), case["d"]
        t["a"] = _operand(_activations(gen, [tokens, k]))
    else:
        rows, k = case["d"], case["h"]
        # Most hidden activations are small, as behind a gate.
        t["a"] = _operand(_activations(gen, [tokens * top_k, k]) * torch.sigmoid(_normal(gen, [tokens * top_k, k], 2.0)))
        gate = torch.gather(torch.softmax(logits, -1), -1, chosen)
        t["gates"] = (gate / gate.sum(-1, keepdim=True)).contiguous()
    t["w"] = _weights(gen, experts, rows, k)
    t["b"] = _normal(gen, [experts, rows], 0.1) if case["bias"] else None
    return t


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if not own:
        return state
    import minicompiler_amd as mc

    mc.library()
    op = case["op"]
    # On the stream that the program's tensors are made on.
    state["mc"], state["stream"] = mc, torch.cuda.current_stream().cuda_stream
    workspace = 0
    if op == "quantize":
        x = state["x"]
        state["codes"] = torch.empty(mc.i8_code_bytes(case["rows"], case["k"]), dtype=torch.int8, device=DEVICE)
        state["scales"] = torch.empty(case["rows"], dtype=torch.float32, device=DEVICE)
        state["out"] = torch.empty(x.shape, dtype=x.dtype, device=DEVICE)
    elif op == "product":
        state["out"] = torch.empty([case["m"], case["n"]], dtype=TYPES[case["out"]], device=DEVICE)
    elif op == "route":
        tokens, top_k = case["tokens"], case["top_k"]
        state["out"] = {"chosen": torch.empty([tokens, top_k], dtype=torch.int32, device=DEVICE),
                        "gates": torch.empty([tokens, top_k], dtype=torch.float32, device=DEVICE),
                        "order": torch.empty(tokens * top_k, dtype=torch.int32, device=DEVICE),
                        "offsets": torch.empty(case["experts"] + 1, dtype=torch.int32, device=DEVICE)}
        workspace = mc.route_workspace_bytes(tokens, case["experts"], top_k)
    elif op == "up":
        shape = [case["tokens"] * case["top_k"], case["h"]]
        state["out"] = torch.empty(shape, dtype=TYPES[case["type"]], device=DEVICE)
    else:
        state["out"] = torch.empty([case["tokens"], case["d"]], dtype=TYPES[case["type"]], device=DEVICE)
        workspace = mc.experts_down_i8_workspace_bytes(CODES[case["type"]], case["tokens"], case["top_k"], case["d"],
                                                       case["h"])
    state["workspace"] = torch.zeros(workspace, dtype=torch.uint8, device=DEVICE) if workspace else None
    torch.cuda.synchronize()
    return state


# ---------------------------------------------------------------- one pass


def _address(t):
    return t.data_ptr() if t is not None else None


def _act_name(case):
    return None if case["act"] == "none" else case["act"]


def _run_own(state):
    mc, case, stream, out = state["mc"], state["case"], state["stream"], state["out"]
    op, workspace = case["op"], _address(state["workspace"])
    if op == "quantize":
        x, codes, scales = state["x"], state["codes"], state["scales"]
        if case["form"] == "rows":
            mc.quantize_i8(CODES[case["type"]], x.data_ptr(), x.stride(0), codes.data_ptr(), scales.data_ptr(),
                           case["rows"], case["k"], out.data_ptr(), stream)
        else:
            mc.quantize_i8_columns(CODES[case["type"]], x.data_ptr(), x.stride(0), codes.data_ptr(), scales.data_ptr(),
                                   case["k"], case["rows"], out.data_ptr(), stream)
        return {"values": out, "scales": scales}
    if op == "route":
        mc.launch_route(CODES[case["type"]], state["logits"].data_ptr(), case["experts"], _address(state["bias"]),
                        case["tokens"], case["experts"], case["top_k"], case["score"], case["groups"],
                        case["top_groups"], case["group_best"], case["normalize"], case["scale"],
                        out["chosen"].data_ptr(), out["gates"].data_ptr(), out["order"].data_ptr(),
                        out["offsets"].data_ptr(), stream, workspace)
        return out
    a, a_scales = state["a"]
    if op == "product":
        b, b_scales = state["b"]
        mc.launch_matmul_i8(a.data_ptr(), a_scales.data_ptr(), b.data_ptr(), b_scales.data_ptr(),
                            _address(state["bias"]), _act_name(case), CODES[case["out"]], out.data_ptr(), case["m"],
                            case["n"], case["k"], stream)
        return out
    w, w_scales = state["w"]
    if op == "up":
        mc.launch_experts_up_i8(a.data_ptr(), a_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(),
                                _address(state["b"]), _act_name(case), CODES[case["type"]], out.data_ptr(),
                                state["order"].data_ptr(), state["offsets"].data_ptr(), case["tokens"], case["top_k"],
                                case["experts"], case["h"], case["d"], stream)
    else:
        mc.launch_experts_down_i8(a.data_ptr(), a_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(),
                                  _address(state["b"]), CODES[case["type"]], out.data_ptr(), state["order"].data_ptr(),
                                  state["offsets"].data_ptr(), state["gates"].data_ptr(), case["tokens"],
                                  case["top_k"], case["experts"], case["d"], case["h"], stream, workspace)
    return out


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        x = state["x"] if case["form"] == "rows" else state["x"].t()
        code, scale = _quantize(x)
        v = (code * scale).to(x.dtype)
        return {"values": v if case["form"] == "rows" else v.t().contiguous(), "scales": scale.squeeze(-1)}
    if op == "route":
        return _route(case, state["logits"], state["bias"])
    codes, scales = state["a"]
    a = codes.float()
    if op == "product":
        b, b_scales = state["b"]
        u = (a @ b.float().t()) * scales.unsqueeze(-1) * b_scales
        if state["bias"] is not None:
            u = u + state["bias"]
        return _act(u, case["act"]).to(TYPES[case["out"]])
    tokens, top_k = case["tokens"], case["top_k"]
    order = state["order"].long()
    if op == "up":
        token = order // top_k
        return _experts(state, a[token], scales[token], tokens * top_k, case["act"]).to(TYPES[case["type"]])
    out = _experts(state, a, scales, tokens * top_k, "none")
    pairs = torch.empty_like(out)
    pairs[order] = out
    y = (pairs.reshape(tokens, top_k, -1) * state["gates"].unsqueeze(-1)).sum(1)
    return y.to(TYPES[case["type"]])


# ---------------------------------------------------------------- work and results


def _bytes(kind):
    return 4 if kind == "f32" else 2


def _operand_bytes(rows, k):
    return rows * (_padded(k) + 4)


def work(case):
    """Each input read once and each output written once; two operations per multiply-add. The experts' products read
    the experts that the tokens choose, on average of even choices."""
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": 2 * n * _bytes(case["type"]) + _operand_bytes(case["rows"], case["k"]), "flops": 0}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        rows = 2 * n if case["act"] == "swiglu" else n
        out = m * n * _bytes(case["out"]) + (4 * rows if case["bias"] else 0)
        return {"bytes": _operand_bytes(m, k) + _operand_bytes(rows, k) + out, "flops": 2 * m * rows * k}
    t, e, top = case["tokens"], case["experts"], case["top_k"]
    if op == "route":
        return {"bytes": t * e * _bytes(case["type"]) + 12 * t * top + 4 * e, "flops": 0}
    d, h = case["d"], case["h"]
    read = e * (1.0 - (1.0 - top / e) ** t)
    if op == "up":
        rows, k = (2 * h if case["act"] == "swiglu" else h), d
        moved = _operand_bytes(t, d) + t * top * h * _bytes(case["type"])
    else:
        rows, k = d, h
        moved = _operand_bytes(t * top, h) + t * d * _bytes(case["type"]) + 4 * t * top
    one = _operand_bytes(rows, k) + (4 * rows if case["bias"] else 0)
    return {"bytes": int(moved + 4 * t * top + read * one), "flops": 2 * t * top * rows * k}


def _exact_operand(operand, k):
    """An operand's values in float64."""
    codes, scales = operand
    return codes[..., :k].double() * scales.double()[..., None]


def _exact_quantize(x):
    """The nearest multiple of the scale by its distance, in float64, some rows at a time."""
    out = torch.empty(x.shape, dtype=torch.float64, device=DEVICE)
    scales = torch.empty(len(x), dtype=torch.float64, device=DEVICE)
    for at in range(0, len(x), 1024):
        b = x[at:at + 1024].double()
        scale = (torch.maximum(b.amax(-1), -b.amin(-1)) / 127.0).float().double()
        below = torch.floor(b / scale[:, None])
        to_below, to_above = b - below * scale[:, None], (below + 1) * scale[:, None] - b
        up = (to_above < to_below) | ((to_above == to_below) & (below % 2 != 0))
        out[at:at + 1024] = (below + up) * scale[:, None]
        scales[at:at + 1024] = scale
    return out, scales


def _exact_act(u, act):
    if act == "relu":
        return u.clamp(min=0.0)
    if act == "gelu":
        return u / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (u + 0.044715 * u ** 3)))
    if act == "swiglu":
        gate, up = u[:, :u.shape[1] // 2], u[:, u.shape[1] // 2:]
        return gate / (1.0 + torch.exp(-gate)) * up
    return u


def _exact_route(case, t):
    """By taking the largest key again and again."""
    l = t["logits"].double()
    tokens, experts = l.shape
    rows = torch.arange(tokens, device=DEVICE)
    if case["score"] == "softmax":
        e = torch.exp(l - l.max(-1, keepdim=True)[0])
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-l))
    plain = t["bias"] is None and not (case["group_best"] > 1 and case["groups"] > 1)
    key = l.clone() if plain else score if t["bias"] is None else score + t["bias"].double()

    def take(keys):
        """The first place of each row's largest, which is then out."""
        places = torch.arange(keys.shape[1], device=DEVICE)
        at = torch.where(keys == keys.max(-1, keepdim=True)[0], places, keys.shape[1]).min(-1)[0]
        value = keys[rows, at].clone()
        keys[rows, at] = -math.inf
        return at, value

    groups = case["groups"]
    if groups > 1:
        each = experts // groups
        sums = torch.stack([sum(take(part)[1] for _ in range(case["group_best"]))
                            for part in (key[:, g * each:(g + 1) * each].clone() for g in range(groups))], -1)
        kept = torch.zeros(tokens, groups, dtype=torch.bool, device=DEVICE)
        for _ in range(case["top_groups"]):
            kept[rows, take(sums)[0]] = True
        key = torch.where(kept.repeat_interleave(each, 1), key, -math.inf)
    else:
        key = key.clone()
    chosen = torch.stack([take(key)[0] for _ in range(case["top_k"])], -1)
    gates = torch.stack([score[rows, chosen[:, j]] for j in range(case["top_k"])], -1)
    if case["normalize"]:
        gates = gates / gates.sum(-1, keepdim=True)
    expert = chosen.reshape(-1)
    order = torch.argsort(expert * expert.numel() + torch.arange(expert.numel(), device=DEVICE))
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=DEVICE),
                         torch.bincount(expert, minlength=experts).cumsum(0)])
    return {"chosen": chosen.int(), "gates": gates * case["scale"], "order": order.int(), "offsets": offsets.int()}


def _exact_experts(case, t):
    order, offsets = t["order"].long(), t["offsets"].tolist()
    top_k, tokens = case["top_k"], case["tokens"]
    up = case["op"] == "up"
    k = case["d"] if up else case["h"]
    a = _exact_operand(t["a"], k)
    out = torch.zeros(tokens * top_k if up else tokens, case["h"] if up else case["d"], dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        at = slice(offsets[e], offsets[e + 1])
        pair = order[at]
        if not len(pair):
            continue
        w = _exact_operand((t["w"][0][e], t["w"][1][e]), k)
        u = torch.mm(a[pair // top_k] if up else a[at], w.t())
        if t["b"] is not None:
            u = u + t["b"][e].double()
        if up:
            out[at] = _exact_act(u, case["act"])
        else:
            out.index_add_(0, pair // top_k, u * t["gates"].reshape(-1)[pair].double()[:, None])
    return out


def exact(case, seed):
    t = _inputs(case, seed)
    op = case["op"]
    if op == "quantize":
        values, scales = _exact_quantize(t["x"] if case["form"] == "rows" else t["x"].t())
        return {"values": values if case["form"] == "rows" else values.t().contiguous(), "scales": scales}
    if op == "route":
        return _exact_route(case, t)
    if op != "product":
        return _exact_experts(case, t)
    u = torch.matmul(_exact_operand(t["a"], case["k"]), _exact_operand(t["b"], case["k"]).t())
    if t["bias"] is not None:
        u = u + t["bias"].double()
    return _exact_act(u, case["act"])
