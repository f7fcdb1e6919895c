"""Cases of the 4-bit weights with group scales and of the mixture-of-experts routing: what is timed, on which inputs.

Every case is a call that a user of the package makes:

  quantize  ``Q4Tensor.from_float`` and ``dequantize``: a checkpoint's weight to 4-bit codes with a scale per group of columns
  linear    ``nn.Q4Linear`` forward: one token through a layer up to a prompt (language-model heads, layers that ternary weights lose)
  experts   ``Q4Tensor.matmul_sorted``: rows sorted by expert times the 4-bit weights of the expert each belongs to
  dispatch  ``route`` and ``Routing.gather``: a serving step sorts its (token, slot) pairs by expert and gathers their rows
  train     the same in training: dispatch, the experts' results combined with the router's weights, and all gradients

``listed()`` names the sizes followed over time, ``draw()`` gives others of the same ranges.  Hidden 4096, FFN 14336 and 1024 key/value
features are the benchmark's layer shapes; heads and expert counts are generic ones.  Weights are N(0, 0.02^2), activations
N(0, 1); routers prefer some experts, as trained ones do, and a padded batch has slots that go to no expert.

The format: columns in groups of 32, 64 or 128 (the last group of a row may be shorter).  A group's scale s is its value of largest
magnitude (the first of equals) over -8, rounded to five significant bits; a weight's code is the whole number nearest to
w / s (ties to even), held in -8 .. 7, and stands for code * s, which is a bfloat16 number.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}

# what the largest listed cases cost; drawn ones stay below
_MOST_LINEAR = 2.0 * 2048 * 4096 * 14336
_MOST_WEIGHTS = 14336 * 4096
_MOST_EXPERTS = 32 * 4096 * 2048
_MOST_ROWS = 4096 * 8 * 4096


def listed():
    return [
        # the smallest product: one token through a key projection, where launch and host latency count
        {"name": "linear_1024x4096_1tok", "kind": "linear", "tokens": 1, "in": 4096, "out": 1024, "group": 128, "dtype": "bfloat16", "bias": False},
        # a language-model head at batch 8, streamed from HBM
        {"name": "linear_65536x4096_8tok_g32", "kind": "linear", "tokens": 8, "in": 4096, "out": 65536, "group": 32, "dtype": "bfloat16", "bias": False},
        # a large batch or a speculated continuation, in fp16
        {"name": "linear_4096x14336_64tok_fp16", "kind": "linear", "tokens": 64, "in": 14336, "out": 4096, "group": 64, "dtype": "float16", "bias": False},
        # the largest: a 2048-token prompt through an up projection
        {"name": "linear_14336x4096_2048tok", "kind": "linear", "tokens": 2048, "in": 4096, "out": 14336, "group": 128, "dtype": "bfloat16", "bias": True},
        # a model that was not cast down, nothing a multiple of anything
        {"name": "linear_1999x3001_77tok_fp32", "kind": "linear", "tokens": 77, "in": 3001, "out": 1999, "group": 32, "dtype": "float32", "bias": True},
        # converting a checkpoint: one bf16 weight, and an odd one in fp32
        {"name": "quantize_14336x4096_g128_bf16", "kind": "quantize", "rows": 14336, "cols": 4096, "group": 128, "dtype": "bfloat16"},
        {"name": "quantize_2047x1999_g32_fp32", "kind": "quantize", "rows": 2047, "cols": 1999, "group": 32, "dtype": "float32"},
        # a decode step of eight tokens, six of 64 experts each: most experts get one row or none
        {"name": "experts_64x2816x2048_8tok_top6", "kind": "experts", "tokens": 8, "top": 6, "experts": 64, "in": 2048, "out": 2816, "group": 128, "dtype": "bfloat16", "padded": False},
        # a prompt through larger experts: some 250 rows each
        {"name": "experts_32x2048x4096_2048tok_top4", "kind": "experts", "tokens": 2048, "top": 4, "experts": 32, "in": 4096, "out": 2048, "group": 64, "dtype": "bfloat16", "padded": True},
        # routing of a decode step
        {"name": "dispatch_16tok_top6_of_64", "kind": "dispatch", "tokens": 16, "top": 6, "experts": 64, "hidden": 2048, "dtype": "bfloat16", "padded": False},
        # a training batch
        {"name": "train_4096tok_top8_of_64", "kind": "train", "tokens": 4096, "top": 8, "experts": 64, "hidden": 4096, "dtype": "bfloat16", "padded": False},
        # a small ragged one in fp32, with padding that goes to no expert
        {"name": "train_777tok_top2_of_8_fp32", "kind": "train", "tokens": 777, "top": 2, "experts": 8, "hidden": 1537, "dtype": "float32", "padded": True},
    ]


def _between(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: as it comes (odd ones among them) or, as often, a round one."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice((1, 1, 16, 128))
    return max(lo, min(hi, (n + step - 1) // step * step))


def draw(rng):
    kind = rng.choice(("linear", "linear", "linear", "quantize", "experts", "experts", "dispatch", "train"))
    dtype, group = rng.choice(("bfloat16", "bfloat16", "float16", "float32")), rng.choice((32, 64, 128))
    if kind == "linear":
        fan_in, fan_out = _between(rng, 512, 14336), _between(rng, 512, 32768)
        fan_out = max(1, min(fan_out, 65536 * 4096 // fan_in))
        tokens = max(1, min(_between(rng, 1, 2048), int(_MOST_LINEAR / (2.0 * fan_in * fan_out) / (1 if _SIZE[dtype] == 2 else 8))))
        return {"kind": kind, "tokens": tokens, "in": fan_in, "out": fan_out, "group": group, "dtype": dtype, "bias": rng.random() < 0.5}
    if kind == "quantize":
        rows, cols = _between(rng, 512, 14336), _between(rng, 512, 14336)
        return {"kind": kind, "rows": max(1, min(rows, _MOST_WEIGHTS // cols)), "cols": cols, "group": group, "dtype": dtype}
    experts = rng.choice((8, 16, 32, 60, 64))
    top, padded = rng.randint(1, min(8, experts)), rng.random() < 0.5
    if kind == "experts":
        fan_in, fan_out = _between(rng, 512, 4096), _between(rng, 512, 4096)
        fan_out = max(1, min(fan_out, _MOST_EXPERTS // (experts * fan_in)))
        tokens = max(1, min(_between(rng, 1, 2048), int(2048 * 4 * 4096 * 2048.0 / (top * fan_in * fan_out) / (1 if _SIZE[dtype] == 2 else 8))))
        return {"kind": kind, "tokens": tokens, "top": top, "experts": experts, "in": fan_in, "out": fan_out, "group": group, "dtype": dtype, "padded": padded}
    hidden = _between(rng, 512, 4096)
    tokens = max(1, min(_between(rng, 1, 4096), _MOST_ROWS // (top * hidden) // (1 if _SIZE[dtype] == 2 else 2)))
    return {"kind": kind, "tokens": tokens, "top": top, "experts": experts, "hidden": hidden, "dtype": dtype, "padded": padded}


def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _routed(gen, case):
    """Expert ids (tokens, top) as a router's top-k gives them, -1 in the slots of padding, and the router's weights."""
    tokens, top, experts = case["tokens"], case["top"], case["experts"]
    logits = _normal(gen, tokens, experts) + _normal(gen, experts)
    values, ids = torch.topk(logits, top, dim=1)
    if case["padded"]:
        ids[tokens - tokens // 8:] = -1
        ids[torch.rand(tokens, top, generator=gen, device="cuda") < 0.01] = -1  # beyond an expert's capacity
    return ids, torch.softmax(values, dim=1)


def _inputs(case, seed):
    """The raw inputs of a case, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    if kind == "quantize":
        return {"w": _normal(gen, case["rows"], case["cols"], std=0.02, dtype=dtype)}
    if kind == "linear":
        return {"w": _normal(gen, case["out"], case["in"], std=0.02, dtype=torch.bfloat16), "x": _normal(gen, case["tokens"], case["in"], dtype=dtype),
                "bias": _normal(gen, case["out"], std=0.01) if case["bias"] else None}
    ids, weights = _routed(gen, case)
    if kind == "experts":
        # bf16 checkpoints; the rows are what gathering gives: those of slots that go to no expert lie behind the last one, zero
        rows = _normal(gen, case["tokens"] * case["top"], case["in"], dtype=dtype)
        valid = ids[ids >= 0]
        rows[valid.numel():] = 0
        offsets = torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = torch.cumsum(torch.bincount(valid, minlength=case["experts"]), 0)
        return {"w": _normal(gen, case["experts"], case["out"], case["in"], std=0.02, dtype=torch.bfloat16), "rows": rows, "offsets": offsets}
    x = _normal(gen, case["tokens"], case["hidden"], dtype=dtype)
    if kind == "dispatch":
        return {"ids": ids, "x": x}
    n = case["tokens"] * case["top"]
    return {"ids": ids, "weights": weights, "x": x, "results": _normal(gen, n, case["hidden"], dtype=dtype), "grad_rows": _normal(gen, n, case["hidden"], std=0.05, dtype=dtype),
            "grad_y": _normal(gen, case["tokens"], case["hidden"], std=0.05, dtype=dtype)}


# ---- the plain forms ----


def _quantize(w, group):
    """(codes int8 (..., rows, groups, group), scales (..., rows, groups)); columns past the last count as zero."""
    cols = w.shape[-1]
    v = torch.nn.functional.pad(w.float(), (0, -cols % group)).unflatten(-1, (-1, group))
    a = v.abs()
    largest = a.amax(-1, keepdim=True)
    at = torch.where(a == largest, torch.arange(group, device=w.device), group).amin(-1, keepdim=True)
    mantissa, exponent = torch.frexp(v.gather(-1, at) * -0.125)
    s = torch.ldexp(torch.round(mantissa * 32.0) / 32.0, exponent)
    ratio = v.double() / torch.where(s == 0, 1.0, s).double()  # 64 bits: the border between two codes is met exactly
    return ratio.round().clamp(-8, 7).to(torch.int8), s.squeeze(-1)


def _values(codes, scales, cols):
    return (codes.float() * scales.unsqueeze(-1)).flatten(-2)[..., :cols]


def _sorted(ids, experts):
    """(order, position, offsets) of a stable sort of the flattened ids; ids outside [0, experts) take no part."""
    flat = ids.flatten()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    sorted_ids, order = torch.sort(key, stable=True)
    place = torch.arange(flat.numel(), device=flat.device, dtype=torch.int32)
    order = torch.where(sorted_ids < experts, order, -1).to(torch.int32)
    position = torch.full_like(place, -1)
    position[order[order >= 0].long()] = place[order >= 0]
    offsets = torch.searchsorted(sorted_ids, torch.arange(experts + 1, device=flat.device)).to(torch.int32)
    return order, position.view(ids.shape), offsets


def _gather(x, order, top):
    return torch.where((order >= 0)[:, None], x[torch.clamp(order, min=0).long() // top], torch.zeros((), dtype=x.dtype, device=x.device))


def _train(state):
    case, x, results, weights = state["case"], state["x"].detach(), state["results"].detach(), state["weights"].detach()
    top = case["top"]
    order, position, _ = _sorted(state["ids"], case["experts"])
    rows = _gather(x, order, top)
    kept, at = position >= 0, torch.clamp(position, min=0).long()
    w = torch.where(kept, weights.float(), 0.0)
    slots = torch.where(kept[..., None], results[at].float(), 0.0)
    gy = state["grad_y"].float()
    y = (slots * w[..., None]).sum(1)
    grad_w = (slots * gy[:, None, :]).sum(-1)
    source = torch.clamp(order, min=0).long()
    grad_results = torch.where((order >= 0)[:, None], gy[source // top] * weights.flatten()[source][:, None].float(), 0.0)
    grad_x = torch.where(kept[..., None], state["grad_rows"][at].float(), 0.0).sum(1)
    return [rows, y.to(x.dtype), grad_x.to(x.dtype), grad_results.to(x.dtype), grad_w.to(weights.dtype)]


def _plain(state):
    kind, case = state["kind"], state["case"]
    if kind == "quantize":
        codes, scales = _quantize(state["w"], case["group"])
        return [_values(codes, scales, case["cols"]), scales.to(torch.bfloat16)]
    if kind == "linear":
        y = state["x"].float() @ _values(state["codes"], state["scales"], case["in"]).t()
        if state["bias"] is not None:
            y = y + state["bias"]
        return y.to(state["x"].dtype)
    if kind == "experts":
        rows, ends = state["rows"], state["offsets"].tolist()
        y = torch.zeros(rows.shape[0], case["out"], dtype=rows.dtype, device=rows.device)
        for e in range(case["experts"]):
            if ends[e + 1] > ends[e]:
                w = _values(state["codes"][e], state["scales"][e], case["in"])
                y[ends[e]:ends[e + 1]] = (rows[ends[e]:ends[e + 1]].float() @ w.t()).to(rows.dtype)
        return y
    if kind == "dispatch":
        order, position, offsets = _sorted(state["ids"], case["experts"])
        return [order, position, offsets, _gather(state["x"], order, case["top"])]
    return _train(state)


# ---- what the tools call ----


def prepare(case, seed):
    state = {"kind": case["kind"], "case": case, **_inputs(case, seed)}
    kind = case["kind"]
    if kind == "train":
        for name in ("x", "results", "weights"):
            state[name].requires_grad_(True)
    if kind in ("linear", "experts"):
        w = state.pop("w")
        if own:
            from t81lib_b200 import torch as t81_torch
            from t81lib_b200.nn import Q4Linear
            q = t81_torch.Q4Tensor.from_float(w, group=case["group"])
            if kind == "linear":
                state["layer"] = Q4Linear.from_quantized(q, bias=state["bias"]).eval().requires_grad_(False)
            else:
                state["q"] = q
        else:
            state["codes"], state["scales"] = _quantize(w, case["group"])
    return state


def run(state):
    if not own:
        return _plain(state)
    from t81lib_b200 import torch as t81_torch
    kind, case = state["kind"], state["case"]
    if kind == "quantize":
        q = t81_torch.Q4Tensor.from_float(state["w"], group=case["group"])
        return [q.dequantize(), q.group_scales()]
    if kind == "linear":
        return state["layer"](state["x"])
    if kind == "experts":
        return state["q"].matmul_sorted(state["rows"], state["offsets"])
    routing = t81_torch.route(state["ids"], case["experts"])
    rows = routing.gather(state["x"])
    if kind == "dispatch":
        return [routing.order, routing.position, routing.offsets, rows]
    y = routing.combine(state["results"], state["weights"])
    grads = torch.autograd.grad([rows, y], [state["x"], state["results"], state["weights"]], [state["grad_rows"], state["grad_y"]])
    return [rows.detach(), y.detach(), *grads]


def work(case):
    kind, size = case["kind"], _SIZE[case["dtype"]]
    if kind == "quantize":
        # the weight in, its values and scales out (the codes between them are half a byte each, written and read)
        rows, cols = case["rows"], case["cols"]
        return {"bytes": rows * cols * (size + 4.0 + 1.0) + 2.0 * rows * math.ceil(cols / case["group"]) * 2, "flops": 0.0}
    if kind == "linear":
        t, i, o = case["tokens"], case["in"], case["out"]
        return {"bytes": o * (i / 2.0 + 2.0 * math.ceil(i / case["group"])) + size * t * (i + o) + (4.0 * o if case["bias"] else 0.0), "flops": 2.0 * t * i * o}
    n = case["tokens"] * case["top"]
    if kind == "experts":
        i, o = case["in"], case["out"]
        used = case["experts"] * (1.0 - (1.0 - case["top"] / case["experts"]) ** case["tokens"])  # experts that get a row, of a router without preferences
        return {"bytes": used * o * (i / 2.0 + 2.0 * math.ceil(i / case["group"])) + size * n * (i + o), "flops": 2.0 * n * i * o}
    h = case["hidden"]
    if kind == "dispatch":
        return {"bytes": 8.0 * n + 8.0 * n + 4.0 * (case["experts"] + 1) + size * h * (case["tokens"] + n), "flops": 0.0}
    # rows out; results in, y out; the gradients of rows, y in, those of x, results, weights out
    return {"bytes": 16.0 * n + 8.0 * n + size * h * (2.0 * case["tokens"] + 4.0 * n + 2.0 * case["tokens"]), "flops": 8.0 * n * h}


# ---- from the definitions, in 64 bits ----


def _exact_weight(w, group):
    """(values, scales) of the last two axes (rows, cols), group by group of columns."""
    w = w.double()
    values, scales = torch.empty_like(w), []
    for lo in range(0, w.shape[-1], group):
        part = w[..., lo:lo + group]
        high, low = part.amax(-1), -part.amin(-1)
        first_high = (part == high[..., None]).to(torch.uint8).argmax(-1)
        first_low = (part == -low[..., None]).to(torch.uint8).argmax(-1)
        positive = (high > low) | ((high == low) & (first_high < first_low))
        largest = torch.where(positive, high, -low)
        step = torch.exp2(torch.floor(torch.log2(torch.where(largest == 0, 1.0, largest).abs() / 8)) - 4)
        s = torch.where(largest == 0, 0.0, torch.round(-largest / 8 / step) * step)
        codes = torch.clamp(torch.round(part / torch.where(s == 0, 1.0, s)[..., None]), -8, 7)
        values[..., lo:lo + group] = codes * s[..., None]
        scales.append(s)
    return values, torch.stack(scales, -1)


def exact(case, seed):
    kind, given = case["kind"], _inputs(case, seed)
    if kind == "quantize":
        return list(_exact_weight(given["w"], case["group"]))
    if kind == "linear":
        y = given["x"].double() @ _exact_weight(given["w"], case["group"])[0].t()
        return y if given["bias"] is None else y + given["bias"].double()
    if kind == "experts":
        ends, rows = given["offsets"].cpu().numpy(), given["rows"].double()
        y = torch.zeros(rows.shape[0], case["out"], dtype=torch.float64, device=rows.device)
        for e in np.flatnonzero(np.diff(ends)):
            torch.matmul(rows[ends[e]:ends[e + 1]], _exact_weight(given["w"][e], case["group"])[0].t(), out=y[ends[e]:ends[e + 1]])
        return y
    ids, top = given["ids"].cpu().numpy().reshape(-1), case["top"]
    flats = np.concatenate([np.flatnonzero(ids == e) for e in range(case["experts"])])
    order = np.full(ids.size, -1, np.int32)
    order[:flats.size] = flats
    position = np.full(ids.size, -1, np.int32)
    position[flats] = np.arange(flats.size)
    x = given["x"].double()
    rows = torch.zeros(ids.size, case["hidden"], dtype=torch.float64, device=x.device)
    at = torch.from_numpy(flats).to(x.device)
    rows[:flats.size] = x[at // top]
    if kind == "dispatch":
        offsets = np.array([np.count_nonzero((ids >= 0) & (ids < e)) for e in range(case["experts"] + 1)], np.int32)
        return [torch.from_numpy(order), torch.from_numpy(position.reshape(-1, top)), torch.from_numpy(offsets), rows]
    weights, results, gy = given["weights"].double().flatten(), given["results"].double()[:flats.size], given["grad_y"].double()
    y, grad_x = torch.zeros_like(x), torch.zeros_like(x)
    y.index_add_(0, at // top, results * weights[at, None])
    grad_x.index_add_(0, at // top, given["grad_rows"].double()[:flats.size])
    grad_results, grad_weights = torch.zeros_like(rows), torch.zeros_like(weights)
    grad_results[:flats.size] = gy[at // top] * weights[at, None]
    grad_weights[at] = (results * gy[at // top]).sum(1)
    return [rows, y, grad_x, grad_results, grad_weights.view(-1, top)]
