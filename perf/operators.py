"""The operators of a mixture-of-experts layer in MXFP4, one pass each.

An operator is a call that a training or serving program makes on tensors it
holds: MX quantisation (and back), a linear layer whose weight is MXFP4 (dense,
with its gradients, or one weight per expert), routing, the sort of routed
tokens by expert, and the weighted sum of the experts' outputs. `run` computes
it in elementary torch operations in 32 bits, or through the package's entry
points. `listed` names the cases compared from change to change; `draw` spreads
more over the same ranges.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32           # elements that share one E8M0 scale
STEP = 256           # elements along K whose scales a row holds together
MOST_ELEMENTS = 8192 * 8192    # of a quantised tensor, a combined one or a dense weight
MOST_FLOPS = 2 * 8192 * 4096 * 4096 * 4
MOST_WEIGHTS = 1 << 30         # elements over all experts

# Route options as routers have them: softmax over all experts, or sigmoid scores with a balancing bias and groups.
SOFTMAX = {"scores": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renormalize": True, "scale": 1.0}
SIGMOID = {"scores": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5}


def listed():
    return [
        # Activations whose rows and groups fit no tile, to MXFP4 and back (a quantised layer's view of its input).
        {"name": "quantize_bf16_5000x4112", "op": "quantize", "dtype": "bf16", "rows": 5000, "k": 4112,
         "columns": False},
        # The operand of a weight gradient: groups along the tokens, transposed.
        {"name": "quantize_columns_bf16_8192x8192", "op": "quantize", "dtype": "bf16", "rows": 8192, "k": 8192,
         "columns": True},
        # One token through a layer: the weight's bytes are all there is.
        {"name": "linear_bf16_1x8192x8192", "op": "linear", "dtype": "bf16", "rows": 1, "n": 8192, "k": 8192,
         "backward": False},
        # A training step of a layer of sizes off every tile: both operands quantised, output and both gradients.
        {"name": "linear_train_bf16_5000x3000x4112", "op": "linear", "dtype": "bf16", "rows": 5000, "n": 3000,
         "k": 4112, "backward": True},
        # Decoding a batch: few rows for each of many experts, most weights read once.
        {"name": "experts_bf16_32of8x128", "op": "experts", "dtype": "bf16", "tokens": 32, "top": 8, "experts": 128,
         "n": 2048, "k": 4096},
        # Prompts: hundreds of rows an expert, unevenly.
        {"name": "experts_bf16_8192of4x32", "op": "experts", "dtype": "bf16", "tokens": 8192, "top": 4, "experts": 32,
         "n": 4096, "k": 4096},
        # Decoding: a few tokens' scores over grouped experts with the balancing bias; all latency.
        {"name": "route_sigmoid_16x256", "op": "route", "dtype": "fp32", "tokens": 16, "experts": 256, "top": 8,
         **SIGMOID, "masked": False, "backward": False},
        # Training: scores and their gradient for a batch of sequences.
        {"name": "route_softmax_train_16384x128", "op": "route", "dtype": "fp32", "tokens": 16384, "experts": 128,
         "top": 8, **SOFTMAX, "masked": False, "backward": True},
        # The same two batches' sorts.
        {"name": "dispatch_32of8x128", "op": "dispatch", "tokens": 32, "top": 8, "experts": 128, "masked": False},
        {"name": "dispatch_16384of8x256", "op": "dispatch", "tokens": 16384, "top": 8, "experts": 256,
         "masked": False},
        # Outputs of a decoded batch's experts, and of a training batch's with both gradients.
        {"name": "combine_bf16_32of8x4096", "op": "combine", "dtype": "bf16", "tokens": 32, "top": 8, "n": 4096,
         "masked": False, "backward": False},
        {"name": "combine_train_bf16_8192of4x4096", "op": "combine", "dtype": "bf16", "tokens": 8192, "top": 4,
         "n": 4096, "masked": False, "backward": True},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "experts", "experts", "route", "dispatch", "combine"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        if op == "quantize":
            case = {"op": op, "dtype": dtype, "rows": _log_uniform(rng, 1, 16384), "k": _log_uniform(rng, 32, 16384),
                    "columns": rng.random() < 0.5}
            if case["rows"] * case["k"] <= MOST_ELEMENTS:
                return case
        elif op == "linear":
            case = {"op": op, "dtype": dtype, "rows": _log_uniform(rng, 1, 8192), "n": _log_uniform(rng, 64, 8192),
                    "k": _log_uniform(rng, 64, 8192), "backward": rng.random() < 0.4}
            if 2 * case["rows"] * case["n"] * case["k"] * (3 if case["backward"] else 1) <= MOST_FLOPS // 2:
                return case
        elif op == "experts":
            experts = rng.choice([8, 16, 32, 60, 64, 128, 256])
            case = {"op": op, "dtype": dtype, "tokens": _log_uniform(rng, 1, 8192), "top": rng.choice([1, 2, 4, 6, 8]),
                    "experts": experts, "n": _log_uniform(rng, 256, 4096), "k": _log_uniform(rng, 256, 4096)}
            if (experts * case["n"] * case["k"] <= MOST_WEIGHTS
                    and 2 * case["tokens"] * case["top"] * case["n"] * case["k"] <= MOST_FLOPS):
                return case
        elif op == "route":
            kind = rng.choice([SOFTMAX, {**SOFTMAX, "renormalize": False}, SIGMOID,
                               {**SIGMOID, "groups": 1, "top_groups": 1}])
            experts = 8 * rng.randint(2, 32) if kind["groups"] > 1 else rng.randint(8, 256)
            return {"op": op, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    "tokens": _log_uniform(rng, 1, 16384), "experts": experts, "top": rng.randint(1, 8), **kind,
                    "masked": rng.random() < 0.3, "backward": rng.random() < 0.4}
        elif op == "dispatch":
            return {"op": op, "tokens": _log_uniform(rng, 1, 16384), "top": rng.choice([1, 2, 4, 6, 8]),
                    "experts": rng.randint(8, 512), "masked": rng.random() < 0.3}
        else:
            case = {"op": op, "dtype": dtype, "tokens": _log_uniform(rng, 1, 8192), "top": rng.choice([1, 2, 4, 6, 8]),
                    "n": _log_uniform(rng, 64, 8192), "masked": rng.random() < 0.3, "backward": rng.random() < 0.4}
            if case["tokens"] * case["top"] * case["n"] * DTYPES[dtype].itemsize <= 2 * 8192 * 4 * 4096:
                return case


# ---- inputs --------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(generator, *shape):
    return torch.randn(shape, device=DEVICE, generator=generator)


def _activations(generator, rows, k, dtype):
    """N(0, 1) with a few channels an order of magnitude larger, as layers' inputs have."""
    channel = torch.where(torch.rand(k, device=DEVICE, generator=generator) < 0.01, 20.0, 1.0)
    return (_randn(generator, rows, k) * channel).to(DTYPES[dtype])


def _assignment(generator, tokens, top, experts):
    """Each token's `top` different experts, some experts several times as popular as others."""
    popularity = _randn(generator, experts)
    noise = -torch.log(-torch.log(torch.rand((tokens, experts), device=DEVICE, generator=generator).clamp(1e-9, 1 - 1e-7)))
    return torch.argsort(popularity + noise, dim=1, descending=True)[:, :top].to(torch.int32).contiguous()


def _mask_rows(assignment):
    """Every seventh row, from the fourth on, has no expert: padding of a batch."""
    assignment[3::7] = -1
    return assignment


def _sorted(assignment, experts):
    """(offsets, order, slots) of an assignment [tokens][top]: its entries by expert, in their order; -1 left out."""
    flat = assignment.reshape(-1).long()
    order = torch.argsort(torch.where(flat < 0, experts, flat), stable=True)
    counts = (flat[:, None] == torch.arange(experts, device=DEVICE)).sum(dim=0)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=DEVICE)
    offsets[1:] = torch.cumsum(counts, 0)
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(flat.numel(), device=DEVICE)
    slots = torch.where(flat < 0, -1, slots)
    order = torch.where(torch.arange(flat.numel(), device=DEVICE) < offsets[-1], order, -1)
    return offsets.to(torch.int32), order.to(torch.int32), slots.view(assignment.shape).to(torch.int32)


def _route_inputs(case, seed):
    """Logits ~ 1.5 N(0, 1) and a bias of steps of 0.001, as a balancing rule leaves it.

    Rows in which two candidates lie closer than scores in 32 bits tell apart, equal ones aside, are drawn again:
    their order is not the formula's but the rounding's.
    """
    generator = _generator(seed)
    tokens, experts = case["tokens"], case["experts"]
    bias = torch.randint(-100, 101, (experts,), device=DEVICE, generator=generator).float() * 0.001
    bias = bias if case["bias"] else None
    offline = torch.rand(experts, device=DEVICE, generator=generator) < 0.06
    logits = torch.empty((tokens, experts), device=DEVICE, dtype=DTYPES[case["dtype"]])
    close = torch.ones(tokens, dtype=torch.bool, device=DEVICE)
    for _ in range(6):
        drawn = (1.5 * _randn(generator, tokens, experts)).to(logits.dtype)
        if case["masked"]:
            drawn[:, offline] = -math.inf
            drawn[3::7] = -math.inf
        logits = torch.where(close[:, None], drawn, logits)
        close = _close_candidates(case, logits.double(), bias)
    d_weights = _randn(generator, tokens, case["top"])
    return logits, bias, d_weights


def _close_candidates(case, logits, bias):
    scores = _exact_scores(case, logits)
    value = scores if bias is None else scores + bias.double()
    size = scores if bias is None else scores + bias.double().abs()
    value = torch.where(torch.isinf(logits), -math.inf, value)
    close = torch.zeros(logits.shape[0], dtype=torch.bool, device=DEVICE)
    if case["groups"] > 1:
        ranked = torch.sort(_group_scores(case, value), dim=1, descending=True).values
        gap = ranked[:, case["top_groups"] - 1] - ranked[:, case["top_groups"]]
        close |= (gap != 0) & (gap < 1e-5)
        value = torch.where(_kept_groups(case, value), value, -math.inf)
    ranked, index = torch.sort(value, dim=1, descending=True)
    size = size.gather(1, index)
    last = min(case["top"], case["experts"] - 1)
    gap = ranked[:, :last] - ranked[:, 1:last + 1]
    return close | ((gap != 0) & (gap < 4e-6 * size[:, :last])).any(dim=1)


def _linear_inputs(case, seed):
    generator = _generator(seed)
    x = _activations(generator, case["rows"], case["k"], case["dtype"])
    weight = _randn(generator, case["n"], case["k"]) / math.sqrt(case["k"])
    if not case["backward"]:
        return x, _pack(weight), None
    d_out = (1e-3 * _randn(generator, case["rows"], case["n"])).to(DTYPES[case["dtype"]])
    return x, weight.to(DTYPES[case["dtype"]]), d_out


def _experts_inputs(case, seed):
    generator = _generator(seed)
    x = _activations(generator, case["tokens"], case["k"], case["dtype"])
    assignment = _assignment(generator, case["tokens"], case["top"], case["experts"])
    weights = [_pack(_randn(generator, case["n"], case["k"]) / math.sqrt(case["k"])) for _ in range(case["experts"])]
    return x, assignment, tuple(torch.stack(parts) for parts in zip(*weights))


def _combine_inputs(case, seed):
    generator = _generator(seed)
    tokens, top, n, dtype = case["tokens"], case["top"], case["n"], DTYPES[case["dtype"]]
    assignment = _assignment(generator, tokens, top, 8 * top)
    if case["masked"]:
        _mask_rows(assignment)
    slots = _sorted(assignment, 8 * top)[2]
    weights = torch.softmax(_randn(generator, tokens, top), dim=1)
    weights = torch.where(slots < 0, 0.0, weights)
    y = _randn(generator, tokens * top, n).to(dtype)
    return y, slots, weights, (1e-3 * _randn(generator, tokens, n)).to(dtype)


def prepare(case, seed):
    op = case["op"]
    state = {"case": case}
    if op == "quantize":
        state["x"] = _activations(_generator(seed), case["rows"], case["k"], case["dtype"])
    elif op == "linear":
        state["x"], state["weight"], state["d_out"] = _linear_inputs(case, seed)
    elif op == "experts":
        state["x"], assignment, state["weight"] = _experts_inputs(case, seed)
        state["plan"] = _sorted(assignment, case["experts"])
        state["host_offsets"] = state["plan"][0].tolist()  # where the plain form splits its rows
    elif op == "route":
        state["logits"], state["bias"], state["d_weights"] = _route_inputs(case, seed)
    elif op == "dispatch":
        state["assignment"] = _assignment(_generator(seed), case["tokens"], case["top"], case["experts"])
        if case["masked"]:
            _mask_rows(state["assignment"])
    else:
        state["y"], state["slots"], state["weights"], state["d_out"] = _combine_inputs(case, seed)
    if own:
        _buffers(state)
    return state


def _buffers(state):
    """Outputs and workspaces, made once as a program makes them."""
    from triton_chip_benchmarks_amd import mx, routing

    case, op = state["case"], state["case"]["op"]
    if op == "quantize":
        rows, k = (case["k"], case["rows"]) if case["columns"] else (case["rows"], case["k"])
        state["packed"] = mx.empty(rows, k, device=DEVICE)
        state["values"] = torch.empty((rows, k), device=DEVICE, dtype=torch.bfloat16)
    elif op == "linear":
        rows, n, k, dtype = case["rows"], case["n"], case["k"], DTYPES[case["dtype"]]
        state["out"] = torch.empty((rows, n), device=DEVICE, dtype=dtype)
        if not case["backward"]:
            state["weight"] = mx.Packed(*state["weight"], k)
            state["workspace"] = mx.linear_workspace(rows, n, k, dtype, device=DEVICE)
        else:
            state["packed"] = mx.empty(n, k, device=DEVICE)
            state["packed_columns"] = mx.empty(k, n, device=DEVICE)
            state["d_x"] = torch.empty((rows, k), device=DEVICE, dtype=dtype)
            state["d_weight"] = torch.empty((n, k), device=DEVICE, dtype=dtype)
            state["workspace"] = mx.linear_backward_workspace(rows, n, k, dtype, device=DEVICE)
    elif op == "experts":
        slots, dtype = case["tokens"] * case["top"], DTYPES[case["dtype"]]
        state["weight"] = mx.Packed(*state["weight"], case["k"])
        state["plan"] = routing.Plan(*state["plan"])
        state["out"] = torch.empty((slots, case["n"]), device=DEVICE, dtype=dtype)
        state["workspace"] = mx.linear_workspace(slots, case["n"], case["k"], dtype, experts=case["experts"],
                                                 device=DEVICE)
    elif op == "route":
        state["experts"] = torch.empty((case["tokens"], case["top"]), device=DEVICE, dtype=torch.int32)
        state["weights"] = torch.empty((case["tokens"], case["top"]), device=DEVICE)
        state["d_logits"] = torch.empty_like(state["logits"])
    elif op == "dispatch":
        state["plan"] = routing.empty_plan(case["tokens"], case["top"], case["experts"], device=DEVICE)
    else:
        state["out"] = torch.empty_like(state["d_out"])
        if case["backward"]:
            state["d_y"] = torch.zeros_like(state["y"])  # rows of no token stay zero
            state["d_weights"] = torch.empty_like(state["weights"])


# ---- one pass ------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from triton_chip_benchmarks_amd import mx, routing

    case, op = state["case"], state["case"]["op"]
    if op == "quantize":
        mx.quantize(state["x"], state["packed"], columns=case["columns"])
        return mx.dequantize(state["packed"], state["values"])
    if op == "linear":
        if not case["backward"]:
            return mx.linear(state["x"], state["weight"], state["out"], workspace=state["workspace"])
        weight = mx.quantize(state["weight"], state["packed"])
        out = mx.linear(state["x"], weight, state["out"], workspace=state["workspace"])
        weight_columns = mx.quantize(state["weight"], state["packed_columns"], columns=True)
        d_x, d_weight = mx.linear_backward(state["d_out"], state["x"], weight_columns, state["d_x"],
                                           state["d_weight"], workspace=state["workspace"])
        return out, d_x, d_weight
    if op == "experts":
        return mx.linear(state["x"], state["weight"], state["out"], plan=state["plan"], workspace=state["workspace"])
    if op == "route":
        options = {"scores": case["scores"], "renormalize": case["renormalize"], "scale": case["scale"]}
        experts, weights = routing.route(state["logits"], case["top"], state["bias"], groups=case["groups"],
                                         top_groups=case["top_groups"], experts=state["experts"],
                                         weights=state["weights"], **options)
        if not case["backward"]:
            return experts, weights
        return experts, weights, routing.route_backward(state["logits"], experts, state["d_weights"],
                                                        d_logits=state["d_logits"], **options)
    if op == "dispatch":
        plan = routing.dispatch(state["assignment"], case["experts"], plan=state["plan"])
        return plan.offsets, plan.order, plan.slots
    out = routing.combine(state["y"], state["slots"], state["weights"], state["out"])
    if not case["backward"]:
        return out
    return (out, *routing.combine_backward(state["d_out"], state["y"], state["slots"], state["weights"],
                                           state["d_y"], state["d_weights"]))


def _run_plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "quantize":
        x = state["x"].float()
        return _rounded(x.t() if case["columns"] else x).to(torch.bfloat16)
    if op == "linear":
        dtype = DTYPES[case["dtype"]]
        x = state["x"].float()
        if not case["backward"]:
            return torch.matmul(_rounded(x), _unpack(*state["weight"], case["k"]).t()).to(dtype)
        weight, d_out = state["weight"].float(), state["d_out"].float()
        out = torch.matmul(_rounded(x), _rounded(weight).t())
        d_x = torch.matmul(_rounded(d_out), _rounded(weight.t()).t())
        d_weight = torch.matmul(_rounded(d_out.t()), _rounded(x.t()).t())
        return out.to(dtype), d_x.to(dtype), d_weight.to(dtype)
    if op == "experts":
        _, order, _ = state["plan"]
        x = _rounded(state["x"].float())
        out = torch.empty((order.numel(), case["n"]), device=DEVICE, dtype=DTYPES[case["dtype"]])
        for e, (first, last) in enumerate(zip(state["host_offsets"], state["host_offsets"][1:])):
            if last > first:
                weight = _unpack(state["weight"][0][e], state["weight"][1][e], case["k"])
                out[first:last] = torch.matmul(x[order[first:last].long() // case["top"]], weight.t()).to(out.dtype)
        return out
    if op == "route":
        logits = state["logits"].float()
        experts, weights = _route(case, logits, state["bias"])
        if not case["backward"]:
            return experts, weights
        return experts, weights, _route_gradient(case, logits, experts, state["d_weights"]).to(state["logits"].dtype)
    if op == "dispatch":
        return _sorted(state["assignment"], case["experts"])
    y, slots, weights = state["y"].float(), state["slots"].long(), state["weights"]
    rows = y[slots.clamp(min=0)]
    out = (rows * torch.where(slots < 0, 0.0, weights)[..., None]).sum(dim=1).to(state["y"].dtype)
    if not case["backward"]:
        return out
    d_out = state["d_out"].float()
    d_weights = torch.where(slots < 0, 0.0, (rows * d_out[:, None]).sum(dim=2))
    d_y = torch.zeros((y.shape[0] + 1, y.shape[1]), device=DEVICE, dtype=state["y"].dtype)  # the last row takes the -1s
    d_y[slots] = (weights[..., None] * d_out[:, None]).to(d_y.dtype)
    return out, d_y[:-1], d_weights


# The plain forms' parts, in 32 bits.


def _groups_of_32(x):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % GROUP)).view(*x.shape[:-1], -1, GROUP)


def _scale_exponents(groups):
    """floor(log2 max|x|) - 2, from -127 to 127; the smallest for a group of zeros."""
    largest = groups.abs().amax(dim=-1)
    exponent = torch.frexp(largest).exponent - 3
    return torch.where(largest == 0, -127, exponent).clamp(-127, 127)


def _rounded(x):
    """x as MXFP4 holds it: E2M1 by groups of 32 along the last axis; NaN where a group is not finite."""
    groups = _groups_of_32(x)
    finite = torch.isfinite(groups).all(dim=-1, keepdim=True)
    groups = torch.where(finite, groups, 0.0)
    exponent = _scale_exponents(groups)[..., None]
    scaled = torch.ldexp(groups, -exponent)
    size = scaled.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6.0)
    value = torch.ldexp(torch.copysign(size, scaled), exponent)
    value = torch.where(finite, value, math.nan)
    return value.reshape(*x.shape[:-1], -1)[..., :x.shape[-1]]


def _pack(x):
    """Codes [rows][ceil(k/32)*16] (two a byte, even k low) and scales [ceil(k/256)][rows][8] of a finite x."""
    groups = _groups_of_32(x)
    exponent = _scale_exponents(groups)
    scaled = torch.ldexp(groups, -exponent[..., None])
    size = scaled.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6.0)
    code = torch.where(size < 2, 2 * size, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.int32)
    code = (code + 8 * torch.signbit(scaled)).reshape(x.shape[0], -1)
    codes = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    blocks = -(-x.shape[1] // STEP)
    scales = torch.full((x.shape[0], blocks * 8), 127, device=DEVICE, dtype=torch.uint8)
    scales[:, :exponent.shape[1]] = (exponent + 127).to(torch.uint8)
    return codes, scales.view(x.shape[0], blocks, 8).permute(1, 0, 2).contiguous()


def _unpack(codes, scales, k):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEVICE)
    table = torch.cat([table, -table])
    values = table[torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1).int()]
    exponent = scales.permute(1, 0, 2).reshape(codes.shape[0], -1)[:, :values.shape[1] // GROUP].int() - 127
    return torch.ldexp(values.view(values.shape[0], -1, GROUP), exponent[..., None]).reshape(values.shape)[:, :k]


def _scores(case, logits):
    if case["scores"] == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    largest = logits.amax(dim=1, keepdim=True)
    powers = torch.exp(logits - torch.where(torch.isinf(largest), 0.0, largest))
    total = powers.sum(dim=1, keepdim=True)
    return torch.where(total == 0, 0.0, powers / total)


def _group_scores(case, value):
    """Sum of each group's two largest, or its one candidate; -inf for a group without any."""
    members = value.view(value.shape[0], case["groups"], -1)
    ranked = torch.sort(members, dim=2, descending=True).values
    if ranked.shape[2] == 1:
        return ranked[..., 0]
    return ranked[..., 0] + torch.where(torch.isinf(ranked[..., 1]), 0.0, ranked[..., 1])


def _kept_groups(case, value):
    order = torch.sort(_group_scores(case, value), dim=1, descending=True, stable=True).indices
    kept = torch.zeros((value.shape[0], case["groups"]), dtype=torch.bool, device=DEVICE)
    kept.scatter_(1, order[:, :case["top_groups"]], True)
    return kept.repeat_interleave(value.shape[1] // case["groups"], dim=1)


def _route(case, logits, bias):
    scores = _scores(case, logits)
    value = scores if bias is None else scores + bias
    value = torch.where(logits == -math.inf, -math.inf, value)
    if case["groups"] > 1:
        value = torch.where(_kept_groups(case, value), value, -math.inf)
    index = torch.arange(case["experts"], device=DEVICE)
    experts = []
    for _ in range(case["top"]):
        largest = value.amax(dim=1, keepdim=True)
        chosen = torch.where(value == largest, index, case["experts"]).amin(dim=1, keepdim=True)
        experts.append(torch.where(torch.isinf(largest), -1, chosen))
        value = torch.where(index == chosen, -math.inf, value)
    experts = torch.cat(experts, dim=1)
    weights = torch.where(experts < 0, 0.0, scores.gather(1, experts.clamp(min=0)))
    if case["renormalize"]:
        total = weights.sum(dim=1, keepdim=True)
        weights = torch.where(total == 0, 0.0, weights / total)
    return experts.to(torch.int32), weights * case["scale"]


def _route_gradient(case, logits, experts, d_weights):
    scores = _scores(case, logits)
    index = experts.long().clamp(min=0)
    d = torch.where(experts < 0, 0.0, d_weights * case["scale"])
    if case["renormalize"]:
        chosen = torch.where(experts < 0, 0.0, scores.gather(1, index))
        total = chosen.sum(dim=1, keepdim=True)
        share = torch.where(total == 0, 0.0, chosen / total)
        d = torch.where((experts < 0) | (total == 0), 0.0, (d - (d * share).sum(dim=1, keepdim=True)) / total)
    d_scores = torch.zeros_like(scores).scatter_add_(1, index, d)
    if case["scores"] == "sigmoid":
        return d_scores * scores * (1 - scores)
    return scores * (d_scores - (d_scores * scores).sum(dim=1, keepdim=True))


# ---- what a pass needs, and what it should give ----------------------------------------


def _packed_bytes(rows, k):
    groups = -(-k // GROUP)
    return rows * groups * (GROUP // 2 + 1)


def work(case):
    op = case["op"]
    item = DTYPES[case["dtype"]].itemsize if "dtype" in case else 0
    if op == "quantize":
        rows, k = (case["k"], case["rows"]) if case["columns"] else (case["rows"], case["k"])
        return {"bytes": rows * k * (item + 2) + _packed_bytes(rows, k), "flops": 0}
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        if not case["backward"]:
            return {"bytes": (m * k + m * n) * item + _packed_bytes(n, k), "flops": 2 * m * n * k}
        return {"bytes": (2 * m * k + 2 * m * n + 2 * n * k) * item, "flops": 6 * m * n * k}
    if op == "experts":
        slots = case["tokens"] * case["top"]
        # Experts that some token chooses, if all were as popular.
        used = case["experts"] * (1 - (1 - case["top"] / case["experts"]) ** case["tokens"])
        return {"bytes": int((case["tokens"] * case["k"] + slots * case["n"]) * item
                             + used * _packed_bytes(case["n"], case["k"]) + slots * 4),
                "flops": 2 * slots * case["n"] * case["k"]}
    if op == "route":
        values = case["tokens"] * case["experts"]
        chosen = case["tokens"] * case["top"]
        return {"bytes": values * item * (2 if case["backward"] else 1) + chosen * (12 if case["backward"] else 8),
                "flops": values * (8 if case["backward"] else 4)}
    if op == "dispatch":
        slots = case["tokens"] * case["top"]
        return {"bytes": 12 * slots + 4 * (case["experts"] + 1), "flops": 0}
    slots, tokens, n = case["tokens"] * case["top"], case["tokens"], case["n"]
    forward = slots * n * item + tokens * n * item + slots * 8
    if not case["backward"]:
        return {"bytes": forward, "flops": 2 * slots * n}
    return {"bytes": forward + slots * n * item + tokens * n * item + slots * 4, "flops": 5 * slots * n}


E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_rounded(x):
    """MXFP4's values of x [rows][k] (64 bits), by the nearest of the eight magnitudes, of two the even code."""
    rows, k = x.shape
    groups = torch.nn.functional.pad(x, (0, -k % GROUP)).view(rows, -1, GROUP)
    largest = groups.abs().amax(dim=2, keepdim=True)
    power = torch.floor(torch.log2(largest))
    # log2 of a value just below a power of two may round up to it.
    power = power - (torch.exp2(power) > largest).double()
    power = torch.where(largest == 0, -127.0, (power - 2).clamp(-127, 127))
    size = groups.abs() / torch.exp2(power)
    code = torch.zeros_like(size)
    for lower, (a, b) in enumerate(zip(E2M1, E2M1[1:])):
        middle = (a + b) / 2
        code += (size >= middle) if lower % 2 else (size > middle)
    value = torch.tensor(E2M1, dtype=torch.float64, device=DEVICE)[code.long()]
    return (torch.sign(groups) * value * torch.exp2(power)).view(rows, -1)[:, :k]


def _exact_operand(codes, scales, k):
    low, high = codes.long() % 16, codes.long() // 16
    code = torch.stack([low, high], dim=2).view(codes.shape[0], -1)[:, :k]
    value = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=DEVICE)[code]
    column = torch.arange(k, device=DEVICE)
    scale = torch.exp2(scales.double() - 127)[column // STEP, :, column % STEP // GROUP]
    return value * scale.t()


def _exact_scores(case, logits):
    return torch.sigmoid(logits) if case["scores"] == "sigmoid" else torch.nan_to_num(torch.softmax(logits, dim=1))


def _exact_route(case, seed):
    logits, bias, d_weights = _route_inputs(case, seed)
    logits = logits.double()
    scores = _exact_scores(case, logits)
    value = scores if bias is None else scores + bias.double()
    value = value.masked_fill(torch.isneginf(logits), -math.inf)
    if case["groups"] > 1:
        group = torch.topk(value.view(value.shape[0], case["groups"], -1), 2, dim=2).values
        group = group[..., 0] + group[..., 1].masked_fill(torch.isneginf(group[..., 1]), 0.0)
        place = (group[:, :, None] < group[:, None, :]).sum(dim=2)  # groups ahead of it; equal ones by their index
        place += torch.tril(group[:, :, None] == group[:, None, :], diagonal=-1).sum(dim=2)
        kept = (place < case["top_groups"]).repeat_interleave(case["experts"] // case["groups"], dim=1)
        value = value.masked_fill(~kept, -math.inf)
    ranked, experts = torch.sort(value, dim=1, descending=True, stable=True)
    ranked, experts = ranked[:, :case["top"]], experts[:, :case["top"]]
    gone = torch.isneginf(ranked)
    chosen = scores.gather(1, experts).masked_fill(gone, 0.0)
    total = chosen.sum(dim=1, keepdim=True) if case["renormalize"] else torch.ones_like(chosen[:, :1])
    weights = case["scale"] * torch.nan_to_num(chosen / total)
    outputs = [experts.masked_fill(gone, -1).to(torch.int32), weights]
    if case["backward"]:
        # Through d(chosen) only: the selection itself has no gradient.
        with torch.enable_grad():
            leaf = torch.where(torch.isneginf(logits), -1e4, logits).requires_grad_()
            score = torch.sigmoid(leaf) if case["scores"] == "sigmoid" else torch.softmax(leaf, dim=1)
            part = score.gather(1, experts) * (~gone)
            if case["renormalize"]:
                part = part / (part.sum(dim=1, keepdim=True) + gone.all(dim=1, keepdim=True))
            (case["scale"] * part * d_weights.double()).sum().backward()
        outputs.append(leaf.grad)
    return tuple(outputs)


def exact(case, seed):
    op = case["op"]
    if op == "quantize":
        x = _activations(_generator(seed), case["rows"], case["k"], case["dtype"]).double()
        return _exact_rounded(x.t().contiguous() if case["columns"] else x)
    if op == "linear":
        x, weight, d_out = _linear_inputs(case, seed)
        x = x.double()
        if not case["backward"]:
            return _exact_rounded(x) @ _exact_operand(*weight, case["k"]).t().contiguous()
        weight, d_out = weight.double(), d_out.double()
        weight_columns = _exact_rounded(weight.t().contiguous()).t().contiguous()
        x_columns = _exact_rounded(x.t().contiguous()).t().contiguous()
        return (_exact_rounded(x) @ _exact_rounded(weight).t().contiguous(), _exact_rounded(d_out) @ weight_columns,
                _exact_rounded(d_out.t().contiguous()) @ x_columns)
    if op == "experts":
        x, assignment, (codes, scales) = _experts_inputs(case, seed)
        x = _exact_rounded(x.double())
        rows = []
        for e in range(case["experts"]):
            token = torch.nonzero(assignment == e)[:, 0]
            rows.append(x[token] @ _exact_operand(codes[e], scales[e], case["k"]).t().contiguous())
        return torch.cat(rows)
    if op == "route":
        return _exact_route(case, seed)
    if op == "dispatch":
        assignment = _assignment(_generator(seed), case["tokens"], case["top"], case["experts"])
        if case["masked"]:
            _mask_rows(assignment)
        flat = assignment.flatten().tolist()
        members = [[] for _ in range(case["experts"])]
        for i, e in enumerate(flat):
            if e >= 0:
                members[e].append(i)
        order = [i for group in members for i in group]
        slots = [-1] * len(flat)
        for slot, i in enumerate(order):
            slots[i] = slot
        offsets = [0]
        for group in members:
            offsets.append(offsets[-1] + len(group))
        order += [-1] * (len(flat) - len(order))
        whole = {"dtype": torch.int32, "device": DEVICE}
        return (torch.tensor(offsets, **whole), torch.tensor(order, **whole),
                torch.tensor(slots, **whole).view(assignment.shape))
    y, slots, weights, d_out = (part.double() if part.is_floating_point() else part.long()
                                for part in _combine_inputs(case, seed))
    out = torch.zeros_like(d_out)
    d_y, d_weights = torch.zeros_like(y), torch.zeros_like(weights)
    for j in range(case["top"]):
        token = torch.nonzero(slots[:, j] >= 0)[:, 0]
        slot = slots[token, j]
        out[token] += weights[token, j, None] * y[slot]
        d_y[slot] = weights[token, j, None] * d_out[token]
        d_weights[token, j] = (d_out[token] * y[slot]).sum(dim=1)
    return (out, d_y, d_weights) if case["backward"] else out
