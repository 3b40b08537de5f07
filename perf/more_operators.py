"""The operators of a feed-forward block in 8-bit floating point, one pass each.

An operator is a call that a training or serving program makes on tensors it
holds: the root-mean-square norm with the residual's addition (and an output in
8 bits), a linear layer whose operands are E4M3 with a power-of-two scale for
each block of 128 (dense, with its gradients, or one weight per expert), and the
gated pair of projections, silu(x . G^T) * (x . U^T), of one weight or of the
experts', with its gradients. `run` computes it in elementary torch operations,
or through the package's entry points. `listed` names the cases compared from
change to change; `draw` spreads more over the same ranges.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 128          # elements along K, and rows of a weight, that share one scale
EPS = 1e-6
MOST_FLOPS = 2 * 8192**3       # of a pass
MOST_WEIGHTS = 1 << 30         # elements over all experts
MOST_ELEMENTS = 16384 * 8192   # of a normed tensor


def listed():
    return [
        # One token through a layer: the weight's bytes are all there is.
        {"name": "linear_bf16_1x8192x8192", "op": "linear", "dtype": "bf16", "rows": 1, "n": 8192, "k": 8192,
         "experts": 0, "top": 1, "backward": False},
        # A prompt through the same layer, its rows quantised on the way.
        {"name": "linear_bf16_8192x8192x8192", "op": "linear", "dtype": "bf16", "rows": 8192, "n": 8192, "k": 8192,
         "experts": 0, "top": 1, "backward": False},
        # A training step of a layer of sizes off every tile: both operands quantised, output and both gradients.
        {"name": "linear_train_bf16_5000x3000x4112", "op": "linear", "dtype": "bf16", "rows": 5000, "n": 3000,
         "k": 4112, "experts": 0, "top": 1, "backward": True},
        # Prompts through experts' projections back: hundreds of rows an expert, unevenly, a short K.
        {"name": "linear_bf16_4096of8x128", "op": "linear", "dtype": "bf16", "rows": 4096, "n": 4096, "k": 1024,
         "experts": 128, "top": 8, "backward": False},
        # A decoded batch through a dense block's two projections: 117 MB of weights.
        {"name": "gated_bf16_16x14336x4096", "op": "gated", "dtype": "bf16", "rows": 16, "n": 14336, "k": 4096,
         "experts": 0, "top": 1, "out": "same", "backward": False},
        # A decoded batch through its experts': two rows an expert, most weights read once.
        {"name": "gated_bf16_32of8x128", "op": "gated", "dtype": "bf16", "rows": 32, "n": 1024, "k": 4096,
         "experts": 128, "top": 8, "out": "same", "backward": False},
        # Prompts through the experts', the output in 8 bits for the projection back.
        {"name": "gated_fp8_bf16_4096of8x128", "op": "gated", "dtype": "bf16", "rows": 4096, "n": 1024, "k": 4096,
         "experts": 128, "top": 8, "out": "fp8", "backward": False},
        # A training step of a dense block: the output, what the gradient needs of it, and both gradients.
        {"name": "gated_train_bf16_5000x3000x4112", "op": "gated", "dtype": "bf16", "rows": 5000, "n": 3000,
         "k": 4112, "experts": 0, "top": 1, "out": "same", "backward": True},
        # One token's norm between two layers: all latency.
        {"name": "norm_bf16_1x8192", "op": "norm", "dtype": "bf16", "rows": 1, "n": 8192, "residual": True,
         "out": "same", "backward": False},
        # A prompt's norm ahead of a layer in 8 bits.
        {"name": "norm_fp8_bf16_16384x8192", "op": "norm", "dtype": "bf16", "rows": 16384, "n": 8192,
         "residual": True, "out": "fp8", "backward": False},
        # A training step's norm: the output, the residual stream and the gradients.
        {"name": "norm_train_bf16_8192x8192", "op": "norm", "dtype": "bf16", "rows": 8192, "n": 8192,
         "residual": True, "out": "same", "backward": True},
        # The same of a width that fills no vector, in 32 bits, without a residual.
        {"name": "norm_train_fp32_1000x5003", "op": "norm", "dtype": "fp32", "rows": 1000, "n": 5003,
         "residual": False, "out": "same", "backward": True},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _flops(case):
    """Of the products: two an element of them, and as many for each of two gradients."""
    width = 2 * case["n"] if case["op"] == "gated" else case["n"]
    return 2 * case["rows"] * case["top"] * width * case["k"] * (3 if case["backward"] else 1)


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "gated", "norm"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    while True:
        if op == "norm":
            case = {"op": op, "dtype": dtype, "rows": _log_uniform(rng, 1, 16384), "n": _log_uniform(rng, 64, 16384),
                    "residual": rng.random() < 0.7, "out": rng.choice(["same", "fp8", "both"]),
                    "backward": rng.random() < 0.4}
            if case["rows"] * case["n"] <= MOST_ELEMENTS // 2:
                return case
            continue
        experts = rng.choice([0, 0, 8, 16, 32, 60, 128, 256])
        case = {"op": op, "dtype": dtype, "rows": _log_uniform(rng, 1, 8192), "n": _log_uniform(rng, 64, 8192),
                "k": _log_uniform(rng, 64, 8192), "experts": experts,
                "top": rng.choice([1, 2, 4, 6, 8]) if experts else 1, "backward": not experts and rng.random() < 0.4}
        if op == "gated":
            case["out"] = "same" if case["backward"] else rng.choice(["same", "fp8"])
            if case["backward"] and dtype == "fp32":
                case["dtype"] = "bf16"  # a training step's activations have 16 bits
        if _flops(case) <= MOST_FLOPS // 2 and 2 * max(experts, 1) * case["n"] * case["k"] <= MOST_WEIGHTS:
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
    uniform = torch.rand((tokens, experts), device=DEVICE, generator=generator).clamp(1e-9, 1 - 1e-7)
    noise = -torch.log(-torch.log(uniform))
    return torch.argsort(popularity + noise, dim=1, descending=True)[:, :top].to(torch.int32).contiguous()


def _sorted(assignment, experts):
    """(offsets, order, slots), int32, of an assignment [tokens][top]: its entries by expert, in their order."""
    flat = assignment.reshape(-1).long()
    order = torch.argsort(flat, stable=True)
    counts = (flat[:, None] == torch.arange(experts, device=DEVICE)).sum(dim=0)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=DEVICE)
    offsets[1:] = torch.cumsum(counts, 0)
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(flat.numel(), device=DEVICE)
    return tuple(part.to(torch.int32) for part in (offsets, order, slots.view(assignment.shape)))


def _product_inputs(case, seed):
    """(x, weight, d_out, assignment): the weight in the layer's type where it is trained, else packed; rows of a routed
    linear layer are in the experts' order already, a gated one takes the tokens."""
    generator = _generator(seed)
    rows, n, k, experts = case["rows"], case["n"], case["k"], case["experts"]
    gated = case["op"] == "gated"
    width = 2 * n if gated else n
    assignment = _assignment(generator, rows, case["top"], experts) if experts else None
    x = _activations(generator, rows if gated or not experts else rows * case["top"], k, case["dtype"])
    if case["backward"]:
        weight = (_randn(generator, width, k) / math.sqrt(k)).to(DTYPES[case["dtype"]])
        return x, weight, (1e-3 * _randn(generator, rows, n)).to(x.dtype), assignment
    weights = [_pack(_randn(generator, width, k) / math.sqrt(k)) for _ in range(max(experts, 1))]
    weight = tuple(torch.stack(parts) for parts in zip(*weights)) if experts else weights[0]
    return x, weight, None, assignment


def _norm_inputs(case, seed):
    """(x, residual, weight, d_out, d_total); the residual's stream is some times as large as what is added to it."""
    generator = _generator(seed)
    rows, n, dtype = case["rows"], case["n"], DTYPES[case["dtype"]]
    x = _activations(generator, rows, n, case["dtype"])
    residual = (4 * _activations(generator, rows, n, "fp32")).to(dtype) if case["residual"] else None
    weight = (1 + 0.1 * _randn(generator, n)).to(dtype)
    d_out = (1e-3 * _randn(generator, rows, n)).to(dtype)
    d_total = (1e-3 * _randn(generator, rows, n)).to(dtype) if case["residual"] else None
    return x, residual, weight, d_out, d_total


def prepare(case, seed):
    state = {"case": case}
    if case["op"] == "norm":
        names = ("x", "residual", "weight", "d_out", "d_total")
        state.update(zip(names, _norm_inputs(case, seed)))
    else:
        state["x"], state["weight"], state["d_out"], assignment = _product_inputs(case, seed)
        state["plan"] = None
        if assignment is not None:
            state["plan"] = _sorted(assignment, case["experts"])
            state["host_offsets"] = state["plan"][0].tolist()  # where the plain form splits its rows
    if own:
        _buffers(state)
    return state


def _buffers(state):
    """Outputs and workspaces, made once as a program makes them."""
    from triton_chip_benchmarks_amd import fp8, norm, routing

    case, x = state["case"], state["x"]

    def like(*shape, dtype=x.dtype):
        return torch.empty(shape, device=DEVICE, dtype=dtype)

    if case["op"] == "norm":
        rows, n = x.shape
        state["out"] = like(rows, n) if case["out"] != "fp8" else None
        state["packed"] = state["values"] = None
        if case["out"] != "same":
            state["packed"], state["values"] = fp8.empty(rows, n, device=DEVICE), like(rows, n, dtype=torch.bfloat16)
        state["total"] = like(rows, n) if case["residual"] else None
        if case["backward"]:
            state["d_x"], state["d_weight"] = like(rows, n), like(n)
            state["workspace"] = norm.rms_norm_backward_workspace(rows, n, device=DEVICE)
        return
    rows, n, k, experts = case["rows"] * case["top"], case["n"], case["k"], max(case["experts"], 1)
    gated = case["op"] == "gated"
    if state["plan"] is not None:
        state["plan"] = routing.Plan(*state["plan"])
    state["out"] = state["packed"] = state["values"] = state["gate_up"] = None
    if case.get("out") == "fp8":
        state["packed"], state["values"] = fp8.empty(rows, n, device=DEVICE), like(rows, n, dtype=torch.bfloat16)
    else:
        state["out"] = like(rows, n)
    if not case["backward"]:
        state["weight"] = fp8.Packed(*state["weight"], k, block=BLOCK)
        space = fp8.gated_workspace if gated else fp8.linear_workspace
        state["workspace"] = space(rows, n, k, x.dtype, experts=experts, device=DEVICE)
        return
    width = 2 * n if gated else n
    state["weight_rows"] = fp8.empty(width, k, block=BLOCK, device=DEVICE)
    state["weight_columns"] = fp8.empty(k, width, block=BLOCK, device=DEVICE)
    state["d_x"], state["d_weight"] = like(rows, k), like(width, k)
    space = fp8.gated_backward_workspace if gated else fp8.linear_backward_workspace
    state["workspace"] = space(rows, n, k, x.dtype, device=DEVICE)
    if gated:
        state["gate_up"] = like(rows, 2 * n)


# ---- one pass ------------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from triton_chip_benchmarks_amd import fp8, norm

    case, x, weight = state["case"], state["x"], state["weight"]
    if case["op"] == "norm":
        normed = norm.rms_norm(x, weight, EPS, residual=state["residual"], out=state["out"], packed=state["packed"],
                               total=state["total"])
        outputs = [part for part in (normed.out, normed.total) if part is not None and part is not x]
        if normed.packed is not None:
            outputs.append(fp8.dequantize(normed.packed, state["values"]))
        if case["backward"]:
            outputs += norm.rms_norm_backward(state["d_out"], normed.total, weight, EPS, d_total=state["d_total"],
                                              d_x=state["d_x"], d_weight=state["d_weight"],
                                              workspace=state["workspace"])
        return tuple(outputs)
    gated, plan, space = case["op"] == "gated", state["plan"], state["workspace"]
    if not case["backward"]:
        if not gated:
            return fp8.linear(x, weight, state["out"], plan=plan, sorted_rows=plan is not None, workspace=space)
        out = fp8.gated(x, weight, state["out"], packed=state["packed"], plan=plan, workspace=space)
        return fp8.dequantize(out, state["values"]) if case["out"] == "fp8" else out
    weight_rows, weight_columns = fp8.quantize_both(weight, state["weight_rows"], state["weight_columns"], block=BLOCK)
    if not gated:
        out = fp8.linear(x, weight_rows, state["out"], workspace=space)
        return (out, *fp8.linear_backward(state["d_out"], x, weight_columns, state["d_x"], state["d_weight"],
                                          workspace=space))
    gate_up = state["gate_up"]
    out = fp8.gated(x, weight_rows, state["out"], gate_up=gate_up, workspace=space)
    return (out, gate_up, *fp8.gated_backward(state["d_out"], gate_up, x, weight_columns, state["d_x"],
                                              state["d_weight"], workspace=space))


def _run_plain(state):
    case = state["case"]
    if case["op"] == "norm":
        return _plain_norm(state)
    x, weight, dtype, n = state["x"].float(), state["weight"], state["x"].dtype, case["n"]
    gated = case["op"] == "gated"
    if not case["backward"]:
        x = _rounded(x)
        if state["plan"] is None:
            product = torch.matmul(x, _unpack(*weight, case["k"]).t())
        else:
            _, order, _ = state["plan"]
            product = torch.empty((order.numel(), 2 * n if gated else n), device=DEVICE)
            for e, (first, last) in enumerate(zip(state["host_offsets"], state["host_offsets"][1:])):
                if last > first:
                    rows = x[order[first:last].long() // case["top"]] if gated else x[first:last]
                    product[first:last] = torch.matmul(rows, _unpack(weight[0][e], weight[1][e], case["k"]).t())
        if not gated:
            return product.to(dtype)
        out = _gate(product)
        return _rounded(out).to(torch.bfloat16) if case["out"] == "fp8" else out.to(dtype)
    weight, d_out = _rounded_block(weight.float()), state["d_out"].float()
    product = torch.matmul(_rounded(x), weight.t())
    outputs = [product.to(dtype)]
    if gated:
        gate_up = product.to(dtype)
        outputs = [_gate(product).to(dtype), gate_up]
        # In 64 bits: what follows is rounded to four.
        gate, up = gate_up.double().chunk(2, dim=1)
        sigmoid = 1 / (1 + torch.exp(-gate))
        d_out = d_out.double()
        d_out = torch.cat([d_out * up * sigmoid * (1 + gate * (1 - sigmoid)), d_out * gate * sigmoid], dim=1).float()
    d_x = torch.matmul(_rounded(d_out), weight)
    d_weight = torch.matmul(_rounded(d_out.t()), _rounded(x.t()).t())
    return (*outputs, d_x.to(dtype), d_weight.to(dtype))


def _plain_norm(state):
    case, x, weight, dtype = state["case"], state["x"], state["weight"].float(), state["x"].dtype
    outputs, total = [], x
    if state["residual"] is not None:
        total = (x.float() + state["residual"].float()).to(dtype)
    values = total.float()
    inverse = torch.rsqrt((values * values).mean(dim=1, keepdim=True) + EPS)
    normed = values * inverse
    if case["out"] != "fp8":
        outputs.append((normed * weight).to(dtype))
    if state["residual"] is not None:
        outputs.append(total)
    if case["out"] != "same":
        # In 64 bits: what follows is rounded to four.
        wide = values.double()
        wide = wide * torch.rsqrt((wide * wide).mean(dim=1, keepdim=True) + EPS) * weight.double()
        outputs.append(_rounded(wide.float()).to(torch.bfloat16))
    if case["backward"]:
        d_out = state["d_out"].float()
        d_normed = d_out * weight
        d_x = inverse * (d_normed - normed * (d_normed * normed).mean(dim=1, keepdim=True))
        if state["d_total"] is not None:
            d_x = d_x + state["d_total"].float()
        d_weight = (d_out * normed).double().sum(dim=0)
        outputs += [d_x.to(dtype), d_weight.to(dtype)]
    return tuple(outputs)


# The plain forms' parts, in 32 bits.


def _gate(product):
    gate, up = product.chunk(2, dim=1)
    return gate / (1 + torch.exp(-gate)) * up


def _scale_exponents(largest):
    """The smallest e with max|x| <= 448 * 2^e, at least -127; -127 for zeros."""
    fraction, exponent = torch.frexp(largest)
    exponent = exponent - 9 + (fraction > 0.875).int()
    return torch.where(largest == 0, -127, exponent).clamp(min=-127)


def _scaled(x, exponent):
    """x * 2^exponent, by exact powers of two: a library's pow(2, e) may be off by a bit, which decides ties."""
    half = exponent.int() // 2
    powers = [((part + 127) << 23).view(torch.float32) for part in (half, exponent.int() - half)]
    return x * powers[0] * powers[1]


def _codes(x, exponent):
    """x / 2^exponent as E4M3 holds it: four bits down to 2^-6, steps of 2^-9 below, ties to even."""
    scaled = _scaled(x, -exponent)
    step = _scaled(torch.ones_like(scaled), torch.frexp(scaled).exponent.clamp(min=-5) - 4)
    return torch.round(scaled / step) * step


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % BLOCK)).view(x.shape[0], -1, BLOCK)


def _rounded(x):
    """x [rows][k] as an operand holds it, a scale for each 128 of a row."""
    blocks = _blocks(x)
    exponent = _scale_exponents(blocks.abs().amax(dim=2, keepdim=True))
    return _scaled(_codes(blocks, exponent), exponent).view(x.shape[0], -1)[:, :x.shape[1]]


def _square_exponents(x):
    """Exponents of the 128 x 128 blocks, [ceil(rows/128)][ceil(k/128)]."""
    rows, k = x.shape
    padded = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, -rows % BLOCK))
    squares = padded.view(padded.shape[0] // BLOCK, BLOCK, padded.shape[1] // BLOCK, BLOCK)
    return _scale_exponents(squares.abs().amax(dim=3).amax(dim=1))


def _spread(exponent, rows, k):
    return exponent.repeat_interleave(BLOCK, dim=0)[:rows].repeat_interleave(BLOCK, dim=1)[:, :k]


def _rounded_block(x):
    exponent = _spread(_square_exponents(x), *x.shape)
    return _scaled(_codes(x, exponent), exponent)


def _pack(x):
    """Codes [rows][k rounded up to 16] and scales [ceil(k/512)][ceil(rows/128)][4] of a weight."""
    rows, k = x.shape
    exponent = _square_exponents(x)
    codes = torch.nn.functional.pad(_codes(x, _spread(exponent, rows, k)), (0, -k % 16)).to(torch.float8_e4m3fn)
    steps = -(-k // (4 * BLOCK))
    scales = torch.full((exponent.shape[0], steps * 4), 127, device=DEVICE, dtype=torch.uint8)
    scales[:, :exponent.shape[1]] = (exponent + 127).to(torch.uint8)
    return codes, scales.view(-1, steps, 4).permute(1, 0, 2).contiguous()


def _unpack(codes, scales, k):
    exponent = scales.permute(1, 0, 2).reshape(scales.shape[1], -1).int() - 127
    return _scaled(codes.float()[:, :k], _spread(exponent, codes.shape[0], k))


# ---- what a pass needs, and what it should give ----------------------------------------


def work(case):
    item, rows, n = DTYPES[case["dtype"]].itemsize, case["rows"], case["n"]
    if case["op"] == "norm":
        values = rows * n
        read = values * item * (2 if case["residual"] else 1) + n * item
        write = values * (item * (case["residual"] + (case["out"] != "fp8")) + 2 * (case["out"] != "same"))
        if case["backward"]:
            read += values * item * (2 if case["residual"] else 1)
            write += values * item + n * item
        return {"bytes": read + write, "flops": values * (4 + 8 * case["backward"])}
    gated, k, top, experts = case["op"] == "gated", case["k"], case["top"], case["experts"]
    width, routed = (2 * n if gated else n), rows * top
    if case["backward"]:
        values = 2 * rows * k + 2 * rows * n + 2 * width * k + (rows * width if gated else 0)
        return {"bytes": values * item, "flops": _flops(case)}
    # Experts that some token chooses, if all were as popular.
    used = experts * (1 - (1 - top / experts)**rows) if experts else 1
    weights = width * k + -(-width // BLOCK) * -(-k // BLOCK)
    in_rows = rows if gated else routed
    out_item = 2 if case.get("out") == "fp8" else item
    return {"bytes": int(in_rows * k * item + routed * n * out_item + used * weights + 4 * routed * bool(experts)),
            "flops": _flops(case)}


def _exact_rounded(x, height=1):
    """E4M3 values of x [rows][k] (64 bits) in blocks of `height` rows by 128."""
    rows, k = x.shape
    magnitude = x.abs()
    tall = torch.nn.functional.pad(magnitude, (0, -k % BLOCK, 0, -rows % height))
    tall = tall.unflatten(1, (-1, BLOCK)).amax(dim=2).unflatten(0, (-1, height)).amax(dim=1)
    power = torch.ceil(torch.log2(tall / 448))
    # log2 of a quotient next to a power of two may land on its other side.
    power = power + (tall > 448 * torch.exp2(power)).double() - (tall <= 448 * torch.exp2(power - 1)).double()
    power = torch.where(tall == 0, -127.0, power).clamp(min=-127)
    scale = torch.exp2(power)[torch.arange(rows, device=DEVICE) // height][:, torch.arange(k, device=DEVICE) // BLOCK]
    size = magnitude / scale
    binade = torch.floor(torch.log2(size.clamp(min=2.0**-6)))
    binade = binade - (torch.exp2(binade) > size.clamp(min=2.0**-6)).double()
    units = size * torch.exp2(3 - binade)  # of the last bit
    low = torch.floor(units)
    above = units - low
    up = (above > 0.5) | ((above == 0.5) & (low % 2 == 1))
    return torch.sign(x) * (low + up) * torch.exp2(binade - 3) * scale


def _exact_operand(codes, scales, k):
    """Values, in 64 bits, of a packed weight."""
    byte = codes.view(torch.uint8).long()[:, :k]
    field, fraction = byte // 8 % 16, (byte % 8).double()
    value = torch.where(field == 0, fraction * 2.0**-9, (8 + fraction) * torch.exp2(field.double() - 10))
    row, column = torch.arange(codes.shape[0], device=DEVICE), torch.arange(k, device=DEVICE)
    scale = scales[column // 512, :, column % 512 // BLOCK].t()[row // BLOCK]
    return torch.where(byte >= 128, -value, value) * torch.exp2(scale.double() - 127)


def _exact_norm(case, seed):
    x, residual, weight, d_out, d_total = (part if part is None else part.double()
                                           for part in _norm_inputs(case, seed))
    dtype, outputs = DTYPES[case["dtype"]], []
    total = x
    if residual is not None:
        total = (x + residual).to(dtype).double()
    scale = 1 / torch.sqrt(total.square().sum(dim=1) / case["n"] + EPS)
    out = total * scale[:, None] * weight
    if case["out"] != "fp8":
        outputs.append(out)
    if residual is not None:
        outputs.append(total)
    if case["out"] != "same":
        outputs.append(_exact_rounded(out))
    if case["backward"]:
        # d(total / rms): the part along total is lost.
        along = (d_out * weight * total).sum(dim=1) * scale.pow(3) / case["n"]
        d_x = d_out * weight * scale[:, None] - total * along[:, None]
        outputs.append(d_x if d_total is None else d_x + d_total)
        outputs.append((d_out * total * scale[:, None]).sum(dim=0))
    return tuple(outputs)


def exact(case, seed):
    if case["op"] == "norm":
        return _exact_norm(case, seed)
    x, weight, d_out, assignment = _product_inputs(case, seed)
    gated, dtype, n = case["op"] == "gated", x.dtype, case["n"]
    x = x.double()
    if case["backward"]:
        weight = _exact_rounded(weight.double(), height=BLOCK)
        out = _exact_rounded(x) @ weight.t().contiguous()
        outputs, d_out = [out], d_out.double()
        if gated:
            out, d_pair = _exact_gate(out, out.to(dtype).double(), d_out)
            outputs = [out[0], out[1]]
            d_out = d_pair
        d_weight = _exact_rounded(d_out.t().contiguous()) @ _exact_rounded(x.t().contiguous()).t().contiguous()
        return (*outputs, _exact_rounded(d_out) @ weight, d_weight)
    x = _exact_rounded(x)
    if assignment is None:
        out = x @ _exact_operand(*weight, case["k"]).t().contiguous()
    else:
        rows, done = [], 0
        for e in range(case["experts"]):
            token = torch.nonzero(assignment == e)[:, 0]
            part = x[token] if gated else x[done:done + token.numel()]
            done += token.numel()
            rows.append(part @ _exact_operand(weight[0][e], weight[1][e], case["k"]).t().contiguous())
        out = torch.cat(rows)
    if not gated:
        return out
    out = torch.nn.functional.silu(out[:, :n]) * out[:, n:]
    return _exact_rounded(out) if case["out"] == "fp8" else out


def _exact_gate(pair, saved, d_out):
    """((out, pair), gradient of the saved pair), the gradient by differentiation."""
    n = d_out.shape[1]
    out = torch.nn.functional.silu(pair[:, :n]) * pair[:, n:]
    with torch.enable_grad():
        leaf = saved.clone().requires_grad_()
        (torch.nn.functional.silu(leaf[:, :n]) * leaf[:, n:] * d_out).sum().backward()
    return (out, pair), leaf.grad
