"""Every kernel of the MXFP4 products by its name, against float64 products of the operands it was given.

A product sums K exact terms in fp32: at most one rounding to 2^-23 of the magnitudes' sum for each of the K / 32
instruction steps and the joins of partial sums (K / 32 + 16 in all), then one rounding to the output type.
"""

import pytest

pytestmark = pytest.mark.gpu

UNIT = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}
SHORT = {"fp32": "f32", "fp16": "f16", "bf16": "bf16"}
TILES = ["128x128", "64x64", "256x128_stream", "128x64_stream", "64x64_stream"]
FEW = ["few_16x8", "few_32x8", "few_32x4"]


def _dtype(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def _random(torch, dtype, *shape, seed=0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=generator).to(_dtype(torch, dtype))


def _name(form, dtype):
    if form.startswith("few_"):
        return f"mx_product_few_{SHORT[dtype]}_{form.removeprefix('few_')}"
    return f"mx_product_{SHORT[dtype]}" + (f"_{form}" if form else "")


def _check(got, a, b, dtype, what=""):
    """`got` against the product of the values a and b (float64, on the device)."""
    k = a.shape[1]
    expected, size = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    bound = (k / 32 + 16) * 2.0**-23 * size
    error = (got.double() - expected).abs()
    assert bool((error <= bound + UNIT[dtype] * (expected.abs() + bound) + 2.0**-24).all()), (what, error.max())


# Rows and n below and past a tile and, in the first, more tiles than a persistent kernel has places; n on and off the
# 16-byte pieces of each type; K of one step, of several, odd, and with a last one in part.
SIZES = [(4200, 2051, 300), (2117, 1029, 513), (300, 264, 1100), (129, 261, 96), (3, 5, 40), (1, 130, 2081),
         (513, 77, 1), (65, 1040, 256)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form", [*TILES, *FEW, ""])
def test_one_weight(gpu, form, dtype):
    import torch

    from triton_chip_benchmarks_amd import mx

    for rows, n, k in SIZES:
        print(f"{_name(form, dtype)} {rows}x{n}x{k}", flush=True)
        a, b = mx.quantize(_random(torch, dtype, rows, k, seed=1)), mx.quantize(_random(torch, dtype, n, k, seed=2))
        guarded = torch.full((rows + 2, n), 7.0, device="cuda", dtype=_dtype(torch, dtype))
        out = guarded[1:-1]
        mx.product(a, b, out, kernel=_name(form, dtype))
        _check(out, mx.dequantize(a).double(), mx.dequantize(b).double(), dtype, (rows, n, k))
        assert (guarded[0] == 7).all() and (guarded[-1] == 7).all()
        again = mx.product(a, b, dtype=out.dtype, kernel=_name(form, dtype))
        assert torch.equal(again, out), (rows, n, k)


def _offsets(torch, counts, first=0):
    offsets = torch.zeros(len(counts) + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.tensor(counts).cumsum(0)
    return offsets + first


def _weights(torch, mx, dtype, experts, n, k):
    parts = [mx.quantize(_random(torch, dtype, n, k, seed=10 + e)) for e in range(experts)]
    return mx.Packed(torch.stack([p.codes for p in parts]), torch.stack([p.scales for p in parts]), k), parts


# Rows of each expert: none, one, a tile's and past it, most of them in one; and how many rows lie behind the last.
COUNTS = [([0, 1, 200, 0, 64, 129, 3], 5), ([0, 0, 33, 0], 0), ([700, 0, 1, 2500], 9), ([1] * 70 + [0] * 30 + [17] * 3, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("form", [*TILES, *FEW, ""])
def test_experts(gpu, form, dtype):
    import torch

    from triton_chip_benchmarks_amd import mx

    for (counts, behind), n, k in zip(COUNTS, (261, 130, 519, 72), (300, 520, 96, 270)):
        rows = sum(counts) + behind
        print(f"{_name(form, dtype)} {rows} of {len(counts)} x {n}x{k}", flush=True)
        a = mx.quantize(_random(torch, dtype, rows, k, seed=1))
        b, parts = _weights(torch, mx, dtype, len(counts), n, k)
        guarded = torch.full((rows + 2, n), 7.0, device="cuda", dtype=_dtype(torch, dtype))
        out = guarded[1:-1]
        offsets = _offsets(torch, counts)
        mx.product(a, b, out, offsets=offsets, kernel=_name(form, dtype))
        values, ends = mx.dequantize(a).double(), offsets.tolist()
        for e, (first, last) in enumerate(zip(ends, ends[1:])):
            if last > first:
                _check(out[first:last], values[first:last], mx.dequantize(parts[e]).double(), dtype, (counts, e))
        assert (out[ends[-1]:] == 7).all() and (guarded[0] == 7).all() and (guarded[-1] == 7).all()


# (rows, n, k, form) of one weight: n past the features of a workgroup; 16 rows of K = 8192 take 70 KiB of LDS.
FEW_ROWS = [(1, 8203, 40, "32x8"), (2, 8203, 1000, "32x8"), (15, 8203, 600, "32x8"), (16, 8200, 8192, "32x8"),
            (16, 1030, 14000, "16x8"), (9, 333, 8200, "16x8"), (1, 70, 100000, "16x8"), (1, 65570, 100, "32x4"),
            (7, 65570, 300, "32x4"), (16, 65600, 40, "32x4")]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k,form", FEW_ROWS)
def test_linear_of_few_rows(gpu, dtype, rows, n, k, form):
    import torch

    from triton_chip_benchmarks_amd import mx

    print(f"linear {dtype} {rows}x{n}x{k}", flush=True)
    assert mx.product_kernel(rows, n, k, _dtype(torch, dtype), linear=True) == f"mx_linear_few_{SHORT[dtype]}_{form}"
    wide = _random(torch, dtype, rows, k + 9, seed=1)
    x = wide[:, 3:k + 3]  # off every vector's alignment
    weight = mx.quantize(_random(torch, dtype, n, k, seed=2))
    out = mx.linear(x, weight)
    _check(out, mx.dequantize(mx.quantize(x)).double(), mx.dequantize(weight).double(), dtype)
    assert torch.equal(mx.linear(x, weight), out)
    assert torch.equal(mx.product(mx.quantize(x), weight, dtype=x.dtype), out)


# Tokens, their choices (how many go to expert 0, the rest spread over the others), sizes, and the form that they run
# on: fewer rows than experts, between one and two an expert, and more than the 16 rows of a pass in one of them.
ROUTED = [(70, 1, 3, 128, 1000, 300, "32x4"), (64, 2, 17, 64, 1030, 288, "32x4"), (64, 2, 33, 64, 1030, 100, "32x4"),
          (100, 2, 40, 100, 700, 512, "32x4"), (64, 2, 17, 64, 200, 520, "32x8"), (40, 1, 33, 33, 300, 264, "32x8"),
          (20, 2, 40, 32, 100, 1000, "16x8"), (20, 1, 17, 30, 130, 96, "16x8"), (3, 2, 0, 16, 333, 40, "16x8")]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,top,first,experts,n,k,form", ROUTED)
def test_linear_of_few_rows_an_expert(gpu, dtype, tokens, top, first, experts, n, k, form):
    import torch

    from triton_chip_benchmarks_amd import mx, routing

    rows = tokens * top
    print(f"linear {dtype} {tokens} of {top}x{experts}, {first} to one, {n}x{k}", flush=True)
    assert mx.product_kernel(rows, n, k, _dtype(torch, dtype), experts, linear=True) == \
        f"mx_linear_few_{SHORT[dtype]}_{form}"
    chosen = torch.zeros(rows, dtype=torch.int32)
    chosen[first:] = 1 + torch.arange(rows - first, dtype=torch.int32) % (experts - 1)
    chosen = chosen[torch.randperm(rows, generator=torch.Generator().manual_seed(rows))].view(tokens, top).contiguous()
    chosen[-1, -1] = -1
    plan = routing.dispatch(chosen.cuda(), experts)
    x = _random(torch, dtype, tokens, k, seed=3)
    weight, parts = _weights(torch, mx, dtype, experts, n, k)
    out = torch.full((rows, n), 7.0, device="cuda", dtype=x.dtype)
    mx.linear(x, weight, out, plan=plan)
    ends, token = plan.offsets.tolist(), plan.order.long() // top
    values = mx.dequantize(mx.quantize(x)).double()
    for e, (start, end) in enumerate(zip(ends, ends[1:])):
        if end > start:
            _check(out[start:end], values[token[start:end]], mx.dequantize(parts[e]).double(), dtype, e)
    assert (out[ends[-1]:] == 7).all()
    routed = torch.zeros(rows, k, device="cuda", dtype=x.dtype)
    routed[:ends[-1]] = x[token[:ends[-1]]]
    for again in (mx.linear(routed, weight, torch.full_like(out, 7.0), plan=plan, sorted_rows=True),
                  mx.product(mx.quantize(routed), weight, torch.full_like(out, 7.0), offsets=plan.offsets)):
        assert torch.equal(again, out)
