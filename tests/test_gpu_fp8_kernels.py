"""Every kernel of FP8 products, by its name, over sizes on and off its tiles, against float64 products on the device;
the tolerances are those of test_gpu_fp8_product.py."""

import math

import pytest

from triton_chip_benchmarks_amd import _native

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16", "e4m3": "bfloat16"}


def kernels(kind):
    """Those that take an operand; a kernel of few rows keeps the gate and up where it is given a place."""
    few = "gated" if kind == "gated_kept" else kind
    starts = {f"fp8_few_{few}_e4m3_{y}_": y for y in TYPES} | {f"fp8_tiles_{kind}_{y}_": y for y in TYPES}
    return [(name, y) for name in _native.kernel_names() for start, y in starts.items() if name.startswith(start)]


# Rows and columns off every tile and many of them; K of one block, its neighbours, and enough for the ring to turn.
DENSE = [(1, 40, 128), (70, 300, 112), (300, 777, 130), (1030, 1160, 1040), (515, 2049, 272)]
ROUTED = [(7, 3, 130, 400), (1500, 9, 272, 640), (700, 256, 200, 256)]


def operand(torch, rows, k, block, generator, experts=None):
    from triton_chip_benchmarks_amd import fp8

    channel = torch.where(torch.rand(k, device="cuda", generator=generator) < 0.05, 10.0, 1.0)
    parts = [fp8.quantize(torch.randn(rows, k, device="cuda", generator=generator) * channel, block=block)
             for _ in range(experts or 1)]
    values = [fp8.dequantize(part, torch.empty(rows, k, device="cuda")).double() for part in parts]
    if experts is None:
        return parts[0], values[0]
    whole = fp8.Packed(torch.stack([p.codes.view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn),
                       torch.stack([p.scales for p in parts]), k, block)
    return whole, values


def offsets_of(torch, rows, experts, generator, hole):
    """Rows of the experts, some without any; `hole` rows are nobody's."""
    cuts = torch.randint(0, rows - hole + 1, (experts - 1,), device="cuda", generator=generator).sort().values
    ends = [0, *cuts.tolist(), rows - hole]
    return torch.tensor(ends, dtype=torch.int32, device="cuda"), ends


def reference(torch, a, b, ends):
    """(a . b^T, its magnitudes), of one weight or of the experts'."""
    if ends is None:
        return a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    parts = [(a[x:y], w) for x, y, w in zip(ends, ends[1:], b)]
    return (torch.cat([x @ w.t().contiguous() for x, w in parts]),
            torch.cat([x.abs() @ w.abs().t().contiguous() for x, w in parts]))


def sizes():
    for rows, n, k in DENSE:
        for a_block, b_block in ((1, 128), (128, 1)):
            yield rows, None, n, k, a_block, b_block
    for rows, experts, n, k in ROUTED:
        yield rows, experts, n, k, 1, 128
        yield rows, experts, n, k, 1, 1


def floor(torch, dtype):
    """Half the spacing of the type's smallest values: fp16 below its 2^-14 rounds by up to 2^-25, however small."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def sums(dtype, k):
    return k * 2.0**-24 if dtype == "float32" else 2.0**-12


@pytest.mark.parametrize("size", list(sizes()), ids=str)
def test_products(gpu, size):
    import torch

    from triton_chip_benchmarks_amd import fp8

    rows, experts, n, k, a_block, b_block = size
    generator = torch.Generator(device="cuda").manual_seed(rows + n + k)
    a, a_values = operand(torch, rows, k, a_block, generator)
    b, b_values = operand(torch, n, k, b_block, generator, experts)
    offsets, ends = offsets_of(torch, rows, experts, generator, 3) if experts else (None, None)
    exact, magnitudes = reference(torch, a_values, b_values, ends)
    live, ran = exact.shape[0], 0
    for name, y in kernels("product"):
        print(f"kernel {name} {size}", flush=True)
        dtype = getattr(torch, TYPES[y])
        out = torch.full((rows, n), 7.0, device="cuda", dtype=dtype)
        fp8.product(a, b, out, offsets=offsets, kernel=name)
        off = sums(TYPES[y], k) * (1 + 2.0**-7) * magnitudes
        bound = off + torch.finfo(dtype).eps / 2 * (exact.abs() + off) + floor(torch, dtype)
        assert ((out[:live].double() - exact).abs() <= bound).all(), name
        assert (out[live:] == 7).all(), name
        ran += 1
    assert ran >= 20


@pytest.mark.parametrize("kind", ["gated", "gated_kept", "gated_fp8"])
@pytest.mark.parametrize("size", list(sizes()), ids=str)
def test_gated(gpu, kind, size):
    import torch

    from triton_chip_benchmarks_amd import fp8, routing

    rows, experts, n, k, a_block, b_block = size
    generator = torch.Generator(device="cuda").manual_seed(rows + n + k + 1)
    a, a_values = operand(torch, rows, k, a_block, generator)
    b, b_values = operand(torch, 2 * n, k, b_block, generator, experts)
    # Sums of some units, so that the gates matter: exact, by the scales.
    lower = max(0, round(math.log2(40 * math.sqrt(k))))
    b.scales.sub_(lower)
    b_values = [v * 2.0**-lower for v in b_values] if experts else b_values * 2.0**-lower
    offsets, ends = offsets_of(torch, rows, experts, generator, 3) if experts else (None, None)
    plan = routing.Plan(offsets, None, None) if experts else None
    pair, magnitudes = reference(torch, a_values, b_values, ends)
    live, ran = pair.shape[0], 0
    gate, up = pair[:, :n], pair[:, n:]
    exact = torch.nn.functional.silu(gate) * up
    for name, y in kernels(kind):
        print(f"kernel {name} {size}", flush=True)
        dtype = getattr(torch, TYPES[y])
        u = torch.finfo(dtype).eps / 2
        off = sums(TYPES[y], k) * (1 + 2.0**-7) * magnitudes
        error = (1.1 * off[:, :n] * up.abs() + torch.nn.functional.silu(gate).abs() * off[:, n:]
                 + 1.1 * off[:, :n] * off[:, n:] + 8 * 2.0**-24 * exact.abs() + 2.0**-120)
        options = {"plan": plan, "sorted_rows": experts is not None, "kernel": name}
        if kind == "gated_fp8":
            packed = fp8.empty(rows, n)
            packed.codes.view(torch.uint8).fill_(3)
            packed.scales.fill_(9)
            fp8.gated(a, b, packed=packed, **options)
            values = fp8.dequantize(packed, torch.empty(rows, n, device="cuda")).double()[:live]
            blocks = -(-n // 128)
            scales = packed.scales.permute(1, 0, 2).reshape(rows, -1)
            scale = torch.exp2(scales[:live, :blocks].double() - 127).repeat_interleave(128, dim=1)[:, :n]
            allowed = error + 2.0**-4 * (exact.abs() + error) + 2.0**-10 * scale
            assert ((values - exact).abs() <= allowed).all(), name
            # The scale: the smallest that holds the block's largest, which is known to within the error.
            padded = torch.nn.functional.pad(torch.stack([exact.abs() - error, exact.abs() + error]),
                                             (0, blocks * 128 - n)).view(2, live, blocks, 128).amax(dim=3)
            assert (scale[:, ::128] * 448 >= padded[0]).all() and (scale[:, ::128] * 224 < padded[1]).all(), name
            codes = packed.codes.view(torch.uint8)
            assert not codes[:live, n:].any() and (codes[live:] == 3).all(), name
            assert (scales[:live, blocks:] == 127).all() and (scales[live:] == 9).all(), name
        else:
            out, kept = (torch.full((rows, width), 7.0, device="cuda", dtype=dtype) for width in (n, 2 * n))
            fp8.gated(a, b, out, gate_up=kept if kind == "gated_kept" else None, **options)
            bound = error + u * (exact.abs() + error) + floor(torch, dtype)
            assert ((out[:live].double() - exact).abs() <= bound).all(), name
            assert (out[live:] == 7).all(), name
            if kind == "gated_kept":
                bound = off + u * (pair.abs() + off) + floor(torch, dtype)
                assert ((kept[:live].double() - pair).abs() <= bound).all(), name
            assert (kept[live if kind == "gated_kept" else 0:] == 7).all(), name
        ran += 1
    assert ran >= (3 if kind == "gated_fp8" else 10)
