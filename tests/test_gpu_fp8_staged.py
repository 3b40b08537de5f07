"""The kernels of few rows that quantise fp32, fp16 or bf16 rows into LDS, each chosen by the rule for some size here: with
up to 16 rows of K about 5800 staged, 70 to 93 KiB of LDS, and with little of it. Against float64 products on the device.

Tolerances: sums to 2^-12 of the magnitudes where the output is not of fp32 (twice the matrix cores' worst), K 2^-24 of
them where it is; silu' is within 1.1, and its fp32 evaluation within eight roundings; then half a step of the output,
2^-4 for E4M3 (2^-10 of the scale below 2^-6 of it).
"""

import pytest

from triton_chip_benchmarks_amd import _native

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}
# (rows, n, K, experts) by kind and kernel; the first of each stages more than 64 KiB.
SIZES = {
    ("product", "1x4"): [(12, 1024, 5800, 8), (1, 4096, 1024, 1)],
    ("product", "1x8"): [(12, 16, 5800, 2), (1, 4096, 4096, 1), (16, 24, 700, 2)],
    ("product", "2x4"): [(12, 2048, 5800, 8), (1, 14336, 1024, 1)],
    ("gated", "2x4"): [(64, 100, 5800, 64), (1, 4096, 1024, 1)],
    ("gated", "2x8"): [(12, 16, 5800, 2), (1, 1024, 4096, 1)],
    ("gated_kept", "2x8"): [(12, 16, 5800, 2), (1, 1024, 4096, 1)],
    ("gated_fp8", "2x1"): [(32, 4096, 5800, 8), (1, 16, 16, 8)],
}
SIZES_32 = {("product", "1x4"): [(24, 512, 5800, 32), (1, 4096, 1024, 1)],
            ("gated", "2x4"): [(12, 1024, 5800, 8), (1, 4096, 1024, 1)]}


def staged_bytes(rows, k):
    """Codes and scales of the rows, pairs of blocks of each, a row a bank group past the one before."""
    blocks = -(-k // 256) * 2
    return min(rows, 16) * (blocks * 128 + 16 + blocks + 2)


def cases():
    for name in TYPES:
        for (kind, shape), sizes in ({**SIZES, **SIZES_32} if name == "f32" else SIZES).items():
            form = "e4m3" if kind == "gated_fp8" else name
            few = "gated" if kind == "gated_kept" else kind
            for size in sizes:
                yield name, kind, f"fp8_few_{few}_{name}_{form}_{shape}", size


def test_the_cases_reach_every_such_kernel_and_most_of_the_lds(gpu):
    reached = {kernel for _, _, kernel, _ in cases()}
    few = {name for name in _native.kernel_names() if name.startswith("fp8_few_")}
    assert reached == {name for name in few if name.split("_")[-3] != "e4m3"}  # X's type, Y's, the shape
    for _, _, kernel, _ in cases():
        assert max(staged_bytes(rows, k) for _, _, of, (rows, _, k, _) in cases() if of == kernel) > 64 * 1024, kernel
    assert staged_bytes(32, 5800) > 90 * 1024


def routes(torch, rows, experts, generator):
    """Tokens' choices, most of them expert 0's, some nobody's."""
    chosen = torch.randint(0, experts, (rows, 1), device="cuda", generator=generator, dtype=torch.int32)
    popular = torch.rand(rows, 1, device="cuda", generator=generator)
    chosen[popular < 0.7] = 0
    chosen[popular > 0.95] = -1
    return chosen


@pytest.mark.parametrize("name,kind,kernel,size", list(cases()), ids=str)
def test_staged_rows(gpu, name, kind, kernel, size):
    import torch

    from triton_chip_benchmarks_amd import fp8, routing

    rows, n, k, experts = size
    dtype = getattr(torch, TYPES[name])
    assert fp8.product_kernel(rows, n, k, dtype, experts, True, kind) == kernel
    print(f"kernel {kernel} {size}", flush=True)
    generator = torch.Generator(device="cuda").manual_seed(rows + n + k)
    width = n if kind == "product" else 2 * n
    channel = torch.where(torch.rand(k, device="cuda", generator=generator) < 0.05, 10.0, 1.0)
    # At a stride and an address of a few elements, as a slice of a wider tensor has.
    x = (torch.randn(rows, k + 11, device="cuda", generator=generator).to(dtype))[:, 3:k + 3]
    x.mul_(channel)
    weight = fp8.empty(width, k, fp8.BLOCK, experts=experts if experts > 1 else None)
    parts = [weight] if experts == 1 else [fp8.Packed(weight.codes[e], weight.scales[e], k, fp8.BLOCK)
                                           for e in range(experts)]
    for part in parts:
        fp8.quantize(torch.randn(width, k, device="cuda", generator=generator) / (2 * k**0.5), part, block=fp8.BLOCK)
    plan = None
    if experts > 1:
        chosen = routes(torch, rows, experts, generator)
        plan = routing.dispatch(chosen, experts)
    held = fp8.dequantize(fp8.quantize(x), torch.empty(rows, k, device="cuda")).double()
    live = rows if plan is None else int(plan.offsets[-1])
    exact, magnitudes = (torch.zeros(live, width, device="cuda", dtype=torch.float64) for _ in range(2))
    ends = [0, rows] if plan is None else plan.offsets.tolist()
    for part, first, last in zip(parts, ends, ends[1:]):
        if last > first:
            mine = held if plan is None else held[plan.order[first:last].long()]
            w = fp8.dequantize(part, torch.empty(width, k, device="cuda")).double().t().contiguous()
            exact[first:last], magnitudes[first:last] = mine @ w, mine.abs() @ w.abs()
    info = torch.finfo(dtype)
    u, floor = info.eps / 2, info.smallest_normal * info.eps / 2
    off = (k * 2.0**-24 if name == "f32" and kind != "gated_fp8" else 2.0**-12) * (1 + 2.0**-7) * magnitudes
    calls = [{}] if plan is None else [{"plan": plan}, {"plan": plan, "sorted_rows": True}]
    for options in calls:
        given = x
        if options.get("sorted_rows"):
            given = torch.zeros_like(x)
            given[:live] = x[plan.order[:live].long()]
        if kind == "product":
            out = torch.full((rows, n), 7.0, device="cuda", dtype=dtype)
            fp8.linear(given, weight, out, **options)
            assert ((out[:live].double() - exact).abs() <= off + u * (exact.abs() + off) + floor).all()
            assert (out[live:] == 7).all()
            continue
        gate, up = exact[:, :n], exact[:, n:]
        value = torch.nn.functional.silu(gate) * up
        error = (1.1 * off[:, :n] * up.abs() + torch.nn.functional.silu(gate).abs() * off[:, n:]
                 + 1.1 * off[:, :n] * off[:, n:] + 8 * 2.0**-24 * value.abs() + 2.0**-120)
        if kind != "gated_fp8":
            out, kept = (torch.full((rows, w), 7.0, device="cuda", dtype=dtype) for w in (n, 2 * n))
            fp8.gated(given, weight, out, gate_up=kept if kind == "gated_kept" else None, **options)
            assert ((out[:live].double() - value).abs() <= error + u * (value.abs() + error) + floor).all()
            assert (out[live:] == 7).all()
            if kind == "gated_kept":
                assert ((kept[:live].double() - exact).abs() <= off + u * (exact.abs() + off) + floor).all()
                assert (kept[live:] == 7).all()
            continue
        packed = fp8.empty(rows, n)
        packed.codes.view(torch.uint8).fill_(3)
        packed.scales.fill_(9)
        fp8.gated(given, weight, packed=packed, **options)
        got = fp8.dequantize(packed, torch.empty(rows, n, device="cuda")).double()[:live]
        scales = packed.scales.permute(1, 0, 2).reshape(rows, -1)
        scale = torch.exp2(scales[:live].double() - 127).repeat_interleave(128, dim=1)[:, :n]
        assert ((got - value).abs() <= error + 2.0**-4 * (value.abs() + error) + 2.0**-10 * scale).all()
        assert (packed.codes.view(torch.uint8)[live:] == 3).all() and (scales[live:] == 9).all()
