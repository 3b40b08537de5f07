"""MX quantisation and the MXFP4 linear layer on the GPU against the float64 oracle.

Codes and scales are exact. A product sums K exact terms in fp32: at most one rounding to 2^-23 of the magnitudes'
sum for each of the K / 32 instruction steps, the terms inside a step and the joins of partial sums (K / 32 + 16 in
all), then one rounding to the output type.
"""

import numpy as np
import pytest

from oracle import mx as oracle

pytestmark = pytest.mark.gpu

UNIT = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}


def _dtype(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def _random(torch, dtype, *shape, seed=0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=generator).to(_dtype(torch, dtype))


def _host(tensor):
    return tensor.double().cpu().numpy()


def _check_operand(packed, x):
    codes, scales = oracle.quantize(x)
    assert np.array_equal(packed.scales.cpu().numpy(), scales)
    assert np.array_equal(packed.codes.cpu().numpy(), codes)


def _check_product(got, expected, size, dtype, k):
    bound = (k / 32 + 16) * 2.0**-23 * size
    tiny = {"fp32": 2.0**-149, "fp16": 2.0**-24, "bf16": 2.0**-133}[dtype]
    error = np.abs(_host(got) - expected)
    assert (error <= bound + UNIT[dtype] * (np.abs(expected) + bound) + tiny).all(), error.max()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (5, 33), (33, 255), (64, 256), (7, 264), (130, 1000)])
@pytest.mark.parametrize("columns", [False, True])
def test_quantize_is_exact(gpu, dtype, rows, k, columns):
    import torch

    from triton_chip_benchmarks_amd import mx

    print(f"quantize {dtype} {rows}x{k} columns={columns}", flush=True)
    x = _random(torch, dtype, rows, k, seed=rows + k)
    x[:, k // 2:] *= 37
    packed = mx.quantize(x, columns=columns)
    _check_operand(packed, _host(x).T if columns else _host(x))
    values = mx.dequantize(packed)
    assert np.array_equal(_host(values), oracle.rounded(_host(x).T if columns else _host(x)))
    if dtype == "fp32":
        assert np.array_equal(_host(mx.dequantize(packed, torch.empty(values.shape, device="cuda"))), _host(values))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("columns", [False, True])
def test_every_16_bit_value_is_quantised_exactly(gpu, dtype, columns):
    """All 65536 bit patterns as one group member beside a largest magnitude of 1, 2^-6 and none, NaN and infinities
    included."""
    import torch

    from triton_chip_benchmarks_amd import mx

    bits = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(_dtype(torch, dtype)).cuda()
    for largest in (0.0, 1.0, 2.0**-6):
        x = torch.zeros(65536 // 8, 8, 32, device="cuda", dtype=bits.dtype)
        x[:, :, 5] = bits.view(-1, 8)
        x[:, :, 17] = largest
        x = x.view(-1, 256)
        x = x.t().contiguous() if columns else x
        packed = mx.quantize(x, columns=columns)
        _check_operand(packed, _host(x).T if columns else _host(x))
        expected = oracle.rounded(_host(x).T if columns else _host(x))
        assert np.array_equal(_host(mx.dequantize(packed)), expected, equal_nan=True)


def test_fp32_extremes_are_quantised_exactly(gpu):
    import torch

    from triton_chip_benchmarks_amd import mx

    powers = torch.arange(-149, 128, dtype=torch.float64)
    x = torch.zeros(277, 64, dtype=torch.float64)
    x[:, 0] = 2.0**powers * 1.75
    x[:, 1] = -(2.0**(powers - 2)) * 1.25  # a tie in every scale
    x[:, 40] = 2.0**powers
    x[:, 41] = (2.0**powers) * 0.624999
    x = x.float().cuda()
    x[5, 3], x[6, 63], x[7, 0] = float("nan"), float("inf"), -0.0
    _check_operand(mx.quantize(x), _host(x))
    assert np.array_equal(_host(mx.dequantize(mx.quantize(x))), oracle.rounded(_host(x)), equal_nan=True)


def test_strides_offsets_and_other_streams(gpu):
    import torch

    from triton_chip_benchmarks_amd import mx

    wide = _random(torch, "bf16", 40, 301, seed=3)
    x = wide[3:36, 5:250]  # rows off every vector's alignment
    _check_operand(mx.quantize(x), _host(x))
    _check_operand(mx.quantize(x, columns=True), _host(x).T)
    repeated = wide[2:3, :100].expand(9, 100)  # a row stride of zero
    _check_operand(mx.quantize(repeated), _host(repeated))
    weight = mx.quantize(_random(torch, "bf16", 50, 245, seed=4))
    expected = mx.linear(x.contiguous(), weight)
    assert torch.equal(mx.linear(x, weight), expected)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mx.linear(x, weight)
    side.synchronize()
    assert torch.equal(got, expected)


SHAPES = [(1, 64, 64), (1, 1, 1), (2, 17, 33), (15, 48, 1000), (16, 130, 256), (17, 64, 4096), (33, 200, 288),
          (64, 64, 512), (65, 129, 100), (128, 256, 768), (200, 333, 1111), (257, 512, 2048), (1000, 744, 1000)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_linear(gpu, dtype, rows, n, k):
    import torch

    from triton_chip_benchmarks_amd import mx

    print(f"linear {dtype} {rows}x{n}x{k}", flush=True)
    x = _random(torch, dtype, rows, k, seed=1)
    w = _random(torch, dtype, n, k, seed=2)
    out = torch.full((rows, n), float("nan"), device="cuda", dtype=x.dtype)
    weight = mx.quantize(w)
    mx.linear(x, weight, out)
    expected, size = oracle.linear(_host(x), _host(w))
    _check_product(out, expected, size, dtype, k)
    again = mx.product(mx.quantize(x), weight, dtype=x.dtype)
    _check_product(again, expected, size, dtype, k)


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_groups_that_are_not_finite_reach_their_rows_only(gpu, rows):
    import torch

    from triton_chip_benchmarks_amd import mx

    x, w = _random(torch, "bf16", rows, 320, seed=5), _random(torch, "bf16", 70, 320, seed=6)
    x[rows // 2, 318], w[69, 0] = float("inf"), float("nan")
    out = mx.linear(x, mx.quantize(w))
    expected, _ = oracle.linear(_host(x), _host(w))
    assert np.array_equal(np.isnan(_host(out)), np.isnan(expected))


def test_scales_of_every_magnitude(gpu):
    import torch

    from triton_chip_benchmarks_amd import mx

    for rows in (4, 100):
        x = _random(torch, "fp32", rows, 512, seed=7) * 2.0 ** torch.randint(-60, 60, (rows, 1), device="cuda").float()
        w = _random(torch, "fp32", 96, 512, seed=8) * 2.0 ** torch.randint(-60, 60, (96, 1), device="cuda").float()
        x[:, 64:96] *= 2.0**-50
        x[1], w[3] = 0, 0
        expected, size = oracle.linear(_host(x), _host(w))
        _check_product(mx.linear(x, mx.quantize(w)), expected, size, "fp32", 512)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k", [(1, 40, 70), (33, 64, 96), (100, 257, 130), (513, 300, 384)])
def test_linear_backward(gpu, dtype, rows, n, k):
    import torch

    from triton_chip_benchmarks_amd import mx

    print(f"linear_backward {dtype} {rows}x{n}x{k}", flush=True)
    x, w, g = (_random(torch, dtype, *s, seed=i) for i, s in enumerate(((rows, k), (n, k), (rows, n))))
    d_x, d_weight = mx.linear_backward(g, x, mx.quantize(w, columns=True))
    (ex, sx), (ew, sw) = oracle.linear_backward(_host(g), _host(x), _host(w))
    _check_product(d_x, ex, sx, dtype, n)
    _check_product(d_weight, ew, sw, dtype, rows)


def test_linear_gradient_is_the_difference_where_quantisation_changes_nothing(gpu):
    """On E2M1's lattice with every scale 2^0 the layer is its product and every sum exact, so one element's step
    changes the loss by its gradient times the step, bit for bit."""
    import torch

    from triton_chip_benchmarks_amd import mx

    generator = torch.Generator().manual_seed(9)
    lattice = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -1, -1.5, -2, -3, -4, -6])
    x, w, g = (lattice[torch.randint(0, 15, s, generator=generator)].cuda() for s in ((64, 96), (160, 96), (64, 160)))
    for m in (x, w, g):
        m[::32], m[:, ::32] = 6, 6
    d_x, d_w = mx.linear_backward(g, x, mx.quantize(w, columns=True))
    loss = lambda x, w: (g.double() * mx.linear(x, mx.quantize(w)).double()).sum().item()  # noqa: E731
    start = loss(x, w)
    for r, c in ((5, 7), (63, 95), (33, 41)):
        for moved, d, value in ((x.clone(), d_x, 3.0), (w.clone(), d_w, -1.5)):
            step = value - moved[r, c].item()
            moved[r, c] = value
            after = loss(moved, w) if d is d_x else loss(x, moved)
            assert after - start == d[r, c].item() * step


PLANS = [(1, 1, 4), (1, 3, 8), (5, 2, 3), (40, 2, 8), (64, 4, 7), (300, 2, 4), (700, 3, 5)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("tokens,top,experts", PLANS)
def test_experts(gpu, dtype, tokens, top, experts):
    """Routed rows through their own weights; entries without an expert, experts without a row, one with most."""
    import torch

    from triton_chip_benchmarks_amd import mx, routing

    print(f"experts {dtype} {tokens} of {top} x {experts}", flush=True)
    n, k = 136, 416
    x, w = _random(torch, dtype, tokens, k, seed=1), _random(torch, dtype, experts, n, k, seed=2)
    rng = np.random.default_rng(tokens)
    chosen = rng.integers(-1, experts, (tokens, top)).astype(np.int32)
    chosen[tokens // 2:] = experts - 1  # most rows to the last one, the same choice twice included
    if experts > 2:
        chosen[chosen == 1] = 0  # and none to expert 1
    plan = routing.dispatch(torch.tensor(chosen).cuda(), experts)
    weight = mx.empty(n, k, experts=experts)
    for e in range(experts):
        mx.quantize(w[e], mx.Packed(weight.codes[e], weight.scales[e], k))
    out = torch.full((tokens * top, n), 7.0, device="cuda", dtype=x.dtype)
    mx.linear(x, weight, out, plan=plan)
    offsets, order = plan.offsets.tolist(), plan.order.cpu().numpy()
    host = _host(x)
    sorted_x = torch.zeros(tokens * top, k, device="cuda", dtype=x.dtype)
    for e in range(experts):
        rows = order[offsets[e]:offsets[e + 1]]
        assert (chosen.reshape(-1)[rows] == e).all()
        if len(rows):
            expected, size = oracle.linear(host[rows // top], _host(w[e]))
            _check_product(out[offsets[e]:offsets[e + 1]], expected, size, dtype, k)
            sorted_x[offsets[e]:offsets[e + 1]] = x[torch.tensor(rows // top).cuda().long()]
    assert (out[offsets[-1]:] == 7).all()  # rows of no expert are not written
    again = torch.full_like(out, 7.0)
    mx.linear(sorted_x, weight, again, plan=plan, sorted_rows=True)
    assert torch.equal(again, out)


# Sizes that run on every kernel of the products (256x128, 128x64 and 64x64 tiles, one or many a workgroup): K of one
# step, of an odd number and with a last one in part, n off the pieces of 16 bytes, more tiles than places.
TILED = [(4100, 4104, 1100), (2600, 3001, 300), (700, 2049, 255), (3000, 515, 5000), (130, 8190, 1056),
         (20, 1000, 40), (90, 300, 7000), (9000, 131, 513)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,n,k", TILED)
def test_products_of_many_tiles(gpu, dtype, rows, n, k):
    """Against float64 on the device, from operands that the oracle's rules fix; twice, to the same bits."""
    import torch

    from triton_chip_benchmarks_amd import mx

    print(f"product {dtype} {rows}x{n}x{k}", flush=True)
    a, b = mx.quantize(_random(torch, dtype, rows, k, seed=1)), mx.quantize(_random(torch, dtype, n, k, seed=2))
    va, vb = mx.dequantize(a).double(), mx.dequantize(b).double()
    out = torch.full((rows, n), float("nan"), device="cuda", dtype=_dtype(torch, dtype))
    mx.product(a, b, out)
    expected, size = va @ vb.t().contiguous(), va.abs() @ vb.abs().t().contiguous()
    bound = (k / 32 + 16) * 2.0**-23 * size
    error = (out.double() - expected).abs()
    assert bool((error <= bound + UNIT[dtype] * (expected.abs() + bound) + 2.0**-24).all()), error.max()
    assert torch.equal(mx.product(a, b, dtype=out.dtype), out)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,experts,n,k", [(5000, 8, 1030, 600), (3000, 60, 264, 1025), (2000, 256, 136, 260),
                                              (1500, 300, 72, 96), (4000, 4, 2056, 2300)])
def test_products_of_many_experts(gpu, dtype, rows, experts, n, k):
    """Uneven experts, some without a row; more of them than a wave's table holds; the rows behind stay."""
    import torch

    from triton_chip_benchmarks_amd import mx

    print(f"product {dtype} {rows} of {experts} x {n}x{k}", flush=True)
    generator = torch.Generator(device="cuda").manual_seed(experts)
    share = torch.rand(experts, device="cuda", generator=generator) ** 4
    share[1] = 0
    counts = (share / share.sum() * (rows - 5)).long()
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    a = mx.quantize(_random(torch, dtype, rows, k, seed=1))
    weights = [mx.quantize(_random(torch, dtype, n, k, seed=10 + e)) for e in range(experts)]
    b = mx.Packed(torch.stack([w.codes for w in weights]), torch.stack([w.scales for w in weights]), k)
    out = torch.full((rows, n), 7.0, device="cuda", dtype=_dtype(torch, dtype))
    mx.product(a, b, out, offsets=offsets)
    va, ends = mx.dequantize(a).double(), offsets.tolist()
    for e in range(experts):
        first, last = ends[e], ends[e + 1]
        if last > first:
            vb = mx.dequantize(weights[e]).double()
            expected = va[first:last] @ vb.t().contiguous()
            bound = (k / 32 + 16) * 2.0**-23 * (va[first:last].abs() @ vb.abs().t().contiguous())
            error = (out[first:last].double() - expected).abs()
            assert bool((error <= bound + UNIT[dtype] * (expected.abs() + bound) + 2.0**-24).all()), (e, error.max())
    assert (out[ends[-1]:] == 7).all()


def test_offsets_that_are_out_of_order_write_nothing_outside(gpu):
    """Offsets past the rows, negative or falling are clamped: whatever lands in the output, nothing else is touched."""
    import torch

    from triton_chip_benchmarks_amd import mx

    for rows in (8, 300):
        guarded = torch.full((rows + 200, 64), 7.0, device="cuda", dtype=torch.bfloat16)
        a = mx.quantize(_random(torch, "bf16", rows, 96, seed=1))
        b = mx.empty(64, 96, experts=4)
        b.codes.zero_()
        b.scales.fill_(127)
        for offsets in ([0, -5, 10**6, 3, 2**31 - 1], [rows, 0, rows, 0, rows], [10**6] * 5):
            mx.product(a, b, guarded[100:100 + rows], offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"))
            torch.cuda.synchronize()
            assert (guarded[:100] == 7).all() and (guarded[100 + rows:] == 7).all()


def test_a_weight_whose_scales_pass_32_bit_offsets(gpu):
    """2^20 features of 257 K steps: 2.2 GB of scales, beyond the tiles' offsets."""
    import torch

    from triton_chip_benchmarks_amd import mx

    n, k = 1 << 20, 257 * 256
    b = mx.Packed(torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda"),
                  torch.full((k // 256, n, 8), 127, dtype=torch.uint8, device="cuda"), k)
    b.codes[n - 3] = 0x22  # ones
    b.scales[256, n - 3] = 128  # twos in the last step
    a = mx.quantize(torch.ones(17, k, device="cuda", dtype=torch.bfloat16))
    out = mx.product(a, b, dtype=torch.float32)
    assert (out[:, n - 3] == k + 256).all() and int(torch.count_nonzero(out)) == 17


def test_empty_calls(gpu):
    import torch

    from triton_chip_benchmarks_amd import mx, routing

    weight = mx.quantize(_random(torch, "bf16", 8, 64))
    none = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    assert mx.linear(none, weight).shape == (0, 8)
    assert mx.quantize(none).codes.shape == (0, 32)
    plan = routing.dispatch(torch.empty(0, 2, device="cuda", dtype=torch.int32), 3)
    assert plan.offsets.tolist() == [0, 0, 0, 0]
    d_x, d_weight = mx.linear_backward(torch.empty(0, 8, device="cuda", dtype=torch.bfloat16), none,
                                       mx.empty(64, 8))
    assert d_x.shape == (0, 64) and not d_weight.any()


def test_a_weight_past_32_bit_offsets(gpu):
    """The last of many experts lies past 2^32 bytes of codes: its rows meet its own weight."""
    import torch

    from triton_chip_benchmarks_amd import mx, routing

    experts, n, k = 40, 8192, 32768  # 5 GiB of codes
    weight = mx.Packed(torch.zeros(experts, n, k // 2, dtype=torch.uint8, device="cuda"),
                       torch.full((experts, k // 256, n, 8), 127, dtype=torch.uint8, device="cuda"), k)
    weight.codes[experts - 1] = 0x22  # all ones
    weight.codes[experts - 1, n - 1] = 0x44  # all twos
    for tokens in (1, 40):
        x = torch.ones(tokens, k, device="cuda", dtype=torch.bfloat16)
        plan = routing.dispatch(torch.full((tokens, 1), experts - 1, device="cuda", dtype=torch.int32), experts)
        out = mx.linear(x, weight, plan=plan)
        assert (out[:, :-1] == k).all() and (out[:, -1] == 2 * k).all()
