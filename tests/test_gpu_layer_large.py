"""Outputs past 32 MiB, which are stored (and, in columns, loaded) past the caches by kernels of their own: the same
bits as the same data in parts that the other kernels take, and the oracle's in sampled rows. Odd widths, rows off every
vector's alignment, rows and columns that end inside a tile."""

import numpy as np
import pytest

from oracle import mx as oracle_mx
from oracle import routing as oracle_routing

pytestmark = pytest.mark.gpu

LARGE = 32 << 20
UNIT = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}


def _random(torch, dtype, *shape, seed=0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    kind = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[dtype]
    return torch.randn(shape, device="cuda", generator=generator).to(kind)


def _host(tensor):
    return tensor.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_quantize_rows(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import mx

    rows, k = 16500, 4099
    print(f"large quantize {dtype} {rows}x{k}", flush=True)
    x = _random(torch, dtype, rows, k + 12, seed=1)[:, 3:k + 3]
    packed = mx.quantize(x)
    assert packed.codes.numel() > LARGE
    for first in range(0, rows, 5501):
        part = mx.quantize(x[first:first + 5501])
        assert part.codes.numel() < LARGE
        assert torch.equal(part.codes, packed.codes[first:first + 5501])
        assert torch.equal(part.scales, packed.scales[:, first:first + 5501])
    sample = [0, 1, 7777, rows - 1]
    codes, scales = oracle_mx.quantize(_host(x[sample]))
    assert np.array_equal(packed.codes[sample].cpu().numpy(), codes)
    assert np.array_equal(packed.scales[:, sample].cpu().numpy(), scales)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_quantize_columns(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import mx

    k, columns = 4099, 16501
    print(f"large quantize_columns {dtype} {k}x{columns}", flush=True)
    x = _random(torch, dtype, k, columns + 12, seed=2)[:, 3:columns + 3]
    packed = mx.quantize(x, columns=True)
    assert packed.codes.numel() > LARGE
    for first in range(0, columns, 5501):
        part = mx.quantize(x[:, first:first + 5501], columns=True)
        assert part.codes.numel() < LARGE
        assert torch.equal(part.codes, packed.codes[first:first + 5501])
        assert torch.equal(part.scales, packed.scales[:, first:first + 5501])
    sample = [0, 127, 128, 9001, columns - 1]
    codes, scales = oracle_mx.quantize(_host(x[:, sample]).T)
    assert np.array_equal(packed.codes[sample].cpu().numpy(), codes)
    assert np.array_equal(packed.scales[:, sample].cpu().numpy(), scales)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_linear_backward(gpu, dtype):
    """The gradient's one quantisation against the three calls, through the same products."""
    import torch

    from triton_chip_benchmarks_amd import mx

    rows, n, k = 4333, 5003, 8203  # operands of 11, 11 and 18 MiB
    print(f"large linear_backward {dtype} {rows}x{n}x{k}", flush=True)
    d_out = _random(torch, dtype, rows, n + 6, seed=3)[:, 3:n + 3]
    x = _random(torch, dtype, rows, k + 6, seed=4)[:, 1:k + 1]
    columns = mx.quantize(_random(torch, dtype, n, k, seed=5), columns=True)
    d_x, d_weight = mx.linear_backward(d_out, x, columns)
    parts = [mx.quantize(d_out), mx.quantize(d_out, columns=True), mx.quantize(x, columns=True)]
    assert sum(part.codes.numel() for part in parts) > LARGE > max(part.codes.numel() for part in parts)
    assert torch.equal(d_x, mx.product(parts[0], columns, dtype=x.dtype))
    assert torch.equal(d_weight, mx.product(parts[1], parts[2], dtype=x.dtype))
    sample = [0, 1, 2500, n - 1]
    expected, size = oracle_mx.linear(_host(d_out[:, sample]).T, _host(x).T)
    bound = (rows / 32 + 16) * 2.0**-23 * size
    assert (np.abs(_host(d_weight[sample]) - expected) <= bound + UNIT[dtype] * (np.abs(expected) + bound)
            + 2.0**-24).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_dequantize(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import mx

    rows, k = 4299, 4099
    print(f"large dequantize {dtype} {rows}x{k}", flush=True)
    packed = mx.quantize(_random(torch, "fp32", rows, k, seed=6))
    kind = _random(torch, dtype, 1).dtype
    out = torch.full((rows + 2, k), 7.0, device="cuda", dtype=kind)
    assert rows * k * out.element_size() > LARGE
    mx.dequantize(packed, out[1:-1])
    assert (out[0] == 7).all() and (out[-1] == 7).all()
    for first in range(0, rows, 1433):
        part = mx.Packed(packed.codes[first:first + 1433], packed.scales[:, first:first + 1433].contiguous(), k)
        values = mx.dequantize(part, torch.empty(1433, k, device="cuda", dtype=kind))
        assert torch.equal(values, out[1 + first:1 + first + 1433])
    sample = [0, 2222, rows - 1]
    exact = oracle_mx.values(packed.codes[sample].cpu().numpy(), packed.scales[:, sample].cpu().numpy(), k)
    # Of N(0, 1): nothing below fp16's smallest, and two significant bits in every type.
    assert np.array_equal(_host(out[1:-1][sample]), exact)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_combine_and_gradients(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import routing

    tokens, top, n = 4300, 3, 4099
    print(f"large combine {dtype} {tokens}x{top}x{n}", flush=True)
    half, rows = tokens // 2, tokens * top
    y, d_out = _random(torch, dtype, rows, n, seed=7), _random(torch, dtype, tokens, n, seed=8)
    weights = _random(torch, "fp32", tokens, top, seed=9)
    generator = torch.Generator().manual_seed(10)
    # The first tokens' rows are the first half of y's, so that a half is a smaller call of its own.
    slots = torch.cat([torch.randperm(rows // 2, generator=generator),
                       rows // 2 + torch.randperm(rows // 2, generator=generator)]).to(torch.int32).view(tokens, top)
    slots[5, 1] = slots[half, 0] = -1
    slots = slots.cuda()
    out = routing.combine(y, slots, weights)
    assert out.numel() * out.element_size() > LARGE
    d_y, d_weights = torch.full_like(y, 7.0), torch.empty_like(weights)
    routing.combine_backward(d_out, y, slots, weights, d_y, d_weights)
    parts = 2 if dtype != "fp32" else 3
    for first in range(0, tokens, -(-tokens // parts)):
        some = slice(first, min(first + -(-tokens // parts), tokens))
        part = routing.combine(y, slots[some].contiguous(), weights[some].contiguous())
        assert part.numel() * part.element_size() < LARGE and torch.equal(part, out[some])
    # Gradients of 400 tokens each, whose rows are gathered: their d_y is small.
    for first in (0, 1900, tokens - 400):
        named = slots[first:first + 400].reshape(-1)
        entries = torch.nonzero(named >= 0)[:, 0]
        local = torch.full_like(named, -1)
        local[entries] = torch.arange(len(entries), dtype=torch.int32, device="cuda")
        small_y, small_weights = routing.combine_backward(
            d_out[first:first + 400], y[named[entries].long()], local.view(400, top).contiguous(),
            weights[first:first + 400].contiguous())
        assert small_y.numel() * small_y.element_size() < LARGE
        assert torch.equal(small_y, d_y[named[entries].long()])
        assert torch.equal(small_weights, d_weights[first:first + 400])
    unnamed = torch.ones(rows, dtype=torch.bool, device="cuda")
    unnamed[slots[slots >= 0].long()] = False
    assert int(unnamed.sum()) == 2 and (d_y[unnamed] == 7).all()
    sample = [0, 5, half, tokens - 1]
    expected, size = oracle_routing.combine(_host(y), slots[sample].cpu().numpy(), _host(weights[sample]))
    bound = top * 2.0**-23 * size
    assert (np.abs(_host(out[sample]) - expected) <= bound + UNIT[dtype] * (np.abs(expected) + bound) + 2.0**-25).all()
    exact_y, exact_weights, size = oracle_routing.combine_backward(_host(d_out[sample]), _host(y),
                                                                   slots[sample].cpu().numpy(), _host(weights[sample]))
    assert (np.abs(_host(d_weights[sample]) - exact_weights) <= (n / 64 + 16) * 2.0**-23 * size).all()
    touched = np.unique(slots[sample].cpu().numpy())
    touched = touched[touched >= 0]
    assert (np.abs(_host(d_y[touched]) - exact_y[touched])
            <= (UNIT[dtype] + 2.0**-23) * np.abs(exact_y[touched]) + 2.0**-25).all()
