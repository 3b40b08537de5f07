"""FP8 quantisation with block scales against the float64 oracle: codes and scales bit for bit."""

import numpy as np
import pytest

from oracle import fp8 as oracle

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


def tensor(torch, values, dtype):
    return torch.tensor(values, dtype=torch.float32).to(getattr(torch, dtype)).cuda()


def host(t):
    return t.detach().cpu().double().numpy()


def operand(packed):
    import torch

    return packed.codes.view(torch.uint8).cpu().numpy(), packed.scales.cpu().numpy()


def check(packed, x, block=1):
    codes, scales = operand(packed)
    expected_codes, expected_scales = oracle.quantize(x, block)
    np.testing.assert_array_equal(scales, expected_scales)
    np.testing.assert_array_equal(codes, expected_codes)


def random(rows, k, seed, spread=20):
    """Values over many binades, some rows and columns far larger than others, zeros among them."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-spread // 2, spread // 2, (1, k)))
    x *= np.exp2(rng.integers(-4, 5, (rows, 1)))
    x[rng.random((rows, k)) < 0.1] = 0.0
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 15), (5, 129), (7, 513), (129, 1000), (2, 4112), (300, 272)])
def test_rows_columns_and_blocks(gpu, dtype, rows, k):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x = tensor(torch, random(rows, k, rows * 131 + k), dtype)
    exact = host(x)
    check(fp8.quantize(x), exact)
    check(fp8.quantize(x, columns=True), exact.T)
    check(fp8.quantize(x, block=128), exact, 128)
    check(fp8.quantize(x, columns=True, block=128), exact.T, 128)
    for block in (1, 128):
        by_rows, by_columns = fp8.quantize_both(x, block=block)
        check(by_rows, exact, block)
        check(by_columns, exact.T, block)


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code_and_its_ties(gpu, dtype):
    """A block for each of E4M3's magnitudes and the midpoints between them (all exact in 16 bits), with 448 to fix the
    scale at 1; then their negatives; then under a scale of 2^-3."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    middles = (oracle.GRID[1:] + oracle.GRID[:-1]) / 2
    points = np.concatenate([oracle.GRID, middles])
    x = np.zeros((len(points), 128))
    x[:, 0], x[:, 5], x[:, 77] = 448.0, points, -points
    for scale in (1.0, 0.125):
        given = tensor(torch, x * scale, dtype)
        np.testing.assert_array_equal(host(given), x * scale)
        check(fp8.quantize(given), x * scale)
        check(fp8.quantize(given, columns=True), (x * scale).T)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_at_their_borders(gpu, dtype):
    """Largest magnitudes at, below and above 448 * 2^e, at both ends of the type, and of nothing but zeros."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    info = torch.finfo(getattr(torch, dtype))
    eps = info.eps
    largest = [448.0, 448 * (1 + eps), 448 * (1 - eps), 1.0, 1.75, 1.75 * (1 + eps), 2.0, info.max, info.tiny,
               info.smallest_normal * info.eps, 0.0, 449.0, 447.0, 512.0]
    x = np.zeros((len(largest), 128))
    x[:, 3], x[:, 100] = largest, -0.3 * np.array(largest)
    given = tensor(torch, x, dtype)
    check(fp8.quantize(given), host(given))
    check(fp8.quantize(given, columns=True), host(given).T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_blocks_that_are_not_finite(gpu, dtype, bad):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x = random(140, 300, 5, spread=8)
    x[3, 140] = bad
    given = tensor(torch, x, dtype)
    x = host(given)
    for block in (1, 128):
        by_rows, by_columns = fp8.quantize_both(given, block=block)
        check(by_rows, x, block)
        check(by_columns, x.T, block)
    values = fp8.dequantize(fp8.quantize(given))
    assert torch.isnan(values[3, 128:256]).all() and torch.isfinite(values[3, :128]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_offsets(gpu, dtype):
    """Rows at an odd stride, from an odd element on; a row repeated by a stride of 0."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    whole = tensor(torch, random(70, 333, 9), dtype)
    for x in (whole[1:, 3:300], whole[::3, 1:130], whole[4:5].expand(60, -1)):
        for block in (1, 128):
            check(fp8.quantize(x, block=block), host(x), block)
            check(fp8.quantize(x, columns=True, block=block), host(x).T, block)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [1, 128])
def test_dequantize(gpu, dtype, block):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x = random(150, 700, 3, spread=8)
    packed = fp8.quantize(tensor(torch, x, "float32"), block=block)
    out = fp8.dequantize(packed, torch.empty(150, 700, device="cuda", dtype=getattr(torch, dtype)))
    exact = oracle.values(*operand(packed), 700, block)
    assert torch.equal(out.cpu(), torch.tensor(exact).to(out.dtype))


def test_large_outputs_and_empty_ones(gpu):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x = torch.randn(9000, 4100, device="cuda").bfloat16()  # 36.9 MB of codes: past the streamed stores' border
    packed = fp8.quantize(x)
    rows = [0, 1, 4500, 8999]
    codes, scales = operand(packed)
    expected_codes, expected_scales = oracle.quantize(host(x[rows]))
    np.testing.assert_array_equal(codes[rows], expected_codes)
    np.testing.assert_array_equal(scales[:, rows], expected_scales)
    both = fp8.quantize_both(x)
    assert torch.equal(both[0].codes.view(torch.uint8), packed.codes.view(torch.uint8))
    assert torch.equal(both[0].scales, packed.scales)
    columns = [0, 7, 2049, 4099]
    codes, scales = operand(both[1])
    expected_codes, expected_scales = oracle.quantize(host(x[:, columns]).T)
    np.testing.assert_array_equal(codes[columns], expected_codes)
    np.testing.assert_array_equal(scales[:, columns], expected_scales)
    values = fp8.dequantize(packed, torch.empty(9000, 4100, device="cuda"))
    exact = oracle.values(*oracle.quantize(host(x[rows])), 4100)
    np.testing.assert_array_equal(host(values[rows]), exact)
    for shape in ((0, 64), (64, 0), (0, 0)):
        empty = torch.empty(shape, device="cuda")
        for block in (1, 128):
            fp8.quantize_both(empty, block=block)
        assert fp8.dequantize(fp8.quantize(empty)).shape == shape
