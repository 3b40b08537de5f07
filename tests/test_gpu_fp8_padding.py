"""The gated pair to an FP8 operand where the columns end inside a tile: what lies past them is nobody's, so a block of the
weight that is not finite makes NaN of the output's blocks that hold its own columns, and of no other."""

import pytest

from triton_chip_benchmarks_amd import _native

pytestmark = pytest.mark.gpu

KERNELS = [name for name in _native.kernel_names() if name.startswith(("fp8_few_gated_fp8_e4m3_", "fp8_tiles_gated_fp8_"))]

# n, K, rows of a weight's scale, and the element of W [2n][K] that is not finite. Past the gates' rows of W lie the ups',
# past the ups' scales of a step of 512 elements those of the next step's first rows.
CASES = [(200, 300, 1, 205, 7), (200, 300, 1, 399, 130), (129, 300, 1, 200, 299), (200, 1100, 1, 3, 600),
         (129, 1100, 128, 3, 600), (136, 1536, 128, 100, 1030)]


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("n,k,block,row,column", CASES)
def test_a_block_that_is_not_finite_stays_in_its_columns(gpu, n, k, block, row, column, value):
    import torch

    from triton_chip_benchmarks_amd import fp8

    rows = 70
    generator = torch.Generator(device="cuda").manual_seed(n + k)
    w = torch.randn(2 * n, k, device="cuda", generator=generator) / k**0.5
    bad = w.clone()
    bad[row, column] = value
    x = fp8.quantize(torch.randn(rows, k, device="cuda", generator=generator))
    first = row // block * block
    hit = {r % n // 128 for r in range(first, min(first + block, 2 * n))}
    assert len(hit) < -(-n // 128)
    for name in KERNELS:
        print(f"kernel {name} {n}x{k}", flush=True)
        clean, broken = (fp8.gated(x, fp8.quantize(weight, block=block), packed=fp8.empty(rows, n), kernel=name)
                         for weight in (w, bad))
        for b in range(-(-n // 128)):
            codes, expected = (p.codes.view(torch.uint8)[:, 128 * b:128 * (b + 1)] for p in (broken, clean))
            scales, expected_scales = (p.scales[0, :, b] for p in (broken, clean))
            if b in hit:
                assert (scales == 255).all() and not codes.any(), (name, b)
            else:
                assert torch.equal(scales, expected_scales) and torch.equal(codes, expected), (name, b)
        for packed in (clean, broken):
            assert not packed.codes.view(torch.uint8)[:, n:].any(), name
    assert len(KERNELS) == 4
