"""CPU checks of which kernel an FP8 product runs on: every one is the choice for some size."""

import pytest
import torch

from triton_chip_benchmarks_amd import _native, fp8

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# (rows, n, k, experts) of each kernel of an output type, by the kind of product; of few rows, X a tensor or an operand.
FEW = {
    "product": {"1x4": (1, 4096, 1024, 1), "1x8": (1, 4096, 4096, 1), "2x4": (1, 14336, 1024, 1)},
    "gated": {"2x4": (1, 4096, 1024, 1), "2x8": (1, 1024, 4096, 1)},
    "gated_fp8": {"2x1": (1, 16, 16, 8)},
}
TILES = {
    "product": {"64x64": (21391, 34, 20, 8), "128x64": (36, 3541, 19, 128), "128x128": (22859, 96, 18, 1),
                "256x128": (2545, 1704, 16, 8), "256x256": (2850, 3080, 16, 8)},
    "gated": {"256x64": (6, 10559, 18, 128), "256x128": (18037, 36, 18, 1), "256x256": (12177, 412, 17, 8)},
    "gated_kept": {"256x64": (688, 1000, 17, 32), "256x128": (15907, 72, 18, 32), "256x256": (2545, 1704, 16, 8)},
    "gated_fp8": {"256x64": (1, 19, 524, 1), "256x128": (15640, 16, 16, 32), "256x256": (16399, 134, 19, 32)},
}
TILES_32 = {
    "product": {"64x64": (18037, 36, 18, 1), "128x64": (31, 7921, 24, 128), "128x128": (4028, 862, 16, 32),
                "256x128": (9225, 335, 18, 128)},
    "gated": {"256x64": (24, 11380, 20, 128)}, "gated_kept": {"256x64": (5609, 120, 18, 1)},
}


def _choices(name):
    dtype = DTYPES[name]
    tiles = TILES_32 if name == "f32" else TILES
    for kind, sizes in tiles.items():
        form = "e4m3" if kind == "gated_fp8" else name
        for tile, (rows, n, k, experts) in sizes.items():
            yield f"fp8_tiles_{kind}_{form}_{tile}", fp8.product_kernel(rows, n, k, dtype, experts, False, kind)
    for kind, sizes in FEW.items():
        form = "e4m3" if kind == "gated_fp8" else name
        for shape, (rows, n, k, experts) in sizes.items():
            yield f"fp8_few_{kind}_{name}_{form}_{shape}", fp8.product_kernel(rows, n, k, dtype, experts, True, kind)
            yield f"fp8_few_{kind}_e4m3_{form}_{shape}", fp8.product_kernel(rows, n, k, dtype, experts, False, kind)
            if kind == "gated":  # of few rows the same kernels keep the gate and up
                yield (f"fp8_few_{kind}_e4m3_{form}_{shape}",
                       fp8.product_kernel(rows, n, k, dtype, experts, False, "gated_kept"))


@pytest.mark.parametrize("name", sorted(DTYPES))
def test_every_kernel_is_some_sizes_choice(name):
    chosen = set()
    for expected, got in _choices(name):
        assert got == expected
        chosen.add(got)
    kernels = {kernel for kernel in _native.kernel_names() if kernel.startswith(("fp8_few_", "fp8_tiles_"))}
    mine = {kernel for kernel in kernels if kernel.rsplit("_", 2)[1] == name
            or (kernel.rsplit("_", 2)[1] == "e4m3" and f"_{name}_e4m3" in kernel)}
    assert mine <= chosen and (name == "f32" or {kernel for kernel in kernels if "gated_fp8_e4m3" in kernel} <= chosen)


def test_sizes_past_a_kernels_limits_take_another():
    # 2^24 - 1 workgroups a launch, 4096 experts for the kernels of few rows, and codes of 16 rows in 96 KiB of LDS.
    assert fp8.product_kernel(8, 64, 64, experts=4096).startswith("fp8_few_")
    assert fp8.product_kernel(16, 64, 8192, linear=True).endswith("e4m3_bf16_1x8")
    assert "bf16_bf16" in fp8.product_kernel(1, 64, 8192, linear=True)
