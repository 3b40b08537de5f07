"""CPU checks of which kernel an FP8 product runs on: every one is the choice for some size."""

import pytest
import torch

from triton_chip_benchmarks_amd import _native, fp8

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# (rows, n, k, experts, of a tensor) of each kernel of an output type, by the kind of product.
FEW = {
    "product": {"1x8": (1, 16, 16, 8, True), "2x4": (64, 1408, 2048, 64, True), "2x8": (12000, 22, 20, 400, True)},
    "gated": {"2x4": (444, 17, 16, 400, True), "2x8": (1, 16, 16, 8, True)},
}
TILES = {
    "product": {"64x64": (1, 17, 18, 1), "128x64": (27, 1248, 16, 128), "128x128": (22859, 96, 18, 1),
                "256x128": (2545, 1704, 16, 8), "256x256": (2850, 3080, 16, 8)},
    "gated": {"256x64": (5, 4222, 18, 32), "256x128": (15640, 16, 16, 32), "256x256": (12177, 412, 17, 8)},
    "gated_kept": {"256x64": (7, 4166, 17, 128), "256x128": (16462, 34, 16, 8), "256x256": (2545, 1704, 16, 8)},
    "gated_fp8": {"256x64": (3, 4655, 126, 128), "256x128": (15640, 16, 16, 32), "256x256": (16399, 134, 19, 32)},
}
TILES_32 = {
    "product": {"64x64": (1, 16, 16, 8), "128x64": (27, 1248, 16, 128), "128x128": (4028, 862, 16, 32),
                "256x128": (9225, 335, 18, 128)},
    "gated": {"256x64": (5, 4222, 18, 32)}, "gated_kept": {"256x64": (11, 2676, 16, 32)},
}


def _choices(name):
    dtype = DTYPES[name]
    tiles = TILES_32 if name == "f32" else TILES
    for kind, sizes in tiles.items():
        form = "e4m3" if kind == "gated_fp8" else name
        for tile, (rows, n, k, experts) in sizes.items():
            yield f"fp8_tiles_{kind}_{form}_{tile}", fp8.product_kernel(rows, n, k, dtype, experts, False, kind)
    for kind, sizes in FEW.items():
        for shape, (rows, n, k, experts, _) in sizes.items():
            yield (f"fp8_few_{kind}_{name}_{name}_{shape}",
                   fp8.product_kernel(rows, n, k, dtype, experts, True, kind))
    yield f"fp8_few_gated_fp8_{name}_e4m3_2x1", fp8.product_kernel(1, 16, 16, dtype, 8, True, "gated_fp8")
    yield "fp8_few_gated_fp8_e4m3_e4m3_2x1", fp8.product_kernel(1, 16, 16, dtype, 8, False, "gated_fp8")
    for shape, size in (("1x8", (1, 19, 16, 400)), ("2x4", (77, 124, 16, 400)), ("2x8", (12592, 22, 21, 400))):
        yield f"fp8_few_product_e4m3_{name}_{shape}", fp8.product_kernel(*size[:3], dtype, size[3])
    for shape, kind, size in (("2x4", "gated", (444, 17, 16, 400)), ("2x8", "gated_kept", (1, 16, 16, 8))):
        yield f"fp8_few_gated_e4m3_{name}_{shape}", fp8.product_kernel(*size[:3], dtype, size[3], False, kind)


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
