"""CPU checks of the compiled code of the FP8 products' persistent kernels: what their counted waits rely on.

The loads go to LDS as inline assembly, which the compiler's wait counts leave out, and vmcnt counts a tile's stores
among them: every wave has to issue at least the stores that the wait after a tile allows for, on every path through the
tile's end that comes before the wait.
"""

import re

import pytest

from triton_chip_benchmarks_amd import _native, audit

STAGES = {"256x256": 2, "256x128": 3, "128x128": 4, "128x64": 3, "64x64": 3, "256x64": 3}
ITEM = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
KERNELS = sorted(name for name in _native.kernel_names() if name.startswith("fp8_tiles_"))


def _expected(kind, dtype, tile):
    """A wave's LDS loads a step, and its stores of 16 bytes and of one a tile."""
    features, rows = map(int, tile.split("x"))
    loads = features // 32 + rows // 32 + 1
    blocks = features // 64 * (rows // 64)  # of 32 x 32 elements, a wave's
    wide = {"product": blocks * ITEM[dtype], "gated": blocks // 2 * ITEM[dtype],
            "gated_kept": (blocks // 2 + blocks) * ITEM[dtype], "gated_fp8": blocks // 2}[kind]
    return loads, wide, 4 * (rows // 64) if kind == "gated_fp8" else 0


@pytest.mark.parametrize("name", KERNELS)
def test_waits_allow_for_the_loads_and_stores_in_flight(name):
    kind, dtype, tile = re.fullmatch(r"fp8_tiles_(\w+)_(\w+?)_(\d+x\d+)", name).groups()
    loads, wide, bytes_ = _expected(kind, dtype, tile)
    stages, lines = STAGES[tile], audit.instructions(name)
    mnemonics = [audit.mnemonic(line) for line in lines]
    at = {m: [i for i, got in enumerate(mnemonics) if got == m] for m in ("buffer_store_dwordx4", "buffer_store_byte")}
    assert len(at["buffer_store_dwordx4"]) == wide, "one store a piece, at one place"
    assert len(at["buffer_store_byte"]) == bytes_
    waits = {int(m.group(1)) for line in lines for m in [re.search(r"vmcnt\((\d+)\)", line)] if m}
    step = (stages - 2) * loads
    after_stores = step + wide + bytes_
    assert {step, after_stores, (stages - 1) * loads, 0} >= waits >= {step, after_stores, (stages - 1) * loads}, waits
    # The matrix instructions of the format: scales applied for outputs of 16 bits and FP8, bf16 for those of fp32.
    matrix = {m for m in mnemonics if "mfma" in m}
    assert matrix == {"v_mfma_f32_32x32x16_bf16" if dtype == "f32" else "v_mfma_scale_f32_32x32x64_f8f6f4"}
    # Nothing skips a store of 16 bytes: the branches between them leave out only an edge's stores of an element.
    first, last = min(sum(at.values(), [])), max(sum(at.values(), []))
    inside = [i for i, m in enumerate(mnemonics) if m.startswith("s_cbranch") and first < i < last]
    assert not (inside and kind == "gated_fp8")
    for i in inside:
        following = mnemonics[i + 1:last + 1]
        until = next((j for j, m in enumerate(following) if m == "buffer_store_dwordx4"), len(following))
        skipped = [m for m in following[:until] if m.startswith("buffer_store")]
        assert skipped and set(skipped) <= {"buffer_store_short", "buffer_store_dword", "buffer_store_short_d16_hi"}, i


def test_few_row_kernels_run_on_the_instructions_of_the_format():
    for name in _native.kernel_names():
        if name.startswith("fp8_few_"):
            matrix = {audit.mnemonic(line) for line in audit.instructions(name) if "mfma" in line}
            output = name.split("_")[-2]
            assert matrix == {"v_mfma_f32_16x16x32_bf16" if output == "f32" else "v_mfma_scale_f32_16x16x128_f8f6f4"}, name
