"""CPU checks of the persistent product kernels' compiled code: what their counted waits rely on.

The loads go to LDS as inline assembly, which the compiler's wait counts leave out, and vmcnt counts a tile's stores
among them: every wave has to issue exactly the stores that the wait after a tile allows for, on every path through
the tile's end that comes before the wait.
"""

import re

import pytest

from triton_chip_benchmarks_amd import _native, audit

# (features, rows, stages) of the tiles; a wave's LDS loads a step and 16-byte stores a tile follow.
TILES = {"256x128": (256, 128, 3), "128x64": (128, 64, 3), "64x64": (64, 64, 3)}
ITEM = {"f32": 4, "f16": 2, "bf16": 2}


def _expected(tile, dtype):
    features, rows, stages = TILES[tile]
    loads = features // 32 + rows // 32 + 1
    stores = features * rows // 4 // 64 * ITEM[dtype] // 16
    return loads, stores, stages


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tile", sorted(TILES))
def test_waits_allow_for_the_loads_and_stores_in_flight(tile, dtype):
    name = f"mx_product_{dtype}_{tile}_stream"
    assert name in _native.kernel_names()
    lines = audit.instructions(name)
    loads, stores, stages = _expected(tile, dtype)
    whole = [i for i, line in enumerate(lines) if audit.mnemonic(line) == "buffer_store_dwordx4"]
    assert len(whole) == stores, "one store a piece, at one place"
    # No branch between a tile's stores: every wave issues all of them.
    between = [audit.mnemonic(line) for line in lines[whole[0]:whole[-1]]]
    assert not [m for m in between if "branch" in m or "exec" in m], between
    waits = {int(m.group(1)) for line in lines for m in [re.search(r"vmcnt\((\d+)\)", line)] if m}
    step, after_stores = (stages - 2) * loads, (stages - 2) * loads + stores
    assert {step, after_stores, (stages - 1) * loads, 0} >= waits >= {step, after_stores, (stages - 1) * loads}, waits
    barriers = [i for i, line in enumerate(lines) if audit.mnemonic(line) == "s_barrier"]
    assert len(barriers) == 3  # the prologue's and one of each of the loop's two steps
    for barrier in barriers[1:]:
        before = " ".join(lines[barrier - 12:barrier])
        assert f"vmcnt({step})" in before and f"vmcnt({after_stores})" in before and "lgkmcnt(0)" in before
    # A step's products lie between its loads, not behind them.
    body = [audit.mnemonic(line) for line in lines[barriers[1]:barriers[2]]]
    dmas = [i for i, m in enumerate(body) if m == "buffer_load_dwordx4"]
    products = [i for i, m in enumerate(body) if m.startswith("v_mfma")]
    assert len(dmas) == loads
    assert sum(i < dmas[-1] for i in products) >= 0.6 * len(products)


def test_products_run_on_the_scaled_fp4_instruction():
    for name in _native.kernel_names():
        if name.startswith(("mx_product_", "mx_linear_few_")):
            matrix = {audit.mnemonic(line) for line in audit.instructions(name) if "mfma" in line}
            assert matrix and matrix <= {"v_mfma_scale_f32_32x32x64_f8f6f4", "v_mfma_scale_f32_16x16x128_f8f6f4"}, name
