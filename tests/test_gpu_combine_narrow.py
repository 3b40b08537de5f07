"""Combine where a row takes fewer lanes than a token has entries: the lanes past the row hold entries too."""

import numpy as np
import pytest

from oracle import routing as oracle

pytestmark = pytest.mark.gpu

UNIT = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n", [1, 8, 9, 63, 513, 520])
def test_rows_of_few_columns_sum_every_entry(gpu, dtype, n):
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"combine {dtype} 5x64x{n}", flush=True)
    tokens, top = 5, 64
    generator = torch.Generator(device="cuda").manual_seed(n)
    rows = tokens * top
    y = torch.randn(rows, n, device="cuda", generator=generator).to(
        {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[dtype])
    weights = torch.randn(tokens, top, device="cuda", generator=generator)
    slots = np.random.default_rng(n).permutation(rows).reshape(tokens, top).astype(np.int32)
    slots[1, ::3] = -1
    guarded = torch.full((tokens + 2, n), 7.0, device="cuda", dtype=y.dtype)
    routing.combine(y, torch.tensor(slots, device="cuda"), weights, guarded[1:-1])
    expected, size = oracle.combine(y.double().cpu().numpy(), slots, weights.double().cpu().numpy())
    # `top` products and sums in fp32, one rounding to the type.
    bound = top * 2.0**-23 * size
    error = np.abs(guarded[1:-1].double().cpu().numpy() - expected)
    assert (error <= bound + UNIT[dtype] * (np.abs(expected) + bound) + 2.0**-25).all()
    assert (guarded[0] == 7).all() and (guarded[-1] == 7).all()
