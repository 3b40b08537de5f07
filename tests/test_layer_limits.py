"""CPU checks of the layer operators' limits: what a launch cannot hold is refused, or runs on another kernel.

HIP takes at most 2^32 - 1 work items a launch, 256 of them a workgroup here: 2^24 - 1 workgroups.
"""

import pytest

from triton_chip_benchmarks_amd import _native, mx

P, BIG = 1 << 20, 1 << 40


# Row tiles of 128 rows (an expert's last one its own) times column tiles.
@pytest.mark.parametrize("rows,experts,n,tiles,kernel", [(69854, 4096, 462720, 2**24 - 1, "mx_product_bf16"),
                                                         (69854, 4096, 462592, 16772574, "mx_product_bf16_128x128")])
def test_a_grid_that_is_rounded_up_to_the_xcds_still_fits_a_launch(rows, experts, n, tiles, kernel):
    assert (rows // 128 + min(rows, experts)) * -(-n // 128) == tiles
    assert mx.product_kernel(rows, n, 32, experts=experts) == kernel


def test_combine_backward_takes_no_more_tokens_than_a_launch_has_workgroups():
    backward = lambda tokens: _native.load().mb_combine_backward(  # noqa: E731
        2, P, BIG, P, BIG, 8, P, BIG, P, BIG, P, BIG, P, BIG, tokens, 2, 8, None)
    assert backward(1 << 24) == _native.MB_ERR_UNSUPPORTED
    assert "at most 16777215 tokens" in _native.last_error()
    assert backward(0) == _native.MB_OK
