"""CPU checks of which kernel a product runs on: the names that mb_mx_product_kernel gives, and what it refuses."""

import pytest
import torch

from triton_chip_benchmarks_amd import _native, mx

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# (rows, n, k, experts) of each kernel of products.
CHOSEN = {
    "few_16x8": (16, 130, 256, 1), "few_32x8": (3, 8203, 512, 1), "few_32x4": (256, 2048, 4096, 128),
    "64x64": (130, 8190, 1056, 1), "128x128": (2600, 3001, 300, 1), "64x64_stream": (20, 1000, 40, 1),
    "128x64_stream": (6851, 5916, 305, 256), "256x128_stream": (4100, 4104, 1100, 1),
    "": (17, 1 << 20, 257 * 256, 1),
}


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_every_kernel_of_products_is_some_sizes_choice(dtype):
    chosen = set()
    for form, (rows, n, k, experts) in CHOSEN.items():
        few, size = form.startswith("few_"), form.removeprefix("few_")
        name = mx.product_kernel(rows, n, k, DTYPES[dtype], experts)
        assert name == "_".join(filter(None, ("mx_product", "few" if few else "", dtype, size)))
        linear = mx.product_kernel(rows, n, k, DTYPES[dtype], experts, linear=True)
        assert linear == (f"mx_linear_few_{dtype}_{size}" if few else name)
        chosen |= {name, linear}
    assert chosen == {name for name in _native.kernel_names()
                      if name.startswith(("mx_product_", "mx_linear_few_")) and f"_{dtype}" in name}


def test_sizes_and_names_that_have_no_kernel_are_refused():
    with pytest.raises(_native.NativeError, match="empty product"):
        mx.product_kernel(0, 64, 64)
    with pytest.raises(_native.NativeError, match="experts"):
        mx.product_kernel(4, 64, 64, experts=5000)
    with pytest.raises(_native.NativeError, match="element type"):
        mx.product_kernel(4, 64, 64, torch.float64)
    library, address, big = _native.load(), 1 << 20, 1 << 40  # never dereferenced: refused before any launch

    def exact(kernel, rows=8, experts=1, offsets=None):
        return library.mb_mx_product_exact(kernel, 2, address, big, address, big, address, big, address, big, address,
                                           big, rows, 64, 96, offsets, big if offsets else 0, experts, None)

    assert exact(None) == _native.MB_ERR_INVALID and "name" in _native.last_error()
    for kernel, options in ((b"mx_product_bf16_32x32", {}), (b"mx_product_f32_64x64", {}), (b"copy_tail", {}),
                            (b"mx_linear_few_bf16_16x8", {}),
                            (b"mx_product_bf16_64x64_stream", {"experts": 300, "offsets": address})):
        assert exact(kernel, **options) == _native.MB_ERR_UNSUPPORTED, kernel
        assert kernel.decode() in _native.last_error()
    assert exact(b"mx_product_bf16_64x64", experts=2) == _native.MB_ERR_INVALID  # without offsets
