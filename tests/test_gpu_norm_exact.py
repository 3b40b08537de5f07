"""The norm's sum, root and products are of 64 bits: an output is the exact value's rounding, and an FP8 code the exact
value's, but for fp32's rounding.

y = fp32(t r w). The sum of n squares in 64 bits is off by less than n 2^-53 of itself (2^-39 at 16384 elements), its root
by half of that; a step of Newton from fp32's reciprocal root, which is within 2^-22, leaves 1.5 * 2^-44 = 2^-43.4; two
products add 2^-52. All of it is under 2^-39: y is the fp32 value nearest to t r w (1 + d), |d| <= 2^-39, whatever n. An
output of 16 bits is rounded a second time. (Sums of fp32 are off by more than 2^-24 at a thousand elements.)
"""

import numpy as np
import pytest

from oracle import fp8 as fp8_oracle
from oracle import norm as oracle

pytestmark = pytest.mark.gpu

OFF = 2.0**-39
# The rows' size and eps: a mean of squares near 1, past 1e30, and below 1e-30, where the root is taken another way.
SIZES = [(1.0, 1e-6), (3e16, 1e-6), (2e-18, 0.0)]


def host(tensor):
    return tensor.double().cpu().numpy()


@pytest.mark.parametrize("dtype,size,eps", [(dtype, *size) for dtype in ("float32", "float16", "bfloat16")
                                            for size in SIZES[:1 if dtype == "float16" else 3]])  # (fp16 holds no others)
@pytest.mark.parametrize("rows,n", [(3, 1), (40, 130), (514, 512), (5, 1024), (514, 1025), (7, 4096), (514, 4104),
                                    (6, 8192), (514, 8192), (3, 16384), (514, 16384)])
def test_outputs_and_codes_are_the_exact_values(gpu, rows, n, dtype, size, eps):
    import torch

    from triton_chip_benchmarks_amd import fp8, norm

    of = getattr(torch, dtype)
    generator = torch.Generator(device="cuda").manual_seed(rows + n)
    x = (size * torch.randn(rows, n, device="cuda", generator=generator)).to(of)
    weight = (1 + 0.2 * torch.randn(n, device="cuda", generator=generator)).to(of)
    normed = norm.rms_norm(x, weight, eps, out=torch.full_like(x, float("nan")), packed=fp8.empty(rows, n))
    exact = oracle.rms_norm(host(x), host(weight), float(np.float32(eps)))  # the library takes eps in fp32
    info = torch.finfo(of)
    again = info.eps / 2 * (1 + 2.0**-20) if dtype != "float32" else 0.0
    floor = info.smallest_normal * info.eps / 2 + 2.0**-149
    assert (np.abs(host(normed.out) - exact) <= (2.0**-24 + OFF + again) * np.abs(exact) + floor).all()
    codes, scales = normed.packed.codes.view(torch.uint8).cpu().numpy()[:, :n], normed.packed.scales.cpu().numpy()
    flat, blocks = scales.transpose(1, 0, 2).reshape(rows, -1), -(-n // 128)
    low, high = ((exact * (1 + sign * OFF)).astype(np.float32).astype(np.float64) for sign in (-1, 1))
    held = flat[:, :blocks]
    low_scale, high_scale = fp8_oracle.scale_codes(low), fp8_oracle.scale_codes(high)
    assert ((held == low_scale) | (held == high_scale)).all()
    low_code, high_code = (fp8_oracle.element_codes(part, held) for part in (low, high))
    assert ((codes == low_code) | (codes == high_code)).all()
    # Hardly a value lies so near to a border that either side of it may be right.
    assert (low_code != high_code).mean() < 1e-4 and (low_scale != high_scale).mean() < 1e-3
