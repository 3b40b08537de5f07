"""FP8 operators and the norm on tensors whose bytes and elements pass 32 bits: rows behind the 2^32nd byte and element
against the same rows alone, and against the oracle."""

import numpy as np
import pytest

from oracle import fp8 as oracle_fp8

pytestmark = pytest.mark.gpu

OVER = 1 << 32


def _host(tensor):
    return tensor.double().cpu().numpy()


def _codes(torch, rows, k, seed):
    """Codes of every finite value, made quickly."""
    codes = torch.randint(0, 256, (rows, k), dtype=torch.uint8, device="cuda",
                          generator=torch.Generator(device="cuda").manual_seed(seed))
    codes.masked_fill_((codes & 127) == 127, 56)
    return codes.view(torch.float8_e4m3fn)


def _operand(torch, rows, k, seed, block=1):
    from triton_chip_benchmarks_amd import fp8

    scales = torch.full((-(-k // 512), -(-rows // block), 4), 120, dtype=torch.uint8, device="cuda")
    scales += torch.arange(4, dtype=torch.uint8, device="cuda")
    return fp8.Packed(_codes(torch, rows, k, seed), scales, k, block)


def _rows(packed, chosen):
    import torch

    from triton_chip_benchmarks_amd import fp8

    codes = packed.codes.view(torch.uint8)[chosen].view(packed.codes.dtype)
    return fp8.Packed(codes, packed.scales[:, chosen].contiguous(), packed.k)


def _values(packed):
    import torch

    codes = packed.codes.view(torch.uint8)
    return oracle_fp8.values(codes.cpu().numpy(), packed.scales.cpu().numpy(), packed.k, packed.block)


def _check_product(out, a, b):
    """out = a . b^T within a rounding to its type and the sums' own: of 128 products to 2^-12 of their magnitudes where
    the output has 16 bits (the matrix cores' FP8 sums), in fp32 where it has 32."""
    x, w = _values(a), _values(b)
    exact, size, k = x @ w.T, np.abs(x) @ np.abs(w).T, x.shape[1]
    bound = 2.0**-8 * np.abs(exact) + 2.0**-12 * size if out.element_size() == 2 else (k / 32 + 16) * 2.0**-23 * size
    assert (np.abs(_host(out) - exact) <= bound).all()


def test_norm_quantisation_and_back(gpu):
    import torch

    from triton_chip_benchmarks_amd import fp8, norm

    rows, n = 530000, 8200
    assert rows * n > OVER
    print(f"large norm {rows}x{n}", flush=True)
    x = torch.empty(rows, n, device="cuda", dtype=torch.bfloat16).normal_(
        generator=torch.Generator(device="cuda").manual_seed(0))
    weight = torch.linspace(0.5, 1.5, n, device="cuda").bfloat16()
    some = torch.tensor([0, 261888, 261889, OVER // n, OVER // n + 1, rows - 1], device="cuda")
    packed = fp8.empty(rows, n)
    out = norm.rms_norm(x, weight, out=torch.empty_like(x), packed=packed).out
    small = fp8.empty(len(some), n)
    expected = norm.rms_norm(x[some], weight, out=torch.empty(len(some), n, device="cuda", dtype=x.dtype), packed=small)
    # (The few rows are normed by more waves each: another order of the row's sum, a rounding apart at most.)
    assert torch.allclose(out[some].float(), expected.out.float(), rtol=2.0**-7, atol=0)
    got = fp8.dequantize(_rows(packed, some)).float()
    assert torch.allclose(got, fp8.dequantize(small).float(), rtol=2.0**-3, atol=2.0**-8)
    d_x, _ = norm.rms_norm_backward(out, x, weight)
    alone, _ = norm.rms_norm_backward(out[some], x[some], weight)
    assert torch.equal(d_x[some], alone)
    del d_x
    fp8.quantize(x, packed)
    alone = fp8.quantize(x[some])
    assert torch.equal(packed.codes[some].view(torch.uint8), alone.codes.view(torch.uint8))
    assert torch.equal(packed.scales[:, some], alone.scales)
    back = fp8.dequantize(packed, out)
    assert torch.equal(back[some], fp8.dequantize(alone))
    del out, back
    both = fp8.quantize_both(x[:, :8192], columns=fp8.empty(8192, rows), rows=fp8.empty(rows, 8192))
    alone = fp8.quantize(x[some, :8192])
    assert torch.equal(both[0].codes[some].view(torch.uint8), alone.codes.view(torch.uint8))
    tail = fp8.quantize(x[529920:, 8000:8192], columns=True)  # the last block along the columns' K, past the 2^32nd byte
    assert both[1].codes.numel() > OVER and 529920 % 128 == 0
    assert torch.equal(both[1].codes[8000:, 529920:].contiguous().view(torch.uint8), tail.codes.view(torch.uint8))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_products_of_long_operands(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import fp8

    kind = {"bf16": torch.bfloat16, "fp32": torch.float32}[dtype]
    rows, n, k = 270000, 96, 16400
    assert rows * k > OVER
    print(f"large operand {dtype} {rows}x{n}x{k}", flush=True)
    a, b = _operand(torch, rows, k, 1), _operand(torch, n, k, 2, 128)
    out = fp8.product(a, b, dtype=kind)
    some = torch.tensor([0, OVER // k, OVER // k + 1, rows - 1], device="cuda")
    _check_product(out[some], _rows(a, some), b)
    for few in (3, 200):  # a as a long weight
        x = _operand(torch, few, k, few)
        _check_product(fp8.product(x, a, dtype=kind)[:, some], x, _rows(a, some))


def test_outputs_and_experts_past_32_bits(gpu):
    import torch

    from triton_chip_benchmarks_amd import fp8

    rows, n, k = 530000, 8200, 128
    assert rows * n > OVER
    print(f"large output {rows}x{n}x{k}", flush=True)
    a, b = _operand(torch, rows, k, 5), _operand(torch, n, k, 6, 128)
    some = torch.tensor([0, 261888, OVER // n, OVER // n + 1, rows - 1], device="cuda")
    out = fp8.product(a, b)
    assert torch.equal(out[some], fp8.product(_rows(a, some), b, kernel=fp8.product_kernel(rows, n, k)))
    del out
    half = _operand(torch, 2 * 4104, k, 7, 128)
    gate_up = torch.empty(rows, 2 * 4104, device="cuda", dtype=torch.bfloat16)
    out = fp8.gated(a, half, gate_up=gate_up)
    kept = torch.empty(len(some), 2 * 4104, device="cuda", dtype=torch.bfloat16)
    name = fp8.product_kernel(rows, 4104, k, kind="gated_kept")
    assert torch.equal(out[some], fp8.gated(_rows(a, some), half, gate_up=kept, kernel=name))
    assert torch.equal(gate_up[some], kept)
    del out, gate_up
    experts, n, k = 130, 4096, 8208
    assert experts * n * k > OVER
    print(f"large experts {experts}x{n}x{k}", flush=True)
    weight = fp8.Packed(_codes(torch, experts * n, k, 8).view(experts, n, k),
                        torch.full((experts, 17, 32, 4), 120, dtype=torch.uint8, device="cuda"), k, 128)
    for rows in (3, 400):
        offsets = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        offsets[1:] = 1  # expert 0 has a row, the last one the others
        offsets[-1] = rows
        x = _operand(torch, rows, k, 9)
        out = fp8.product(x, weight, offsets=offsets)
        for e, chosen in ((0, [0]), (experts - 1, [1, rows - 1])):
            some, features = torch.tensor(chosen, device="cuda"), torch.tensor([0, 127, 128, n - 1], device="cuda")
            mine = fp8.dequantize(fp8.Packed(weight.codes[e], weight.scales[e], k, 128))[features].float()
            exact, size = (_host(f(fp8.dequantize(_rows(x, some)).float())) @ _host(f(mine)).T
                           for f in (lambda v: v, torch.abs))
            assert (np.abs(_host(out[some][:, features]) - exact) <= 2.0**-8 * np.abs(exact) + 2.0**-12 * size).all()
