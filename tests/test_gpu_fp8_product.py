"""FP8 products with block scales, linear layers, the gated pair and their gradients against the float64 oracle.

Tolerances, per element, of |error| <= rounding |exact| + sums * (the same sum of magnitudes) + floor, with u = eps / 2
of the output's type:
  rounding  u of the product's one rounding.
  sums      16-bit outputs: the FP8 matrix instructions drop what lies some bits below a block's largest product, 2^-13
            of the sum of its 128 magnitudes where that was looked for; twice that. fp32 ones: products are exact, and a
            sum of K of them in any order is off by less than K 2^-24 of the magnitudes.
Of a gated product g / (1 + e^-g) u the errors add up (d silu / d g is within 1.1), with eight roundings of 2^-24 of the
fp32 evaluation.
"""

import numpy as np
import pytest

from oracle import fp8 as oracle

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


def half_step(torch, dtype):
    return torch.finfo(getattr(torch, dtype)).eps / 2


def sums(dtype, k):
    return k * 2.0**-24 if dtype == "float32" else 2.0**-12


def host(t):
    return t.detach().cpu().double().numpy()


def tensor(torch, values, dtype):
    return torch.tensor(values, dtype=torch.float32).to(getattr(torch, dtype)).cuda()


def normal(torch, rows, k, dtype, seed, scale=1.0):
    """N(0, scale) with some channels ten times as large."""
    rng = np.random.default_rng(seed)
    channel = np.where(rng.random(k) < 0.05, 10.0, 1.0)
    return tensor(torch, rng.standard_normal((rows, k)) * channel * scale, dtype)


def floor(torch, dtype):
    """Half the spacing of the type's smallest values."""
    info = torch.finfo(getattr(torch, dtype))
    return info.smallest_normal * info.eps / 2


def close(torch, out, exact, magnitudes, dtype, k):
    error = np.abs(host(out) - exact)
    bound = half_step(torch, dtype) * np.abs(exact) + sums(dtype, k) * magnitudes * (1 + 2.0**-7) + floor(torch, dtype)
    assert out.dtype == getattr(torch, dtype) and (error <= bound).all(), float((error / bound).max())


def gate_bound(torch, pair, pair_magnitudes, dtype, k):
    """(silu(g) u, how far it may be off): the pair's sums are off by s times their magnitudes, silu' is within 1.1."""
    n = pair.shape[1] // 2
    off = sums(dtype, k) * pair_magnitudes
    out = oracle.gate(pair)
    silu = pair[:, :n] * oracle.sigmoid(pair[:, :n])
    error = (1.1 * off[:, :n] * np.abs(pair[:, n:]) + np.abs(silu) * off[:, n:] + 1.1 * off[:, :n] * off[:, n:]
             + 8 * 2.0**-24 * np.abs(out))
    return out, error * (1 + 2.0**-7) + half_step(torch, dtype) * (np.abs(out) + error) + floor(torch, dtype)


# One row to past every border of rows and features a wave or workgroup takes; K of one code, a part of a 16-byte piece,
# a block and its neighbours, an odd number of blocks, and more than a scale dword.
SHAPES = [(1, 1, 1), (1, 200, 128), (3, 130, 129), (16, 64, 511), (17, 96, 640), (5, 48, 4112), (33, 260, 1040),
          (64, 128, 272), (130, 300, 96), (257, 513, 384), (600, 700, 2000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_linear_and_product(gpu, dtype, rows, n, k):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x, w = normal(torch, rows, k, dtype, 1), normal(torch, n, k, dtype, 2, k**-0.5)
    weight = fp8.quantize(w, block=128)
    exact, magnitudes = oracle.linear(host(x), host(w))
    close(torch, fp8.linear(x, weight), exact, magnitudes, dtype, k)
    out = torch.full((rows, n), float("nan"), device="cuda", dtype=x.dtype)
    close(torch, fp8.product(fp8.quantize(x), weight, out), exact, magnitudes, dtype, k)
    # The other blocks: a weight with a scale a row, rows that share theirs.
    a, b = oracle.rounded(host(x), 128), oracle.rounded(host(w))
    out = fp8.product(fp8.quantize(x, block=128), fp8.quantize(w), dtype=x.dtype)
    close(torch, out, a @ b.T, np.abs(a) @ np.abs(b).T, dtype, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_gated(gpu, dtype, rows, n, k):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x, w = normal(torch, rows, k, dtype, 3), normal(torch, 2 * n, k, dtype, 4, k**-0.5)
    weight = fp8.quantize(w, block=128)
    pair, magnitudes = oracle.linear(host(x), host(w))
    exact, bound = gate_bound(torch, pair, magnitudes, dtype, k)
    gate_up = torch.full((rows, 2 * n), float("nan"), device="cuda", dtype=x.dtype)
    for given in (x, fp8.quantize(x)):
        options = {"dtype": x.dtype} if given is not x else {}
        for kept in (None, gate_up):
            out = fp8.gated(given, weight, gate_up=kept, **options)
            assert out.dtype is x.dtype and (np.abs(host(out) - exact) <= bound).all()
        close(torch, gate_up, pair, magnitudes, dtype, k)
        gate_up.fill_(float("nan"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_gated_to_an_operand(gpu, dtype, rows, n, k):
    """Each value is within half a step of E4M3 (2^-4 of it, 2^-10 of the scale below 2^-6 of it) of one that the sums
    allow, under a scale that is the exact one or, where the block's largest may lie either side of a border, its
    neighbour."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    x, w = normal(torch, rows, k, dtype, 5), normal(torch, 2 * n, k, dtype, 6, k**-0.5)
    weight = fp8.quantize(w, block=128)
    pair, magnitudes = oracle.linear(host(x), host(w))
    exact, error = gate_bound(torch, pair, magnitudes, "bfloat16", k)
    error = error - half_step(torch, "bfloat16") * (np.abs(exact) + error)  # fp32 values: not rounded to 16 bits
    for given in (x, fp8.quantize(x)):
        packed = fp8.gated(given, weight, packed=fp8.empty(rows, n))
        codes, scales = packed.codes.view(torch.uint8).cpu().numpy(), packed.scales.cpu().numpy()
        assert not codes[:, n:].any()
        flat = scales.transpose(1, 0, 2).reshape(rows, -1)
        blocks = -(-n // 128)
        assert (flat[:, blocks:] == 127).all()
        low, high = (oracle.scale_codes(np.maximum(np.abs(exact) + sign * error, 0)) for sign in (-1, 1))
        assert ((flat[:, :blocks] >= low) & (flat[:, :blocks] <= high)).all()
        values = oracle.values(codes, scales, n)
        scale = np.exp2(np.repeat(flat[:, :blocks].astype(np.float64), 128, axis=1)[:, :n] - 127)
        allowed = error + 2.0**-4 * (np.abs(exact) + error) + 2.0**-10 * scale
        assert (np.abs(values - exact) <= allowed).all()


def routed(torch, tokens, top, experts, seed, masked=False):
    from triton_chip_benchmarks_amd import routing

    rng = np.random.default_rng(seed)
    popular = rng.standard_normal(experts) * 1.5
    chosen = np.argsort(-(popular + rng.gumbel(size=(tokens, experts))), axis=1)[:, :top].astype(np.int32)
    if masked:
        chosen[2::5] = -1
    return chosen, routing.dispatch(torch.tensor(chosen).cuda(), experts)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,top,experts,n,k,masked", [(1, 1, 1, 40, 128, False), (3, 2, 8, 72, 200, False),
                                                           (32, 4, 60, 130, 384, True), (300, 2, 7, 144, 272, True),
                                                           (700, 3, 5, 260, 640, False), (40, 2, 300, 64, 128, False)])
def test_routed(gpu, dtype, tokens, top, experts, n, k, masked):
    """Linear layers and gated pairs of experts; what lies past the last routed row stays as it was."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    chosen, plan = routed(torch, tokens, top, experts, 11, masked)
    x = normal(torch, tokens, k, dtype, 12)
    linear, pair = fp8.empty(n, k, 128, experts=experts), fp8.empty(2 * n, k, 128, experts=experts)
    weights = []
    for e in range(experts):
        w = normal(torch, 2 * n, k, dtype, 100 + e, k**-0.5)
        weights.append(host(w))
        fp8.quantize(w, fp8.Packed(pair.codes[e], pair.scales[e], k, 128), block=128)
        fp8.quantize(w[:n], fp8.Packed(linear.codes[e], linear.scales[e], k, 128), block=128)
    order = plan.order.cpu().numpy()
    live = int(plan.offsets[-1])
    expert_of = chosen.reshape(-1)[order[:live]]
    rows = host(x)[order[:live] // top]
    exact_pair, magnitudes = np.zeros((live, 2 * n)), np.zeros((live, 2 * n))
    exact, exact_magnitudes = np.zeros((live, n)), np.zeros((live, n))
    for e in range(experts):
        at = expert_of == e
        if at.any():
            exact_pair[at], magnitudes[at] = oracle.linear(rows[at], weights[e])
            exact[at], exact_magnitudes[at] = oracle.linear(rows[at], weights[e][:n])
    total = tokens * top

    def fresh(*shape):
        return torch.full(shape, 7.0, device="cuda", dtype=x.dtype)

    sorted_x = x[torch.tensor(np.maximum(order, 0) // top).cuda().long()].contiguous()
    operand = fp8.quantize(sorted_x)
    for out in (fp8.linear(x, linear, fresh(total, n), plan=plan),
                fp8.linear(sorted_x, linear, fresh(total, n), plan=plan, sorted_rows=True),
                fp8.product(operand, linear, fresh(total, n), offsets=plan.offsets)):
        close(torch, out[:live], exact, exact_magnitudes, dtype, k)
        assert (out[live:] == 7).all()
    gated, bound = gate_bound(torch, exact_pair, magnitudes, dtype, k)
    for given, options in ((x, {}), (sorted_x, {"sorted_rows": True}), (operand, {"sorted_rows": True})):
        gate_up, out = fresh(total, 2 * n), fresh(total, n)
        fp8.gated(given, pair, out, gate_up=gate_up, plan=plan, **options)
        assert (np.abs(host(out[:live]) - gated) <= bound).all() and (out[live:] == 7).all()
        close(torch, gate_up[:live], exact_pair, magnitudes, dtype, k)
        assert (gate_up[live:] == 7).all()
        packed = fp8.empty(total, n)
        packed.codes.view(torch.uint8).fill_(3)
        packed.scales.fill_(9)
        fp8.gated(given, pair, packed=packed, plan=plan, **options)
        values = host(fp8.dequantize(packed, torch.empty(total, n, device="cuda")))[:live]
        largest = np.abs(gated).max(axis=1, keepdims=True)
        assert (np.abs(values - gated) <= bound + 2.0**-4 * (np.abs(gated) + bound) + 2.0**-16 * largest).all()
        assert (packed.codes.view(torch.uint8)[live:] == 3).all()
        assert (packed.scales[:, live:] == 9).all()


BACKWARD = [(1, 1, 1), (5, 64, 129), (130, 200, 96), (128, 128, 128), (300, 72, 257), (513, 260, 640)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", BACKWARD)
def test_linear_backward(gpu, dtype, rows, n, k):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x, w = normal(torch, rows, k, dtype, 21), normal(torch, n, k, dtype, 22, k**-0.5)
    d = normal(torch, rows, n, dtype, 23, 0.01)
    _, columns = fp8.quantize_both(w, block=128)
    d_x, d_w = fp8.linear_backward(d, x, columns)
    (exact_x, magnitudes_x), (exact_w, magnitudes_w) = oracle.linear_backward(host(d), host(x), host(w))
    close(torch, d_x, exact_x, magnitudes_x, dtype, n)
    close(torch, d_w, exact_w, magnitudes_w, dtype, rows + 128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,k", BACKWARD)
def test_gated_backward(gpu, dtype, rows, n, k):
    """The gradient of [gate | up] is evaluated in fp32 and rounded to codes: a value that fp32's error (under 16 roundings
    of 2^-24 of its terms) takes across a border is off by a step, 2^-3 of it, or, in a block whose largest lies next to a
    border of the scale, by its smallest step. Where that happens is known from the exact values."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    x, w = normal(torch, rows, k, dtype, 31), normal(torch, 2 * n, k, dtype, 32, k**-0.5)
    d, pair = normal(torch, rows, n, dtype, 33, 0.01), normal(torch, rows, 2 * n, dtype, 34)
    _, columns = fp8.quantize_both(w, block=128)
    d_x, d_w = fp8.gated_backward(d, pair, x, columns)
    exact = oracle.gate_backward(host(d), host(pair))
    g, u = np.split(host(pair), 2, axis=1)
    s = oracle.sigmoid(g)
    terms = np.concatenate([np.abs(host(d) * u) * s * (1 + np.abs(g) * (1 - s)), np.abs(host(d) * g) * s], axis=1)
    off = 16 * 2.0**-24 * terms
    weight, x_columns = oracle.rounded(host(w), 128), oracle.rounded(host(x).T).T

    def unsure(values, error):
        """How far the operand's values may be from the exact values' ones."""
        return np.abs(oracle.rounded(values + error) - oracle.rounded(values - error))

    d_rows, d_columns = oracle.rounded(exact), oracle.rounded(exact.T)
    slack_x = unsure(exact, off) @ np.abs(weight)
    slack_w = unsure(exact.T, off.T) @ np.abs(x_columns)
    for out, value, magnitudes, slack, depth in (
            (d_x, d_rows @ weight, np.abs(d_rows) @ np.abs(weight), slack_x, 2 * n),
            (d_w, d_columns @ x_columns, np.abs(d_columns) @ np.abs(x_columns), slack_w, rows + 128)):
        error = np.abs(host(out) - value)
        bound = (half_step(torch, dtype) * (np.abs(value) + slack) + sums(dtype, depth) * (magnitudes + slack)
                 * (1 + 2.0**-7) + slack + floor(torch, dtype))
        assert (error <= bound).all(), float((error / bound).max())


def test_gated_gradient_against_differences(gpu):
    """The formula's gradient of [gate | up] is what differences of the oracle's output say, and the kernel's d_x for a
    weight of the identity is that gradient, as its operand holds it."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    rng = np.random.default_rng(41)
    n = 64
    pair, d = rng.standard_normal((6, 2 * n)) * 2, rng.standard_normal((6, n))
    pair[0, :8] = [-90, -30, -8, 0, 8, 30, 90, 1e-3]
    gradient, step = oracle.gate_backward(d, pair), 1e-5
    for j in range(2 * n):
        moved = [oracle.gate(pair + sign * step * (np.arange(2 * n) == j)) for sign in (1, -1)]
        difference = ((moved[0] - moved[1]) * d).sum(axis=1) / (2 * step)
        np.testing.assert_allclose(difference, gradient[:, j], rtol=1e-6, atol=1e-7)
    pair32, d32 = tensor(torch, pair, "float32"), tensor(torch, d, "float32")
    gradient = oracle.gate_backward(host(d32), host(pair32))
    identity = torch.eye(2 * n, device="cuda")
    _, columns = fp8.quantize_both(identity, block=128)
    d_x, _ = fp8.gated_backward(d32, pair32, identity[:6].contiguous(), columns)
    held = oracle.rounded(gradient)
    # Values to 2^-4; the borders' neighbours may go either way.
    assert (np.abs(host(d_x) - held) <= 2.0**-3 * np.abs(held) + 2.0**-9).all()
    assert (np.abs(host(d_x) - held) <= 1e-6 * np.abs(held)).mean() > 0.98


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite(gpu, dtype):
    """A block with a NaN makes NaN of its row of the output alone, or, in a weight's block of 128 rows, of those columns."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    for rows in (3, 200):
        x, w = normal(torch, rows, 300, dtype, 51), normal(torch, 300, 300, dtype, 52)
        bad = x.clone()
        bad[1, 200] = float("inf")
        out = fp8.linear(bad, fp8.quantize(w, block=128))
        assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, *range(2, rows)]]).all()
        bad = w.clone()
        bad[140, 7] = float("nan")
        out = fp8.linear(x, fp8.quantize(bad, block=128))
        assert torch.isnan(out[:, 128:256]).all() and torch.isfinite(out[:, :128]).all()
        assert torch.isfinite(out[:, 256:]).all()
        out = fp8.gated(x, fp8.quantize(bad, block=128))  # ups 0 .. 149 are rows 150 ..: block 1 holds 128 .. 255
        assert torch.isnan(out[:, 128:]).all() and torch.isnan(out[:, :106]).all()
        # Not NaN; products of sums of some hundred each may pass fp16's 65504.
        assert not torch.isnan(out[:, 106:128]).any()


def test_extremes_of_the_gate(gpu):
    """Gates far out: silu goes to g, and to -0, without NaN."""
    import torch

    from triton_chip_benchmarks_amd import fp8

    gates = torch.tensor([-3e4, -200.0, -90.0, -20.0, -1.0, 0.0, 1.0, 20.0, 90.0, 3e4], device="cuda")
    # K = 256: x = (gate, 0.., 1, 0..), so that the two products are gate and 1, exact powers of codes or nearly.
    x = torch.zeros(10, 256, device="cuda")
    x[:, 0], x[:, 128] = gates, 1.0
    w = torch.zeros(2, 256, device="cuda")
    w[0, 0], w[1, 128] = 1.0, 1.0
    out = host(fp8.gated(x, fp8.quantize(w)))[:, 0]
    held = oracle.rounded(host(x))[:, 0]
    exact = held * oracle.sigmoid(held)
    assert (np.abs(out - exact) <= 8 * 2.0**-24 * np.abs(exact) + 2.0**-120).all()


def test_empty_calls(gpu):
    import torch

    from triton_chip_benchmarks_amd import fp8

    x = torch.randn(4, 64, device="cuda")
    weight = fp8.quantize(torch.randn(32, 64, device="cuda"), block=128)
    assert fp8.linear(x[:0], weight).shape == (0, 32)
    assert fp8.gated(x[:0], weight).shape == (0, 16)
    assert fp8.linear(x, fp8.empty(0, 64, 128)).shape == (4, 0)
    columns = fp8.quantize(torch.randn(32, 64, device="cuda"), columns=True, block=128)
    d_x, d_w = fp8.linear_backward(torch.empty(0, 32, device="cuda"), x[:0], columns)
    assert d_x.shape == (0, 64) and d_w.shape == (32, 64) and not d_w.any()
    d_x, d_w = fp8.gated_backward(torch.empty(0, 16, device="cuda"), torch.empty(0, 32, device="cuda"), x[:0], columns)
    assert d_x.shape == (0, 64) and d_w.shape == (32, 64) and not d_w.any()
