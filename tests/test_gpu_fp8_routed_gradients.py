"""Gradients of routed linear layers and gated pairs on FP8, by the calls that there are: the rows' gradient by a routed
product with the weights' columns, an expert's weight gradient by a call on its rows, a token's by the sum of its rows.
Against the float64 oracle, each step on its own input."""

import numpy as np
import pytest

from oracle import fp8 as oracle

pytestmark = pytest.mark.gpu

TOKENS, TOP, EXPERTS, N, K = 90, 2, 5, 72, 200


def host(tensor):
    return tensor.double().cpu().numpy()


def setting(torch, dtype, width):
    """(x, weights of the experts, their operands both ways, plan): expert 3 has no rows and expert 4 one."""
    from triton_chip_benchmarks_amd import fp8, routing

    generator = torch.Generator(device="cuda").manual_seed(width)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=generator).to(dtype)

    chosen = torch.stack([torch.randperm(3, device="cuda", generator=generator)[:TOP] for _ in range(TOKENS)]).int()
    chosen[7] = torch.tensor([4, -1])
    plan = routing.dispatch(chosen, EXPERTS)
    x, w = normal(TOKENS, K), [normal(width, K) / K**0.5 for _ in range(EXPERTS)]
    rows, columns = fp8.empty(width, K, fp8.BLOCK, experts=EXPERTS), fp8.empty(K, width, fp8.BLOCK, experts=EXPERTS)
    for e in range(EXPERTS):
        fp8.quantize_both(w[e], fp8.Packed(rows.codes[e], rows.scales[e], K, fp8.BLOCK),
                          fp8.Packed(columns.codes[e], columns.scales[e], width, fp8.BLOCK), block=fp8.BLOCK)
    return x, w, rows, columns, plan, normal


def near(torch, mine, exact, magnitudes, dtype, depth):
    """One rounding, and sums: of fp32, or to 2^-12 of the magnitudes by the FP8 instruction."""
    info = torch.finfo(dtype)
    off = (depth * 2.0**-24 if dtype is torch.float32 else 2.0**-12) * (1 + 2.0**-7) * magnitudes
    bound = off + info.eps / 2 * (np.abs(exact) + off) + info.smallest_normal * info.eps / 2
    assert (np.abs(host(mine) - exact) <= bound).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_linear(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import fp8, routing

    kind = getattr(torch, dtype)
    x, w, rows, columns, plan, normal = setting(torch, kind, N)
    ends, live = plan.offsets.tolist(), int(plan.offsets[-1])
    assert ends[3] == ends[4] == live - 1
    token = plan.order[:live].long() // TOP
    y = fp8.linear(x, rows, torch.zeros(TOKENS * TOP, N, device="cuda", dtype=kind), plan=plan)
    d_y = normal(TOKENS * TOP, N)
    d_rows = torch.zeros(TOKENS * TOP, K, device="cuda", dtype=kind)
    fp8.linear(d_y, columns, d_rows, plan=plan, sorted_rows=True)
    gathered = x[token].contiguous()
    for e, (first, last) in enumerate(zip(ends, ends[1:])):
        one = fp8.Packed(columns.codes[e], columns.scales[e], N, fp8.BLOCK)
        mine = fp8.linear_backward(d_y[first:last], gathered[first:last], one)
        if first == last:
            assert mine[0].shape == (0, K) and not mine[1].any()
            continue
        near(torch, y[first:last], *oracle.linear(host(gathered[first:last]), host(w[e])), kind, K)
        exact_x, exact_w = oracle.linear_backward(host(d_y[first:last]), host(gathered[first:last]), host(w[e]))
        near(torch, d_rows[first:last], *exact_x, kind, N)
        near(torch, mine[0], *exact_x, kind, N)
        near(torch, mine[1], *exact_w, kind, last - first + 128)
    assert not d_rows[live:].any() and not y[live:].any()
    d_x = routing.combine(d_rows, plan.slots, torch.ones(TOKENS, TOP, device="cuda"))
    exact = np.zeros((TOKENS, K))
    np.add.at(exact, token.cpu().numpy(), host(d_rows[:live]))
    size = np.zeros((TOKENS, K))
    np.add.at(size, token.cpu().numpy(), np.abs(host(d_rows[:live])))
    bound = 2 * 2.0**-24 * size + torch.finfo(kind).eps / 2 * np.abs(exact) * (1 + 2.0**-7) + 2.0**-24
    assert (np.abs(host(d_x) - exact) <= bound).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_gated(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import fp8

    kind = getattr(torch, dtype)
    x, w, rows, columns, plan, normal = setting(torch, kind, 2 * N)
    ends, live = plan.offsets.tolist(), int(plan.offsets[-1])
    token = plan.order[:live].long() // TOP
    gate_up = torch.zeros(TOKENS * TOP, 2 * N, device="cuda", dtype=kind)
    fp8.gated(x, rows, gate_up=gate_up, plan=plan)
    d_out, gathered = normal(TOKENS * TOP, N), x[token].contiguous()
    for e, (first, last) in enumerate(zip(ends, ends[1:])):
        one = fp8.Packed(columns.codes[e], columns.scales[e], 2 * N, fp8.BLOCK)
        d_x, d_w = fp8.gated_backward(d_out[first:last], gate_up[first:last], gathered[first:last], one)
        if first == last:
            assert d_x.shape == (0, K) and not d_w.any()
            continue
        near(torch, gate_up[first:last], *oracle.linear(host(gathered[first:last]), host(w[e])), kind, K)
        # The gradient of [gate | up] is within 16 roundings of fp32 of its terms: where a code's border, or a scale's, lies
        # between, the operands differ by what the exact values either side of it do.
        pair, d = host(gate_up[first:last]), host(d_out[first:last])
        exact = oracle.gate_backward(d, pair)
        g, u = np.split(pair, 2, axis=1)
        s = oracle.sigmoid(g)
        terms = np.concatenate([np.abs(d * u) * s * (1 + np.abs(g) * (1 - s)), np.abs(d * g) * s], axis=1)
        off = 16 * 2.0**-24 * terms
        weight, x_columns = oracle.rounded(host(w[e]), 128), oracle.rounded(host(gathered[first:last]).T).T

        def unsure(values, error):
            return np.abs(oracle.rounded(values + error) - oracle.rounded(values - error))

        for mine, held, other, slack, depth in (
                (d_x, oracle.rounded(exact), weight, unsure(exact, off), 2 * N),
                (d_w, oracle.rounded(exact.T), x_columns, unsure(exact.T, off.T), last - first + 128)):
            value, more = held @ other, slack @ np.abs(other)
            size = np.abs(held) @ np.abs(other) + more
            info = torch.finfo(kind)
            sums = (depth * 2.0**-24 if kind is torch.float32 else 2.0**-12) * (1 + 2.0**-7)
            bound = (more + sums * size) * (1 + info.eps) + info.eps / 2 * np.abs(value) \
                + info.smallest_normal * info.eps / 2
            assert (np.abs(host(mine) - value) <= bound).all()
