"""GPU test of the mixture-of-experts command: every step runs, together they agree with float64 products, and the
whole layer gives the same output replayed from a graph."""

import json

import numpy as np
import pytest

from oracle import mx as oracle_mx
from oracle import routing as oracle_routing

pytestmark = pytest.mark.gpu


def test_quick_run_times_every_step_and_checks_the_layer(gpu, tmp_path):
    from triton_chip_benchmarks_amd import experts

    output = tmp_path / "experts.json"
    assert experts.main(["--quick", "--output", str(output)]) == 0
    rows = json.loads(output.read_text())["results"]
    assert [row["step"] for row in rows] == [*experts.Layer.STEPS, "layer"]
    assert all(row["median_ms"] > 0 and row["normwise_error"] <= experts.TOLERANCE for row in rows)


@pytest.mark.parametrize("tokens,hidden,inner,count,top", [(1, 256, 96, 8, 2), (37, 320, 160, 6, 3), (70, 96, 33, 5, 1)])
def test_layer_agrees_with_the_oracle_and_with_its_graph(gpu, tokens, hidden, inner, count, top):
    import torch

    from triton_chip_benchmarks_amd import experts, mx

    print(f"layer {tokens}x{hidden}x{inner} experts={count} top={top}", flush=True)
    layer = experts.Layer(tokens, hidden, inner, count, top, torch.bfloat16, seed=tokens)
    eager = layer.run().clone()

    def weight(packed, e):
        return mx.dequantize(mx.Packed(packed.codes[e], packed.scales[e], packed.k)).double().cpu().numpy()

    chosen, weights = oracle_routing.route(layer.logits.double().cpu().numpy(), top)
    assert np.array_equal(layer.experts.cpu().numpy(), chosen)
    x = oracle_mx.rounded(layer.x.double().cpu().numpy())
    expected = np.zeros((tokens, hidden))
    for t in range(tokens):
        for share, e in zip(weights[t], chosen[t]):
            gate, up = np.split(weight(layer.up_weight, e) @ x[t], 2)
            inside = oracle_mx.rounded((gate / (1 + np.exp(-gate)) * up)[None])[0]
            expected[t] += share * (weight(layer.down_weight, e) @ inside)
    # bf16 gate, up, silu and product: four roundings of 2^-9 (2^-7 together). Each may move an E2M1 code by one
    # step, at most half of a value, where it lies within that of a code's limit (share about 2^-7 * 4): an error of
    # 1/2 * sqrt(2^-5) = 0.09 of the norm at most, before the averaging over rows.
    error = np.linalg.norm(eager.double().cpu().numpy() - expected) / np.linalg.norm(expected)
    assert error < 0.1, error

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run()
    for _ in range(3):
        layer.out.fill_(float("nan"))
        layer.experts.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layer.out, eager)


@pytest.mark.parametrize("tokens,n,k,count,top", [(3, 96, 40, 6, 2), (150, 72, 96, 4, 3)])
def test_gradients_of_routed_rows_through_the_same_calls(gpu, tokens, n, k, count, top):
    """The input's gradient is a routed product with the weights' columns and a sum over a token's choices; an
    expert's weight gradient the linear layer's of its rows."""
    import torch

    from triton_chip_benchmarks_amd import mx, routing

    print(f"routed gradients {tokens}x{n}x{k} experts={count} top={top}", flush=True)
    generator = torch.Generator(device="cuda").manual_seed(tokens)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=generator)

    def host(tensor):
        return tensor.double().cpu().numpy()

    def close(got, expected, size, depth):
        # fp32 sums as everywhere: a rounding for each of depth / 32 steps and 16 joins.
        assert (np.abs(host(got) - expected) <= ((depth / 32 + 16) * 2.0**-23 + 2.0**-24) * size + 2.0**-149).all()

    x, w, logits = normal(tokens, k), normal(count, n, k), normal(tokens, count)
    logits[1] = float("-inf")  # a token without experts
    chosen, _ = routing.route(logits, top)
    plan = routing.dispatch(chosen, count)
    offsets, order = plan.offsets.tolist(), plan.order.long()
    d_y = normal(tokens * top, n)
    columns = mx.empty(k, n, experts=count)
    for e in range(count):
        mx.quantize(w[e], mx.Packed(columns.codes[e], columns.scales[e], n), columns=True)
    d_rows = mx.linear(d_y, columns, plan=plan, sorted_rows=True)
    d_x = routing.combine(d_rows, plan.slots, torch.ones(tokens, top, device="cuda"))
    expected, size = np.zeros((tokens, k)), np.zeros((tokens, k))
    for e, (first, last) in enumerate(zip(offsets, offsets[1:])):
        token = order[first:last] // top
        part = mx.Packed(columns.codes[e], columns.scales[e], n)
        _, d_w = mx.linear_backward(d_y[first:last], x[token], part)
        assert d_w.shape == (n, k)
        if first == last:
            assert not d_w.any()
            continue
        (ex, sx), (ew, sw) = oracle_mx.linear_backward(host(d_y[first:last]), host(x[token]), host(w[e]))
        close(d_w, ew, sw, last - first)
        for t, row, rounding in zip(token.tolist(), ex, sx):
            expected[t] += row
            size[t] += rounding
    # A token's `top` rows are rounded to fp32 and added.
    close(d_x, expected, size, n + 32 * top)
    assert not d_x[1].any()
