"""GPU tests of the mixture-of-experts command on FP8: every step runs, together they agree with float64 products, a graph
gives the same output on every replay, and the command's own check tells a wrong weight."""

import json

import numpy as np
import pytest

from oracle import fp8 as oracle_fp8
from oracle import norm as oracle_norm
from oracle import routing as oracle_routing

pytestmark = pytest.mark.gpu

SIZES = [(1, 256, 96, 8, 2), (37, 320, 160, 6, 3), (70, 96, 33, 5, 1), (300, 520, 136, 4, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_quick_run_times_every_step_and_checks_the_layer(gpu, tmp_path, dtype):
    from triton_chip_benchmarks_amd import experts

    output = tmp_path / "experts.json"
    assert experts.main(["--quick", "--weights", "fp8", "--dtype", dtype, "--output", str(output)]) == 0
    rows = json.loads(output.read_text())["results"]
    assert [row["step"] for row in rows] == [*experts.Fp8Layer.STEPS, "layer"]
    assert all(row["weights"] == "fp8" and row["median_ms"] > 0 and row["normwise_error"] <= experts.TOLERANCE
               for row in rows)


@pytest.mark.parametrize("tokens,hidden,inner,count,top", SIZES)
def test_layer_agrees_with_the_oracle_and_with_its_graph(gpu, tokens, hidden, inner, count, top):
    import torch

    from triton_chip_benchmarks_amd import experts

    print(f"fp8 layer {tokens}x{hidden}x{inner} experts={count} top={top}", flush=True)
    layer = experts.Fp8Layer(tokens, hidden, inner, count, top, torch.bfloat16, seed=tokens)
    eager = layer.run().clone()
    assert experts.check(layer) <= experts.TOLERANCE

    def host(tensor):
        return tensor.double().cpu().numpy()

    chosen, weights = oracle_routing.route(host(layer.logits), top)
    assert np.array_equal(layer.experts.cpu().numpy(), chosen)
    total = host((layer.before.float() + layer.x.float()).bfloat16())
    assert np.array_equal(host(layer.total), total)
    x = oracle_fp8.rounded(oracle_norm.rms_norm(total, host(layer.norm_weight), 1e-6))
    expected = np.zeros((tokens, hidden))
    up, down = ([host(experts._values(packed, e)) for e in range(count)] for packed in (layer.up_weight,
                                                                                         layer.down_weight))
    for t in range(tokens):
        for share, e in zip(weights[t], chosen[t]):
            inside = oracle_fp8.rounded(oracle_fp8.gate((up[e] @ x[t])[None]))[0]
            expected[t] += share * (down[e] @ inside)
    # The norm's rounding to bf16 (2^-8) moves a code of x by a step, 2^-3 of the value, where it lies within that of the
    # border (a share of about 2^-8 * 2^4 / 2 of them), and so do the products' roundings for the inner operand: an error
    # of 2^-3 * sqrt(2^-5) = 0.022 each of the norm, 0.05 with what the gate adds to the first.
    error = np.linalg.norm(host(eager) - expected) / np.linalg.norm(expected)
    assert error < 0.05, error

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run()
    for _ in range(3):
        for tensor in (layer.out, layer.normed, layer.total, layer.y):
            tensor.fill_(float("nan"))
        if layer.few:
            layer.inner.fill_(float("nan"))
        else:
            layer.inner.codes.view(torch.uint8).fill_(0x7f)
        layer.experts.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layer.out, eager)


@pytest.mark.parametrize("tokens", [5, 40])
@pytest.mark.parametrize("which", ["up_weight", "down_weight"])
def test_another_experts_weight_does_not_pass_the_check(gpu, monkeypatch, which, tokens):
    import torch

    from triton_chip_benchmarks_amd import experts

    layer = experts.Fp8Layer(tokens, 256, 96, 8, 2, torch.bfloat16)
    assert layer.few == (tokens == 5)
    right = experts._values
    monkeypatch.setattr(experts, "_values", lambda packed, e: right(packed, (e + 1) % 8) if packed is getattr(layer, which)
                        else right(packed, e))
    assert experts.check(layer) > 0.3
