"""Routing, dispatch and combine on the GPU against the float64 oracle.

Choices and the sort are exact. Scores take a few roundings to 2^-23 and softmax sums at most 16 + 6 + 1 levels; an
exponential's relative error grows with the distance of its logit from the largest, which stays below 2^5 here.
"""

import numpy as np
import pytest

from oracle import routing as oracle

pytestmark = pytest.mark.gpu

UNIT = {"fp32": 2.0**-24, "fp16": 2.0**-11, "bf16": 2.0**-8}
SCORE_TOLERANCE = (32 + 24 + 8) * 2.0**-23


def _dtype(torch, name):
    return {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[name]


def _host(tensor):
    return tensor.double().cpu().numpy()


def _separated_logits(torch, dtype, tokens, experts, seed):
    """Logits of which no two of a token score alike in 32 bits: a shuffled ladder of steps of 1/64 around 0."""
    rng = np.random.default_rng(seed)
    ladder = (np.arange(experts) - experts // 2) / 64.0 * (64.0 / max(64, experts // 8))
    rows = np.stack([rng.permutation(ladder) for _ in range(tokens)]) if tokens else np.zeros((0, experts))
    return torch.tensor(rows).to(_dtype(torch, dtype)).cuda()


OPTIONS = [{"scores": "softmax"}, {"scores": "softmax", "renormalize": False, "scale": 2.0},
           {"scores": "sigmoid", "renormalize": False}, {"scores": "sigmoid", "scale": 2.5}]


def _oracle_options(options):
    return {("kind" if name == "scores" else name): value for name, value in options.items()}


@pytest.mark.parametrize("tokens,experts,top", [(1, 1, 1), (3, 2, 2), (5, 8, 2), (7, 63, 6), (9, 64, 8), (4, 65, 3),
                                                (6, 128, 8), (33, 256, 8), (3, 257, 4), (2, 512, 10), (5, 1000, 64),
                                                (2, 1024, 8)])
@pytest.mark.parametrize("options", OPTIONS)
def test_route_and_gradient(gpu, tokens, experts, top, options):
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"route {tokens}x{experts} top {top} {options}", flush=True)
    logits = _separated_logits(torch, "fp32", tokens, experts, seed=experts)
    chosen, weights = routing.route(logits, top, **options)
    expected, expected_weights = oracle.route(_host(logits), top, **_oracle_options(options))
    assert np.array_equal(chosen.cpu().numpy(), expected)
    assert np.allclose(_host(weights), expected_weights, rtol=SCORE_TOLERANCE, atol=0)
    g = torch.randn(tokens, top, device="cuda", generator=torch.Generator(device="cuda").manual_seed(top))
    d_logits = routing.route_backward(logits, chosen, g, **options)
    exact = oracle.route_backward(_host(logits), expected, _host(g), **_oracle_options(options))
    # Differences of terms up to scale * |g|, each with the scores' relative error.
    bound = 4 * SCORE_TOLERANCE * options.get("scale", 1.0) * np.abs(_host(g)).sum(axis=1, keepdims=True)
    assert (np.abs(_host(d_logits) - exact) <= bound).all()


@pytest.mark.parametrize("experts,top,groups,top_groups", [(8, 2, 1, 1), (60, 4, 4, 2), (64, 16, 16, 5), (128, 8, 1, 1),
                                                           (232, 7, 1, 1), (256, 8, 8, 4), (256, 17, 1, 1),
                                                           (300, 8, 1, 1)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_many_tokens(gpu, experts, top, groups, top_groups, scores):
    """Enough tokens for every form of the kernels, logits of few values: of equal ones the lower index, whatever
    lane holds it; the last tokens end inside a workgroup."""
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"route many x {experts} top {top} of {groups}/{top_groups}", flush=True)
    generator = torch.Generator(device="cuda").manual_seed(experts)
    tokens = 4099
    logits = (torch.randint(-40, 41, (tokens, experts), device="cuda", generator=generator) / 16.0).bfloat16()
    logits[5::7] = -float("inf")
    logits[:, 3] = -float("inf")
    options = {"scores": scores, "groups": groups, "top_groups": top_groups, "scale": 2.0}
    chosen, weights = routing.route(logits, top, **options)
    sample = np.r_[0:40, tokens - 40:tokens]
    expected, expected_weights = oracle.route(_host(logits)[sample], top, **_oracle_options(options))
    if groups == 1:  # sums of two scores of few values may tie in 64 bits and not in 32
        assert np.array_equal(chosen.cpu().numpy()[sample], expected)
        assert np.allclose(_host(weights)[sample], expected_weights, rtol=SCORE_TOLERANCE, atol=0)
    few = [routing.route(logits[i:i + 1000], top, **options) for i in range(0, tokens, 1000)]  # a wave a token
    assert torch.equal(chosen, torch.cat([part[0] for part in few]))
    assert torch.allclose(weights, torch.cat([part[1] for part in few]), rtol=SCORE_TOLERANCE, atol=0)
    g = torch.randn(tokens, top, device="cuda", generator=generator)
    d_logits = routing.route_backward(logits, chosen, g, scores=scores, scale=2.0)
    exact = oracle.route_backward(_host(logits)[sample], chosen.cpu().numpy()[sample], _host(g)[sample], kind=scores,
                                  scale=2.0)
    bound = 8 * SCORE_TOLERANCE * np.abs(_host(g)[sample]).sum(axis=1, keepdims=True) + UNIT["bf16"] * np.abs(exact)
    assert (np.abs(_host(d_logits)[sample] - exact) <= bound + 2.0**-25).all()


def test_a_lone_choice_has_no_gradient(gpu):
    """Renormalised, its weight is the scale whatever its logit."""
    import torch

    from triton_chip_benchmarks_amd import routing

    for tokens in (33, 5000):
        logits = torch.randn(tokens, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
        for scores in ("softmax", "sigmoid"):
            chosen, weights = routing.route(logits, 1, scores=scores, scale=1.5)
            assert (weights == 1.5).all()
            assert not routing.route_backward(logits, chosen, torch.ones_like(weights), scores=scores).any()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_route_takes_16_bit_logits_strided(gpu, dtype):
    import torch

    from triton_chip_benchmarks_amd import routing

    wide = torch.zeros(12, 301, device="cuda", dtype=_dtype(torch, dtype))
    logits = wide[1:11, 3:131]
    logits.copy_(_separated_logits(torch, dtype, 10, 128, seed=1))
    chosen, weights = routing.route(logits, 4)
    expected, expected_weights = oracle.route(_host(logits), 4)
    assert np.array_equal(chosen.cpu().numpy(), expected)  # 16-bit logits tie: the lower index first
    assert np.allclose(_host(weights), expected_weights, rtol=SCORE_TOLERANCE, atol=0)
    g = torch.ones(10, 4, device="cuda") * torch.tensor([1.0, -2.0, 0.5, 3.0], device="cuda")
    d_logits = routing.route_backward(logits, chosen, g)
    exact = oracle.route_backward(_host(logits), expected, _host(g))
    bound = 4 * SCORE_TOLERANCE * 6.5 + UNIT[dtype] * np.abs(exact) + 2.0**-25
    assert (np.abs(_host(d_logits) - exact) <= bound).all()


@pytest.mark.parametrize("groups,top_groups", [(8, 4), (8, 1), (4, 4), (64, 9), (2, 1), (16, 3)])
def test_groups_and_bias(gpu, groups, top_groups):
    import torch

    from triton_chip_benchmarks_amd import routing

    experts, top = 256 if groups < 64 else 128, 6
    logits = _separated_logits(torch, "fp32", 21, experts, seed=groups)
    # Steps of 2^-5 beside a ladder whose scores are never that far apart in exact multiples.
    bias = torch.tensor(np.random.default_rng(3).integers(-4, 5, experts) / 32.0 + np.arange(experts) * 1e-4).float().cuda()
    chosen, weights = routing.route(logits, top, bias, scores="sigmoid", groups=groups, top_groups=top_groups, scale=2.5)
    expected, expected_weights = oracle.route(_host(logits), top, _host(bias), kind="sigmoid", groups=groups,
                                              top_groups=top_groups, scale=2.5)
    assert np.array_equal(chosen.cpu().numpy(), expected)
    assert np.allclose(_host(weights), expected_weights, rtol=SCORE_TOLERANCE, atol=0)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_masked_tied_and_non_finite_logits(gpu, scores):
    import torch

    from triton_chip_benchmarks_amd import routing

    inf, nan = float("inf"), float("nan")
    logits = torch.zeros(8, 16)
    logits[0] = -inf                       # nothing left
    logits[1, 3:] = -inf                   # fewer experts than the choice takes
    logits[2] = 1.0                        # all tied
    logits[3, 7] = nan
    logits[4] = nan
    logits[5, 2], logits[5, 9] = 200.0, -200.0  # scores of 1 and 0
    logits[6] = torch.finfo(torch.float32).min  # the type's lowest value masks nothing
    logits[7, :] = -inf
    logits[7, 15] = 3.0
    for groups, top_groups in ((1, 1), (4, 2)):
        chosen, weights = routing.route(logits.cuda(), 5, scores=scores, groups=groups, top_groups=top_groups)
        expected, expected_weights = oracle.route(logits.numpy(), 5, kind=scores, groups=groups,
                                                  top_groups=top_groups)
        assert np.array_equal(chosen.cpu().numpy(), expected), (chosen, expected)
        assert np.allclose(_host(weights), expected_weights, rtol=SCORE_TOLERANCE, atol=1e-44, equal_nan=True)
    finite = [0, 1, 2, 5, 6, 7]
    chosen, _ = routing.route(logits[finite].cuda(), 5, scores=scores)
    g = torch.randn(len(finite), 5, generator=torch.Generator().manual_seed(0))
    d_logits = routing.route_backward(logits[finite].cuda(), chosen, g.cuda(), scores=scores)
    exact = oracle.route_backward(logits[finite].numpy(), chosen.cpu().numpy(), g.numpy(), kind=scores)
    assert np.allclose(_host(d_logits), exact, atol=8 * SCORE_TOLERANCE * 5 * 3)
    assert not d_logits[0].any() and torch.isfinite(d_logits).all()


def test_route_gradient_against_differences(gpu):
    """Central differences of the loss in fp32 weights: h = 2^-5, truncation h^2, rounding 2^-23 * |loss| / h."""
    import torch

    from triton_chip_benchmarks_amd import routing

    logits = _separated_logits(torch, "fp32", 4, 16, seed=5) * 40
    g = torch.tensor([[0.5, -1.0, 2.0]] * 4).cuda()
    for options in OPTIONS:
        chosen, _ = routing.route(logits, 3, **options)
        d_logits = routing.route_backward(logits, chosen, g, **options)
        h = 2.0**-5
        for t, e in ((0, int(chosen[0, 0])), (1, int(chosen[1, 2])), (2, int(logits[2].argmin())), (3, int(chosen[3, 1]))):
            loss = []
            for sign in (1, -1):
                moved = logits.clone()
                moved[t, e] += sign * h
                again, weights = routing.route(moved, 3, **options)
                assert torch.equal(again, chosen)
                loss.append((weights.double() * g).sum().item())
            scale = 3.5 * options.get("scale", 1.0)
            assert abs((loss[0] - loss[1]) / (2 * h) - d_logits[t, e].item()) <= scale * (h * h + 64 * 2.0**-23 / h)


@pytest.mark.parametrize("tokens,top,count", [(1, 1, 1), (1, 8, 8), (3, 2, 5), (64, 1, 3), (100, 6, 60), (512, 8, 256),
                                              (513, 8, 128), (3000, 4, 1000), (5000, 2, 1024), (9001, 7, 512)])
def test_dispatch(gpu, tokens, top, count):
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"dispatch {tokens}x{top} over {count}", flush=True)
    rng = np.random.default_rng(tokens)
    experts = rng.integers(-1, count, (tokens, top)).astype(np.int32)
    experts[rng.random((tokens, top)) < 0.3] = count - 1  # one expert has a third
    experts[-1, 0] = count + 5  # outside: no expert
    plan = routing.dispatch(torch.tensor(experts).cuda(), count)
    flat = np.where((experts < 0) | (experts >= count), count, experts).reshape(-1)
    order = np.argsort(flat, kind="stable")
    total = int((flat < count).sum())
    slots = np.empty_like(order)
    slots[order] = np.arange(order.size)
    assert plan.offsets.tolist() == np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=count)[:count])]).tolist()
    assert np.array_equal(plan.order.cpu().numpy(), np.where(np.arange(order.size) < total, order, -1))
    assert np.array_equal(plan.slots.cpu().numpy().reshape(-1), np.where(flat < count, slots, -1))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,top,n", [(1, 1, 1), (1, 8, 64), (3, 2, 7), (5, 6, 511), (4, 3, 512), (9, 4, 520),
                                          (2, 64, 100), (65, 2, 1500), (7, 8, 4096)])
def test_combine_and_gradients(gpu, dtype, tokens, top, n):
    import torch

    from triton_chip_benchmarks_amd import routing

    print(f"combine {dtype} {tokens}x{top}x{n}", flush=True)
    generator = torch.Generator(device="cuda").manual_seed(n)
    rows = tokens * top + 2
    y = torch.randn(rows, n, device="cuda", generator=generator).to(_dtype(torch, dtype))
    d_out = torch.randn(tokens, n, device="cuda", generator=generator).to(y.dtype)
    weights = torch.randn(tokens, top, device="cuda", generator=generator)
    slots = torch.tensor(np.random.default_rng(n).permutation(rows)[:tokens * top].reshape(tokens, top).astype(np.int32))
    slots[tokens // 2, top - 1] = -1
    slots[-1, 0] = rows  # outside
    y_nan = y.clone()
    named = set(slots.reshape(-1).tolist())
    for row in range(rows):
        if row not in named:
            y_nan[row] = float("nan")  # rows no slot names are not read
    slots, host_slots = slots.cuda(), slots.numpy()
    out = routing.combine(y_nan, slots, weights)
    expected, size = oracle.combine(_host(y), host_slots, _host(weights))
    unit = UNIT[dtype]
    assert (np.abs(_host(out) - expected) <= top * 2.0**-23 * size + unit * np.abs(expected) * 1.01 + 2.0**-25).all()
    d_y = torch.full_like(y, 7.0)
    d_y, d_weights = routing.combine_backward(d_out, y_nan, slots, weights, d_y)
    exact_y, exact_weights, size = oracle.combine_backward(_host(d_out), _host(y), host_slots, _host(weights))
    for row in range(rows):
        if row in named:
            assert (np.abs(_host(d_y[row]) - exact_y[row]) <= (unit + 2.0**-23) * np.abs(exact_y[row]) + 2.0**-25).all()
        else:
            assert (d_y[row] == 7).all()
    assert (np.abs(_host(d_weights) - exact_weights) <= (n / 64 + 16) * 2.0**-23 * size).all()


def test_a_layer_in_a_graph_replays_to_the_eager_result(gpu):
    """Route, dispatch, both products, combine captured once; replays with new inputs and eager work in between."""
    import torch

    from triton_chip_benchmarks_amd import mx, routing

    tokens, experts, top, hidden, inner = 24, 8, 2, 256, 192
    generator = torch.Generator(device="cuda").manual_seed(0)
    up, down = mx.empty(inner, hidden, experts=experts), mx.empty(hidden, inner, experts=experts)
    for weight, n, k in ((up, inner, hidden), (down, hidden, inner)):
        for e in range(experts):
            mx.quantize(torch.randn(n, k, device="cuda", generator=generator) / k**0.5,
                        mx.Packed(weight.codes[e], weight.scales[e], k))
    x = torch.empty(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    logits = torch.empty(tokens, experts, device="cuda")
    plan = routing.empty_plan(tokens, top, experts)
    rows = tokens * top
    buffers = {"experts": torch.empty(tokens, top, device="cuda", dtype=torch.int32),
               "weights": torch.empty(tokens, top, device="cuda")}
    h, y = torch.empty(rows, inner, device="cuda", dtype=x.dtype), torch.empty(rows, hidden, device="cuda", dtype=x.dtype)
    out = torch.empty_like(x)
    spaces = (mx.linear_workspace(rows, inner, hidden, x.dtype, experts),
              mx.linear_workspace(rows, hidden, inner, x.dtype, experts))

    def layer():
        chosen, weights = routing.route(logits, top, **buffers)
        routing.dispatch(chosen, experts, plan)
        mx.linear(x, up, h, plan=plan, workspace=spaces[0])
        mx.linear(h, down, y, plan=plan, sorted_rows=True, workspace=spaces[1])
        routing.combine(y, plan.slots, weights, out)

    def fill():
        x.copy_(torch.randn(tokens, hidden, device="cuda", generator=generator))
        logits.copy_(torch.randn(tokens, experts, device="cuda", generator=generator))

    fill()
    layer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for _ in range(4):
        fill()
        layer()
        torch.cuda.synchronize()
        eager = out.clone()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.isfinite(out).all()
