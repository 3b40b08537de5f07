"""FP8 operators and the norm off the current stream, in graphs, and two at once: what they allocate is their stream's
memory, and the results are those of the same calls one after the other."""

import pytest

pytestmark = pytest.mark.gpu


def _calls(torch, rows=40):
    from triton_chip_benchmarks_amd import fp8, norm, routing

    generator = torch.Generator(device="cuda").manual_seed(rows)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=generator).bfloat16()

    def parts(*operands):
        return tuple(tensor for operand in operands for tensor in (operand.codes, operand.scales))

    x, w, pair_w, d_y, d_h = normal(rows, 96), normal(64, 96), normal(144, 96), normal(rows, 64), normal(rows, 72)
    weight, columns = fp8.quantize_both(w, block=128)
    pair, pair_columns = fp8.quantize_both(pair_w, block=128)
    up = fp8.empty(144, 96, 128, experts=8)
    for e in range(8):
        fp8.quantize(normal(144, 96), fp8.Packed(up.codes[e], up.scales[e], 96, 128), block=128)
    chosen, _ = routing.route(normal(rows, 8), 2)
    plan = routing.dispatch(chosen, 8)
    operand, gate_up, scale = fp8.quantize(x), normal(rows, 144), normal(96)
    routed = fp8.quantize(normal(2 * rows, 96))
    kept = torch.empty(rows, 144, device="cuda", dtype=torch.bfloat16)
    out = fp8.empty(rows, 72)

    def to_operand(stream):
        fp8.gated(x, pair, packed=out, stream=stream)
        return tuple(tensor.view(torch.uint8) for tensor in parts(out))

    return {
        "quantize": lambda stream: parts(fp8.quantize(x, stream=stream)),
        "quantize_both": lambda stream: parts(*fp8.quantize_both(x, stream=stream)),
        "dequantize": lambda stream: (fp8.dequantize(weight, stream=stream),),
        "product": lambda stream: (fp8.product(operand, weight, stream=stream),),
        "linear": lambda stream: (fp8.linear(x, weight, stream=stream),),
        "linear_backward": lambda stream: fp8.linear_backward(d_y, x, columns, stream=stream),
        "gated": lambda stream: (fp8.gated(x, pair, gate_up=kept, stream=stream), kept),
        "gated_of_an_operand": lambda stream: (fp8.gated(operand, pair, stream=stream),),
        "gated_to_an_operand": to_operand,
        "gated_routed": lambda stream: (fp8.gated(x, up, plan=plan, stream=stream),),
        "product_routed": lambda stream: (fp8.product(routed, up, offsets=plan.offsets, stream=stream),),
        "gated_backward": lambda stream: fp8.gated_backward(d_h, gate_up, x, pair_columns, stream=stream),
        "norm": lambda stream: norm.rms_norm(x, scale, residual=x, stream=stream)[::2],
        "norm_backward": lambda stream: norm.rms_norm_backward(x, x, scale, d_total=x, stream=stream),
    }


def _bits(torch, tensors):
    return [tensor.contiguous().view(torch.uint8).clone() for tensor in tensors]


@pytest.mark.parametrize("rows", [40, 1300])
def test_outputs_and_workspaces_are_the_streams_memory(gpu, monkeypatch, rows):
    import torch

    from triton_chip_benchmarks_amd import fp8, mx

    calls = _calls(torch, rows)
    side = torch.cuda.Stream()
    made = []

    def recorded(*arguments):
        made.append(allocate(*arguments))
        return made[-1]

    allocate = mx.allocate
    monkeypatch.setattr(mx, "allocate", recorded)
    monkeypatch.setattr(fp8, "allocate", recorded)
    for name, call in calls.items():
        print(f"streams {name} {rows}", flush=True)
        here = _bits(torch, call(None))
        torch.cuda.synchronize()
        del made[:]
        there = call(side)
        torch.cuda.synchronize()
        segments = torch.cuda.memory_snapshot()
        for tensor in made:
            if tensor.numel():
                start = tensor.data_ptr()
                owner = [s["stream"] for s in segments if s["address"] <= start < s["address"] + s["total_size"]]
                assert owner == [side.cuda_stream], name
        assert all(torch.equal(mine, theirs) for mine, theirs in zip(here, _bits(torch, there))), name


@pytest.mark.parametrize("rows", [40, 1300])
def test_graphs_give_the_same_on_every_replay(gpu, rows):
    import torch

    for name, call in _calls(torch, rows).items():
        print(f"graph {name} {rows}", flush=True)
        eager = _bits(torch, call(None))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = call(None)
        for _ in range(3):
            for tensor in outputs:
                tensor.view(torch.uint8).fill_(0x5a)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(mine, theirs) for mine, theirs in zip(eager, _bits(torch, outputs))), name
            again = call(None)  # eager work between the replays
            assert all(torch.equal(mine, theirs) for mine, theirs in zip(eager, _bits(torch, again))), name


def test_two_at_once_with_workspaces_of_their_own(gpu):
    """Calls of two streams that run together, the persistent kernels among them, and two graphs replayed so."""
    import torch

    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    sets = [_calls(torch, rows) for rows in (1300, 1700)]
    for name in sets[0]:
        print(f"together {name}", flush=True)
        expected = [_bits(torch, calls[name](None)) for calls in sets]
        torch.cuda.synchronize()
        results = [calls[name](side) for calls, side in zip(sets, sides) for _ in range(1)]
        torch.cuda.synchronize()
        for mine, theirs in zip(expected, results):
            assert all(torch.equal(a, b) for a, b in zip(mine, _bits(torch, theirs))), name
        graphs, outputs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
        for graph, calls in zip(graphs, sets):
            with torch.cuda.graph(graph):
                outputs.append(calls[name](None))
        for _ in range(3):
            for tensors in outputs:
                for tensor in tensors:
                    tensor.view(torch.uint8).fill_(0x5a)
            torch.cuda.synchronize()
            for graph, side in zip(graphs, sides):
                with torch.cuda.stream(side):
                    graph.replay()
            torch.cuda.synchronize()
            for mine, theirs in zip(expected, outputs):
                assert all(torch.equal(a, b) for a, b in zip(mine, _bits(torch, theirs))), name


def test_gradients_of_no_rows_are_cleared_in_the_streams_order(gpu):
    import torch

    from triton_chip_benchmarks_amd import fp8, norm

    side = torch.cuda.Stream()
    columns = fp8.quantize(torch.ones(64, 96, device="cuda", dtype=torch.bfloat16), columns=True, block=128)
    d_weight = torch.zeros(64, 96, device="cuda", dtype=torch.bfloat16)
    d_scale = torch.zeros(96, device="cuda", dtype=torch.bfloat16)
    d_out, d_inner, gate_up, x = (torch.empty(0, width, device="cuda", dtype=torch.bfloat16)
                                  for width in (64, 32, 64, 96))

    def late_ones():
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # about 10 ms
            d_weight.fill_(1.0)
            d_scale.fill_(1.0)

    late_ones()
    fp8.linear_backward(d_out, x, columns, d_weight=d_weight, stream=side)
    norm.rms_norm_backward(x, x, d_scale.clone(), d_weight=d_scale, stream=side)
    torch.cuda.synchronize()
    assert (d_weight == 0).all() and (d_scale == 0).all()
    late_ones()
    fp8.gated_backward(d_inner, gate_up, x, columns, d_weight=d_weight, stream=side)
    torch.cuda.synchronize()
    assert (d_weight == 0).all()
