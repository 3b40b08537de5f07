"""A feed-forward block on FP8, as a training step and as a routed serving step run it: norm, gated pair and projection
with their gradients through one another, in a graph too, against float64; and rows that name an expert twice."""

import numpy as np
import pytest

from oracle import fp8 as o8
from oracle import norm as on

pytestmark = pytest.mark.gpu

SIZES = [(1, 72, 160), (33, 200, 130), (300, 264, 520)]


def _host(tensor):
    return tensor.double().cpu().numpy()


def _block(torch, rows, inner, hidden, kind):
    """One training step as calls, its tensors, and its results by name."""
    from triton_chip_benchmarks_amd import fp8, norm

    generator = torch.Generator(device="cuda").manual_seed(rows)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=generator).to(kind)

    x, residual, g, d_out = normal(rows, hidden), normal(rows, hidden), normal(hidden), normal(rows, hidden)
    up, down = normal(2 * inner, hidden) / hidden**0.5, normal(hidden, inner) / inner**0.5
    gate_up = torch.empty(rows, 2 * inner, device="cuda", dtype=kind)

    def run():
        (up_rows, up_columns), (down_rows, down_columns) = (fp8.quantize_both(w, block=fp8.BLOCK) for w in (up, down))
        normed = norm.rms_norm(x, g, residual=residual)
        h = fp8.gated(normed.out, up_rows, gate_up=gate_up)
        out = fp8.linear(h, down_rows)
        d_h, d_down = fp8.linear_backward(d_out, h, down_columns)
        d_normed, d_up = fp8.gated_backward(d_h, gate_up, normed.out, up_columns)
        d_x, d_g = norm.rms_norm_backward(d_normed, normed.total, g, d_total=d_out)
        return {"total": normed.total, "normed": normed.out, "gate_up": gate_up, "h": h, "out": out, "d_h": d_h,
                "d_down": d_down, "d_normed": d_normed, "d_up": d_up, "d_x": d_x, "d_g": d_g}

    return run, {"x": x, "residual": residual, "g": g, "d_out": d_out, "up": up, "down": down}


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,inner,hidden", SIZES)
def test_training_step(gpu, dtype, rows, inner, hidden):
    """Each step against the oracle on its own input, so that a rounding is no error of the steps behind it."""
    import torch

    kind, unit = {"bf16": (torch.bfloat16, 2.0**-8), "fp16": (torch.float16, 2.0**-11),
                  "fp32": (torch.float32, 2.0**-24)}[dtype]
    print(f"block {dtype} {rows}x{inner}x{hidden}", flush=True)
    run, given = _block(torch, rows, inner, hidden, kind)
    results = run()
    got, at = ({name: _host(tensor) for name, tensor in part.items()} for part in (results, given))
    # Sums of products: in fp32 for fp32 outputs, of the matrix cores' FP8 instruction (2^-12 of the magnitudes) for others.
    sums = (max(inner, hidden, rows) / 16 + 24) * 2.0**-23 if dtype == "fp32" else 2.0**-12

    def near(name, exact, size, share=sums):
        bound = share * size
        assert (np.abs(got[name] - exact) <= bound + unit * (np.abs(exact) + bound) + 2.0**-25).all(), name

    near("total", at["x"] + at["residual"], 0)
    exact = on.rms_norm(got["total"], at["g"], 1e-6)
    near("normed", exact, np.abs(exact), 8 * 2.0**-23)  # the mean's, root's, quotient's and two products' roundings
    near("gate_up", *o8.linear(got["normed"], at["up"]))
    # h is made of the sums, not of gate_up's roundings: of the exact sums within their own errors.
    pair, size = o8.linear(got["normed"], at["up"])
    gate, by = np.split(pair, 2, axis=1)
    gate_size, by_size = np.split(size, 2, axis=1)
    silu = gate * o8.sigmoid(gate)
    # |silu'| <= 1.1; 16 roundings of fp32 in the sigmoid and the products.
    near("h", silu * by, 1.1 * gate_size * (np.abs(by) + sums * by_size) + np.abs(silu) * by_size
         + (16 * 2.0**-23 / sums) * np.abs(silu * by))
    near("out", *o8.linear(got["h"], at["down"]))
    (d_h, d_h_size), (d_down, d_down_size) = o8.linear_backward(at["d_out"], got["h"], at["down"])
    near("d_h", d_h, d_h_size)
    near("d_down", d_down, d_down_size)
    # The gradient of [gate | up] in fp32 may lie beside a code's border where the exact one does: 2^-4 of a value, for few
    # of them; a normwise bound of 2^-7 counts a hundredth of them moved.
    d_pair = o8.gate_backward(got["d_h"], got["gate_up"])
    for name, exact in zip(("d_normed", "d_up"), (part[0] for part in o8.linear_backward(d_pair, got["normed"],
                                                                                       at["up"]))):
        error = np.linalg.norm(got[name] - exact) / np.linalg.norm(exact)
        assert error <= 2.0**-7, (name, error)
    d_x, d_g = on.rms_norm_backward(got["d_normed"], got["total"], at["g"], 1e-6, at["d_out"])
    inverse = 1 / np.sqrt((got["total"]**2).mean(axis=1, keepdims=True) + 1e-6)
    terms = np.abs(got["d_normed"] * at["g"]) * inverse
    along = (np.abs(got["d_normed"] * at["g"] * got["total"])).mean(axis=1, keepdims=True)
    size = terms + np.abs(got["total"]) * inverse**3 * along + np.abs(at["d_out"])
    near("d_x", d_x, size, (hidden / 64 + 24) * 2.0**-23)
    near("d_g", d_g, (np.abs(got["d_normed"] * got["total"]) * inverse).sum(0), (rows / 64 + 24) * 2.0**-23)

    eager = {name: tensor.clone() for name, tensor in results.items()}
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        for tensor in captured.values():
            tensor.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for name, tensor in captured.items():
            assert torch.equal(tensor, eager[name]), name
        run()  # eager work between the replays


def test_a_token_that_names_an_expert_twice_has_two_rows(gpu):
    import torch

    from triton_chip_benchmarks_amd import fp8, routing

    generator = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(9, 160, device="cuda", generator=generator).bfloat16()
    weight = fp8.empty(2 * 72, 160, fp8.BLOCK, experts=4)
    for e in range(4):
        fp8.quantize(torch.randn(2 * 72, 160, device="cuda", generator=generator).bfloat16(),
                     fp8.Packed(weight.codes[e], weight.scales[e], 160, fp8.BLOCK), block=fp8.BLOCK)
    chosen = torch.tensor([[3, 3], [0, 3], [-1, 2], [2, 2], [-1, -1], [0, 0], [3, 3], [1, 7], [0, -5]],
                          dtype=torch.int32, device="cuda")  # -1, -5 and 7: none
    plan = routing.dispatch(chosen, 4)
    out = torch.full((18, 72), 7.0, device="cuda", dtype=torch.bfloat16)
    fp8.gated(x, weight, out, plan=plan)
    slots, used = plan.slots.tolist(), int(plan.offsets[-1])
    assert used == 13 and (out[used:] == 7).all()
    for t, row in enumerate(chosen.tolist()):
        for e, slot in zip(row, slots[t]):
            if not 0 <= e < 4:
                assert slot < 0
                continue
            one = fp8.Packed(weight.codes[e], weight.scales[e], 160, fp8.BLOCK)
            exact = o8.gate(o8.rounded(_host(x[t:t + 1])) @ _host(fp8.dequantize(one)).T)
            # bf16's rounding, and sums to 2^-12 of magnitudes that a cancelling sum may pass by far: 2^-5 of the row's
            # largest.
            assert np.abs(_host(out[slot]) - exact[0]).max() <= 2.0**-5 * np.abs(exact).max(), (t, e)
