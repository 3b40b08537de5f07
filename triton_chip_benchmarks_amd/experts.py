#!/usr/bin/env python3
"""One mixture-of-experts layer on the MXFP4 matrix cores, step by step and whole.

A serving step of such a layer calls, on the tokens' activations and the
router's logits:
  route      the experts of every token and their weights
  dispatch   the sort of the choices by expert
  up         gate and up projection, quantised activations times each expert's weight
  activate   silu(gate) * up (torch)
  down       the projection back
  combine    the weighted sum of the experts' outputs
Each step and the whole layer, captured into HIP graphs, are timed by device events
(common.measure) and priced against what they have to read, write and compute;
every step's output is checked against float64 products and sums of its input.
The replays follow one another, so weights that fit the 256 MiB memory-side cache
(those of a few tokens) are read from there, and their share of the bound, which
is HBM's, may pass 100%.
The reference has no counterpart: its matrix rows price products alone, not what
a layer needs around them.
"""

from __future__ import annotations

import argparse
from pathlib import Path
import sys

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
    from triton_chip_benchmarks_amd import mx, roofline, routing
    from triton_chip_benchmarks_amd.common import (add_common_arguments, emit_results, measure, positive_int,
                                                   setup_device)
else:
    from . import mx, roofline, routing
    from .common import add_common_arguments, emit_results, measure, positive_int, setup_device


class Layer:
    """Weights, buffers and the steps of a layer; `run` is one pass. Nothing is allocated after construction."""

    def __init__(self, tokens: int, hidden: int, inner: int, experts: int, top: int, dtype, device="cuda",
                 seed: int = 0):
        import torch

        self.shape = {"tokens": tokens, "hidden": hidden, "inner": inner, "experts": experts, "top": top}
        generator = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape):
            return torch.randn(shape, device=device, generator=generator)

        def weight(n, k):
            packed = mx.empty(n, k, device, experts)
            for e in range(experts):
                mx.quantize(normal(n, k) / k**0.5, mx.Packed(packed.codes[e], packed.scales[e], k))
            return packed

        self.up_weight, self.down_weight = weight(2 * inner, hidden), weight(hidden, inner)
        self.x, self.logits = normal(tokens, hidden).to(dtype), 1.5 * normal(tokens, experts)
        rows = tokens * top

        def buffer(*shape, of=dtype):
            return torch.empty(shape, device=device, dtype=of)

        self.experts, self.weights = buffer(tokens, top, of=torch.int32), buffer(tokens, top, of=torch.float32)
        self.plan = routing.empty_plan(tokens, top, experts, device)
        self.gate_up, self.gate, self.y = buffer(rows, 2 * inner), buffer(rows, inner), buffer(rows, hidden)
        self.out = buffer(tokens, hidden)
        self.up_space = mx.linear_workspace(rows, 2 * inner, hidden, dtype, experts, device)
        self.down_space = mx.linear_workspace(rows, hidden, inner, dtype, experts, device)

    def route(self):
        routing.route(self.logits, self.shape["top"], experts=self.experts, weights=self.weights)

    def dispatch(self):
        routing.dispatch(self.experts, self.shape["experts"], self.plan)

    def up(self):
        mx.linear(self.x, self.up_weight, self.gate_up, plan=self.plan, workspace=self.up_space)

    def activate(self):
        import torch

        gate, up = self.gate_up.chunk(2, dim=1)
        torch.ops.aten.silu.out(gate, out=self.gate)
        self.gate.mul_(up)

    def down(self):
        mx.linear(self.gate, self.down_weight, self.y, plan=self.plan, sorted_rows=True, workspace=self.down_space)

    def combine(self):
        routing.combine(self.y, self.plan.slots, self.weights, self.out)

    STEPS = ("route", "dispatch", "up", "activate", "down", "combine")

    def run(self):
        for step in self.STEPS:
            getattr(self, step)()
        return self.out


def work(layer: Layer, step: str) -> dict:
    """Bytes that a step has to move and operations it has to make, each input read and each output written once."""
    tokens, hidden, inner, experts, top = (layer.shape[name] for name in
                                           ("tokens", "hidden", "inner", "experts", "top"))
    item, rows = layer.x.element_size(), tokens * top
    used = int((layer.plan.offsets[1:] > layer.plan.offsets[:-1]).sum())

    def packed(n, k):
        return n * -(-k // mx.GROUP) * (mx.GROUP // 2 + 1)

    return {"route": {"bytes": tokens * experts * 4 + rows * 8, "flops": 4 * tokens * experts},
            "dispatch": {"bytes": 12 * rows + 4 * (experts + 1), "flops": 0},
            "up": {"bytes": (tokens * hidden + rows * 2 * inner) * item + used * packed(2 * inner, hidden),
                   "flops": 4 * rows * inner * hidden},
            "activate": {"bytes": 3 * rows * inner * item, "flops": 4 * rows * inner},
            "down": {"bytes": (rows * inner + rows * hidden) * item + used * packed(hidden, inner),
                     "flops": 2 * rows * inner * hidden},
            "combine": {"bytes": (rows + tokens) * hidden * item + 8 * rows, "flops": 2 * rows * hidden}}[step]


def _values(packed, e: int):
    return mx.dequantize(mx.Packed(packed.codes[e], packed.scales[e], packed.k)).double()


def check(layer: Layer, tokens: int = 32) -> float:
    """Normwise distance of the first tokens' rows from float64 products and sums, the largest of the steps'. Each step
    is compared on the layer's own input to it: a value of 16 bits that rounds to its neighbour is then no error of the
    steps behind, where it may move an E2M1 code by as much as the code."""
    import torch

    layer.run()
    tokens = min(tokens, layer.shape["tokens"])
    x = mx.dequantize(mx.quantize(layer.x[:tokens])).double()
    expected = torch.zeros((tokens, layer.shape["hidden"]), dtype=torch.float64, device=layer.x.device)
    squares = {step: [0.0, 0.0] for step in ("up", "activate", "down", "combine")}

    def compare(step, got, exact):
        squares[step][0] += float((got.double() - exact).square().sum())
        squares[step][1] += float(exact.square().sum())

    for t, (shares, chosen, slots) in enumerate(zip(layer.weights[:tokens].tolist(), layer.experts[:tokens].tolist(),
                                                    layer.plan.slots[:tokens].tolist())):
        for share, e, slot in zip(shares, chosen, slots):
            if e < 0:
                continue
            gate_up, inner, y = (part[slot:slot + 1] for part in (layer.gate_up, layer.gate, layer.y))
            compare("up", gate_up, x[t:t + 1] @ _values(layer.up_weight, e).t().contiguous())
            gate, up = gate_up.double().chunk(2, 1)
            compare("activate", inner, torch.nn.functional.silu(gate) * up)
            inner = mx.dequantize(mx.quantize(inner)).double()
            compare("down", y, inner @ _values(layer.down_weight, e).t().contiguous())
            expected[t] += share * y[0].double()
    compare("combine", layer.out[:tokens], expected)
    distances = [(error / size)**0.5 if size else float(error != 0) for error, size in squares.values()]
    return max(distances) if all(distance == distance for distance in distances) else float("nan")


# Of 2^-8 each: the one rounding of a product or a sum, the two of the activation; and as much again for fp32 sums.
TOLERANCE = 2.0**-6


def build_parser():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--tokens", type=positive_int, nargs="+", default=[1, 32, 4096])
    parser.add_argument("--hidden", type=positive_int, default=4096)
    parser.add_argument("--inner", type=positive_int, default=1024, help="an expert's inner width")
    parser.add_argument("--experts", type=positive_int, default=128)
    parser.add_argument("--top", type=positive_int, default=8)
    parser.add_argument("--dtype", choices=["bf16", "fp16"], default="bf16")
    parser.add_argument("--seed", type=int, default=0)
    parser.add_argument("--quick", action="store_true", help="small sizes: a smoke check, not a measurement")
    add_common_arguments(parser)
    return parser


def main(argv=None) -> int:
    import torch

    args = build_parser().parse_args(argv)
    if args.quick:
        args.tokens, args.hidden, args.inner, args.experts, args.top = [5], 256, 96, 8, 2
        args.warmup, args.rep, args.rounds = 5, 10, 3
    metadata = setup_device(args)
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16}[args.dtype]
    rows = []
    print(f"{'tokens':>7s} {'step':9s} {'us':>9s} {'GB/s':>9s} {'TFLOP/s':>9s} {'% of bound':>10s}")
    for tokens in args.tokens:
        layer = Layer(tokens, args.hidden, args.inner, args.experts, args.top, dtype, seed=args.seed)
        error = check(layer)
        if not error <= TOLERANCE:
            raise RuntimeError(f"a step of {tokens} tokens is {error:.3g} from the float64 products")
        for step in (*Layer.STEPS, "layer"):
            timing = measure(layer.run if step == "layer" else getattr(layer, step), args)
            parts = [work(layer, s) for s in (Layer.STEPS if step == "layer" else (step,))]
            total = {unit: sum(part[unit] for part in parts) for unit in ("bytes", "flops")}
            peak = roofline.PEAKS["tensor_fp4"][0] * 1e12
            bound = sum(max(part["bytes"] / (roofline.HBM_PEAK_GBPS * 1e9), part["flops"] / peak) for part in parts)
            seconds = timing["median_ms"] * 1e-3
            rows.append({"step": step, "dtype": args.dtype, **layer.shape, **total, "bound_us": bound * 1e6,
                         "fraction_of_bound": bound / seconds, "normwise_error": error, **timing})
            print(f"{tokens:7d} {step:9s} {seconds * 1e6:9.2f} {total['bytes'] / seconds / 1e9:9.1f} "
                  f"{total['flops'] / seconds / 1e12:9.2f} {100 * bound / seconds:10.1f}", flush=True)
        del layer
    emit_results("experts", metadata, args, rows)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
