"""What a step of the mixture-of-experts layer on FP8 is priced at."""

from types import SimpleNamespace

import pytest
import torch

from triton_chip_benchmarks_amd import experts


@pytest.mark.parametrize("tokens", [3, 30])
def test_work_counts_used_experts_once_and_every_choice(tokens):
    layer = object.__new__(experts.Fp8Layer)
    layer.shape = {"tokens": tokens, "hidden": 200, "inner": 140, "experts": 4, "top": 2}
    layer.x = torch.empty(tokens, 200, dtype=torch.bfloat16)
    layer.plan = SimpleNamespace(offsets=torch.tensor([0, 4, 4, 2 * tokens, 2 * tokens], dtype=torch.int32))
    # Two of four experts have rows; 200 and 140 columns are two blocks, 280 rows three, 200 two. Few rows lie between the
    # steps in 16 bits, others as an operand.
    rows = 2 * tokens
    between = rows * 140 * 2 if rows <= experts.FEW_ROWS else rows * 142
    assert experts.work(layer, "norm") == {"bytes": (4 * tokens + 1) * 200 * 2, "flops": 5 * tokens * 200}
    assert experts.work(layer, "gated") == {"bytes": tokens * 200 * 2 + 2 * (280 * 200 + 6) + between,
                                            "flops": 4 * rows * 140 * 200}
    assert experts.work(layer, "down") == {"bytes": between + 2 * (200 * 140 + 4) + rows * 200 * 2,
                                           "flops": 2 * rows * 140 * 200}
    assert all(experts.work(layer, step)["bytes"] > 0 for step in layer.STEPS)


def test_weights_are_of_a_known_format():
    assert experts.build_parser().parse_args([]).weights == "mxfp4"
    with pytest.raises(SystemExit):
        experts.build_parser().parse_args(["--weights", "fp6"])
