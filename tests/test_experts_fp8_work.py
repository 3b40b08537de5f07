"""What a step of the mixture-of-experts layer on FP8 is priced at."""

from types import SimpleNamespace

import pytest
import torch

from triton_chip_benchmarks_amd import experts


def test_work_counts_used_experts_once_and_every_choice():
    layer = object.__new__(experts.Fp8Layer)
    layer.shape = {"tokens": 3, "hidden": 200, "inner": 140, "experts": 4, "top": 2}
    layer.x = torch.empty(3, 200, dtype=torch.bfloat16)
    layer.plan = SimpleNamespace(offsets=torch.tensor([0, 4, 4, 6, 6], dtype=torch.int32))
    # Two of four experts have rows; 200 and 140 columns are two blocks, 280 rows three, 200 two.
    assert experts.work(layer, "norm") == {"bytes": 13 * 200 * 2, "flops": 5 * 3 * 200}
    assert experts.work(layer, "gated") == {"bytes": 3 * 200 * 2 + 2 * (280 * 200 + 6) + 6 * 142,
                                            "flops": 4 * 6 * 140 * 200}
    assert experts.work(layer, "down") == {"bytes": 6 * 142 + 2 * (200 * 140 + 4) + 6 * 200 * 2,
                                           "flops": 2 * 6 * 140 * 200}
    assert all(experts.work(layer, step)["bytes"] > 0 for step in layer.STEPS)


def test_weights_are_of_a_known_format():
    assert experts.build_parser().parse_args([]).weights == "mxfp4"
    with pytest.raises(SystemExit):
        experts.build_parser().parse_args(["--weights", "fp6"])
