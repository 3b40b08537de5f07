"""CPU tests of the mixture-of-experts command: its arguments and what each step is priced at."""

from types import SimpleNamespace
from pathlib import Path
import subprocess
import sys

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_runs_as_a_plain_script():
    script = ROOT / "triton_chip_benchmarks_amd" / "experts.py"
    completed = subprocess.run([sys.executable, str(script), "--help"], capture_output=True, text=True, timeout=120,
                               check=False)
    assert completed.returncode == 0, completed.stderr[-2000:]
    assert "--tokens" in completed.stdout


@pytest.mark.parametrize("argument", ["--tokens", "--hidden", "--inner", "--experts", "--top"])
def test_sizes_are_positive(argument):
    from triton_chip_benchmarks_amd import experts

    with pytest.raises(SystemExit):
        experts.build_parser().parse_args([argument, "0"])


def test_work_counts_used_experts_once_and_every_choice():
    import torch

    from triton_chip_benchmarks_amd import experts

    layer = SimpleNamespace(shape={"tokens": 3, "hidden": 64, "inner": 40, "experts": 4, "top": 2},
                            x=torch.empty(3, 64, dtype=torch.bfloat16),
                            plan=SimpleNamespace(offsets=torch.tensor([0, 4, 4, 6, 6], dtype=torch.int32)))
    # Two of four experts have rows; 64 columns are two groups of 17 bytes, 40 are two as well.
    assert experts.work(layer, "up") == {"bytes": (3 * 64 + 6 * 80) * 2 + 2 * 80 * 34, "flops": 2 * 6 * 80 * 64}
    assert experts.work(layer, "down") == {"bytes": (6 * 40 + 6 * 64) * 2 + 2 * 64 * 34, "flops": 2 * 6 * 40 * 64}
    assert experts.work(layer, "combine")["bytes"] == (6 + 3) * 64 * 2 + 48
    assert {step for step in experts.Layer.STEPS if experts.work(layer, step)["bytes"] <= 0} == set()
