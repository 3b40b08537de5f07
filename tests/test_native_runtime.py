"""CPU check: a process has one HIP runtime, whichever of torch and the library its program asks for first."""

import ast
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
FIRST = {"library": "from triton_chip_benchmarks_amd import _native\n_native.load()\nimport torch",
         "torch": "import torch\nfrom triton_chip_benchmarks_amd import _native\n_native.load()"}


@pytest.mark.parametrize("first", sorted(FIRST))
def test_a_process_has_one_hip_runtime(first):
    program = FIRST[first] + "\nprint({line.split()[-1] for line in open('/proc/self/maps') if 'libamdhip64' in line})"
    shown = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert shown.returncode == 0, shown.stderr
    assert len(ast.literal_eval(shown.stdout)) == 1, shown.stdout
