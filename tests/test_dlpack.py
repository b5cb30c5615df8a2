"""Memory shared with other libraries by DLPack (dlpack_checks.py). The GPU's run in a process of their own that imports
torch before the module: imported after it, torch brings a second HIP runtime into the process, which is refused."""

import subprocess
import sys
from pathlib import Path

import pytest

pytest.importorskip("torch")

import dlpack_checks as checks  # noqa: E402

SCRIPT = Path(__file__).with_name("dlpack_checks.py")


@pytest.mark.parametrize("check", checks.SHARED, ids=lambda c: c.__name__)
def test_on_the_host(check):
    check("cpu", "cpu")


@pytest.mark.parametrize("check", checks.HOST, ids=lambda c: c.__name__)
def test_of_the_host(check):
    check()


@pytest.mark.gpu
def test_on_the_gpu():
    run = subprocess.run([sys.executable, "-u", str(SCRIPT)], capture_output=True, text=True, timeout=110)
    assert run.returncode == 0 and run.stdout.splitlines()[-1] == "all passed", run.stdout + run.stderr


@pytest.mark.gpu
def test_a_second_runtime_is_refused():
    program = ("import vectorcore_amd as vc, torch\n"
               "x = vc.Tensor([1.0, 2.0], device='hip')\n"
               "try:\n"
               "    x.__dlpack__()\n"
               "except RuntimeError as e:\n"
               "    print(e)\n")
    run = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=110,
                         cwd=SCRIPT.parents[1])
    assert run.returncode == 0 and "import torch before" in run.stdout, run.stdout + run.stderr
