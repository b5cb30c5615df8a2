"""Recorded work and memory that another library writes (shared_memory_checks.py). The GPU's run in a process of their own
that imports torch before the module."""

import subprocess
import sys
from pathlib import Path

import pytest

pytest.importorskip("torch")

import shared_memory_checks as checks  # noqa: E402

SCRIPT = Path(__file__).with_name("shared_memory_checks.py")


@pytest.mark.parametrize("check", checks.RECORDED + checks.KEPT, ids=lambda c: c.__name__)
def test_on_the_host(check):
    check("cpu", "cpu")


@pytest.mark.gpu
def test_on_the_gpu():
    run = subprocess.run([sys.executable, "-u", str(SCRIPT)], capture_output=True, text=True, timeout=110)
    assert run.returncode == 0 and run.stdout.splitlines()[-1] == "all passed", run.stdout + run.stderr
