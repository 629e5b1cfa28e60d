"""A refused argument of the extension is a Python exception, not the end of the process (which it was
when the extension carried a static C++ runtime of its own). Run in a child process for that reason."""

import subprocess
import sys

import pytest
import torch

_CHILD = """
import torch
from ohara_b200.ops._ext import ext
for call in ({calls}):
    try:
        call()
    except (RuntimeError, ValueError, TypeError) as error:
        print("refused:", str(error).splitlines()[0])
    else:
        raise SystemExit("accepted")
"""


def _run(calls: str) -> subprocess.CompletedProcess:
    return subprocess.run([sys.executable, "-c", _CHILD.format(calls=calls)], capture_output=True,
                          text=True, timeout=300)


def test_host_checks_raise():
    proc = _run("lambda: ext().token_logprobs(torch.zeros(2, 3), None, 1.0, True, 0, -100), "
                "lambda: ext().rmsnorm_fwd(torch.zeros(2, 8), None, torch.zeros(8), 1e-5)")
    assert proc.returncode == 0 and proc.stdout.count("refused:") == 2, proc.stdout + proc.stderr


@pytest.mark.skipif(torch.cuda.is_available(), reason="the call succeeds with a device")
def test_errors_of_the_kernel_launchers_raise():
    proc = _run("lambda: ext().status(False), ")       # a std::runtime_error of the torch-free code
    assert proc.returncode == 0 and "refused: ohara_b200:" in proc.stdout, proc.stdout + proc.stderr


@pytest.mark.gpu
def test_errors_of_the_kernel_launchers_raise_on_a_device():
    proc = _run("lambda: ext().cross_entropy_rows(torch.zeros(2, 200_000, device='cuda').bfloat16(), "
                "torch.zeros(2, dtype=torch.long, device='cuda'), None, -1, False, False), ")
    assert proc.returncode == 0 and "too large" in proc.stdout, proc.stdout + proc.stderr
