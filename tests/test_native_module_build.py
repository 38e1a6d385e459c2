"""The host module belongs to the torch that it was built against: under another one it is not used, and Python packs the slots."""

from __future__ import annotations

import subprocess
import sys

import pytest

from tests.conftest import REPO_ROOT

PROGRAM = """
import torch
{change}
from kernelcode_generate_amd import native
native.load_library()
try:
    from kernelcode_generate_amd import _kg_call
    print("loaded", native._FAST_CALL is _kg_call.call)
except ImportError as error:
    print("refused", native._FAST_CALL, error)
try:
    native.quantize_rows(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4), torch.zeros(4, 16))
except native.NativeLibraryError as error:
    print(error)
"""


def output_of(change):
    run = subprocess.run([sys.executable, "-c", PROGRAM.format(change=change)], capture_output=True, text=True, cwd=REPO_ROOT, timeout=120)
    assert run.returncode == 0, run.stderr
    return run.stdout.splitlines()


def test_the_torch_that_is_installed():
    first, call = output_of("")
    assert first == "loaded True" and "not a device pointer" in call


@pytest.mark.parametrize("change", ["torch.__version__ = '2.0.0+other'", "torch.version.git_version = '0' * 40", "del torch.version.git_version"])
def test_another_torch(change):
    first, call = output_of(change)
    assert first.startswith("refused None built against torch ") and "not a device pointer" in call
