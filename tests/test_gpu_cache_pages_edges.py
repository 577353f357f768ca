"""GPU tests of the page operators on states and sizes at the edge of what they take."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from tests.test_gpu_cache_pages import DEV, _caches, _dev, _deverr, _lib, _ops

pytestmark = pytest.mark.gpu

MANY_FORKS = """
import torch
from nanokv_b200 import _lib, ops
i32 = dict(dtype=torch.int32, device="cuda")
tables, lens, refs = torch.full((2560, 2), -1, **i32), torch.zeros(2560, **i32), torch.ones(40, **i32)
for n in range({first}, {last}):
    none = torch.full((n,), -1, **i32)
    assert bool((ops.fork_pages([], tables, lens, refs, none, none, 16) == -2).all())
assert _lib.read_device_error(clear=True) == 0
print("all made")
"""


@pytest.mark.parametrize("first,last", [(2400, 2413), (1, 2)])
def test_forks_around_48_kb_of_plan(cuda_lib, first, last):
    """The plan's shared memory crosses the default limit; in a process where no larger call went before."""
    pkg = Path(__file__).resolve().parents[1] / "nanokv-llm_b200"
    run = subprocess.run([sys.executable, "-c", MANY_FORKS.format(first=first, last=last)], cwd=pkg,
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "all made" in run.stdout, run.stderr[-2000:]
