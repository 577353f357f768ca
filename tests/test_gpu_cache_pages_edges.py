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


def _fork(tables, lens, refs, src, dst, kind="views"):
    """fork_pages on 8 pages of 16 tokens: (out_pages, tables, lens, refs, moved pages, error word)."""
    caches, pd = _caches(7, kind, 8, 16, 1)
    before = [c.clone() for c in caches]
    t, n, r = _dev(tables), _dev(lens), _dev(refs)
    out = _ops().fork_pages(caches, t, n, r, _dev(src), _dev(dst), 16, page_dim=pd).tolist()
    moved = {p for a, b in zip(caches, before) for p in range(8)
             if not torch.equal(a[p].view(torch.uint8), b[p].view(torch.uint8))}
    return out, t.tolist(), n.tolist(), r.tolist(), moved, _deverr()


@pytest.mark.parametrize("kind", ["views", "fp8"])
def test_fork_of_a_partial_page_that_nobody_holds(cuda_lib, kind):
    """Page 2 is row 0's last, with a count of 0: it is the lowest free page as
    well. No fork of row 0 is made; row 1's, behind it, is."""
    tables = [[4, 2, -1], [5, 1, -1], [7, -1, -1], [-1, -1, -1]]
    refs = [1, 1, 0, 0, 1, 1, 1, 1]
    out, t, n, r, moved, err = _fork(tables, [20, 20, 3, 0], refs, [0, 1], [2, 3], kind)
    assert out == [-2, 2] and err == _lib().DEVERR_PAGES
    assert t == [[4, 2, -1], [5, 1, -1], [-1, -1, -1], [5, 2, -1]]
    assert n == [20, 20, 0, 20] and r == [1, 1, 1, 0, 1, 2, 1, 0] and moved == {2}


def test_fork_of_a_partial_page_that_a_target_gives_up(cuda_lib):
    """Row 0's last page is counted once, for row 1's table, which gives it up in the same call."""
    tables = [[4, 2, -1], [2, -1, -1]]
    out, t, n, r, moved, err = _fork(tables, [20, 3], [1, 1, 1, 1, 1, 1, 1, 1], [0], [1])
    assert out == [-2] and err == _lib().DEVERR_PAGES
    assert t == [[4, 2, -1], [-1] * 3] and n == [20, 0] and r == [1, 1, 0, 1, 1, 1, 1, 1] and not moved


@pytest.mark.parametrize("entry", [-1, 8, -5, 1 << 30])
@pytest.mark.parametrize("length,at", [(32, 0), (32, 1), (40, 0), (40, 1), (40, 2)])
def test_fork_of_a_row_that_lacks_a_page(cuda_lib, entry, length, at):
    """A full page that is none of the cache is missing in the branch too; of a partial one no fork is made."""
    row = [4, 2, 6]
    row[at] = entry
    tables = [row, [7, -1, -1], [-1] * 3, [3, 5, -1]]
    out, t, n, r, moved, err = _fork(tables, [length, 3, 0, 24], [0, 0, 1, 1, 1, 1, 1, 1], [0, 3], [1, 2])
    assert err == _lib().DEVERR_PAGES and t[0] == row and t[3] == tables[3]
    refs = [0, 0, 1, 2, 1, 1, 1, 0]
    if at == length // 16:
        assert out == [-2, 0] and t[1] == [-1] * 3 and t[2] == [3, 0, -1] and n == [length, 0, 24, 24]
        refs[0], taken = 1, {0}
    else:
        new = [0] if length % 16 else []
        branch = [-1 if p == entry else p for p in row[:length // 16]] + new
        last = len(new)
        assert out == [0 if new else -1, last] and t[1] == branch + [-1] * (3 - len(branch))
        assert t[2] == [3, last, -1] and n == [length, length, 24, 24]
        for p in (4, 2):
            refs[p] += p in branch
        refs[0] = 1
        refs[1] = last
        taken = {0, last}
    assert r == refs and moved == taken


@pytest.mark.parametrize("given_up", [False, True])
def test_fork_of_a_full_page_that_nobody_holds(cuda_lib, given_up):
    """Page 0 is row 0's first, full page, with no count, or with row 2's alone,
    which row 2 gives up: it is not handed out, but counted for row 0 again."""
    tables = [[0, 4, -1], [5, 1, -1], [0 if given_up else -1, -1, -1], [-1] * 3]
    refs = [1 if given_up else 0, 1, 0, 0, 1, 1, 1, 1]
    out, t, n, r, moved, err = _fork(tables, [32, 20, 3 if given_up else 0, 0], refs, [0, 1], [2, 3])
    assert out == [-1, 2] and err == _lib().DEVERR_PAGES
    assert t == [[0, 4, -1], [5, 1, -1], [0, 4, -1], [5, 2, -1]] and n == [32, 20, 32, 20]
    assert r == [2, 1, 1, 0, 2, 2, 1, 1] and moved == {2}


@pytest.mark.parametrize("count", [0, -3])
def test_fork_of_an_unheld_page_where_none_is_handed_out(cuda_lib, count):
    tables = [[0, 4, -1], [-1] * 3]
    out, t, n, r, moved, err = _fork(tables, [32, 0], [count, 1, 1, 1, 1, 1, 1, 1], [0], [1])
    assert out == [-1] and err == _lib().DEVERR_PAGES
    assert t == [[0, 4, -1]] * 2 and n == [32, 32] and r == [2, 1, 1, 1, 2, 1, 1, 1] and not moved
