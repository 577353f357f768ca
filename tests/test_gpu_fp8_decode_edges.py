"""GPU tests of what the 8-bit decode makes of rows at the edge of its number
formats and of table entries that name no page."""

import pytest
import torch

from oracle.fp8_cache import decode_fp8_ref
from tests.test_gpu_fp8_cache import DEV, SCALE, Cache, _deverr, _ops, _q

pytestmark = pytest.mark.gpu


def _within(c, q, out, tables, lens):
    k, v, ke, ve = (t.to(DEV) for t in (c.k, c.v, c.ke, c.ve))
    ref, bound = decode_fp8_ref(q, k, v, ke, ve, tables.to(DEV), lens, SCALE)
    off = (out.double() - ref).abs()
    assert torch.isfinite(out.float()).all()
    assert bool((off <= bound).all()), f"{(off - bound).max().item()} over the bound"


@pytest.mark.parametrize("rows,Hk,g", [(4, 2, 4), (50, 2, 4), (100, 1, 12), (300, 2, 1)])
def test_many_light_values_behind_a_heavy_one(cuda_lib, rows, Hk, g):
    """Every warp's first token weighs 2^26 times as much as each of the others
    (V's scales), and is zero but in dim 0: the others are the result."""
    n = 1500
    c = Cache(rows, [n] * rows, Hk, 128)
    c.k.zero_()
    c.v.fill_(0x38)  # 1.0
    c.ke.fill_(127)
    c.ve.fill_(127 - 13)
    pages = c.tables.long()
    for t in range(0, 256, 32):
        at = pages[:, t // 128]
        c.v[at, t % 128, :, 1:] = 0
        c.ve[at, :, t % 128] = 127 + 13
    q = _q(rows, rows, Hk * g)
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)
    _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE, out=out)
    _within(c, q, out, c.tables, c.lens_t())
    assert _deverr() == 0


@pytest.mark.parametrize("Hk,g,block", [(8, 4, 64), (8, 2, 16), (7, 3, 64), (3, 16, 128), (8, 8, 32)])
@pytest.mark.parametrize("rows", [400, 10])
def test_an_entry_without_a_page_counts_as_zeros(cuda_lib, Hk, g, block, rows):
    """Long rows whose tables name no page in places, behind rows of one token
    whose pages' unused exponent bytes are 255."""
    from nanokv_b200 import _lib

    lens = [1000 if i % 10 == 9 else 1 for i in range(rows)]
    c = Cache(Hk, lens, Hk, block, spare=1)
    zero = next(p for p in range(c.blocks) if not bool((c.tables == p).any()))
    c.k[zero] = c.v[zero] = 0
    c.ke[zero] = c.ve[zero] = 127
    bad, tables = c.tables.clone(), c.tables.clone()
    for b in range(9, rows, 10):
        for j, entry in ((200 // block, -1), (500 // block, c.blocks), (999 // block, -7)):
            bad[b, j], tables[b, j] = entry, zero
    q = _q(Hk, rows, Hk * g)
    out = torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)
    _ops().paged_decode_fp8(q, *c.dev(), bad.to(DEV), c.lens_t(), SCALE, out=out)
    assert _deverr() == _lib.DEVERR_DECODE_BLOCK
    _within(c, q, out, tables, c.lens_t())
