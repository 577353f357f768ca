"""GPU tests of every form in which nkv_paged_decode_fp8 launches: thread-block
clusters of one and of several CTAs a (row, kv head), and the split over the
SMs with its join. Outputs start as NaN, so a head that a form does not write
shows. The bound per element is derived in oracle/fp8_cache.py:
decode_fp8_ref."""

import pytest
import torch

from tests.test_gpu_fp8_cache import DEV, SCALE, Cache, _check_decode, _deverr, _ops, _q

pytestmark = pytest.mark.gpu


def _nan_out(q):
    return torch.full(q.shape, float("nan"), dtype=torch.bfloat16, device=DEV)


def _decode(c, q, **kw):
    out = _nan_out(q)
    _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE, out=out, **kw)
    return out


# A table of one 128-token tile: one CTA a (row, kv head), whatever the group.
@pytest.mark.parametrize("g", range(1, 17))
@pytest.mark.parametrize("block,lens", [(128, [100]), (16, [128, 0, 1, 77]), (64, [65] * 40)])
def test_one_tile_tables(cuda_lib, g, block, lens):
    c = Cache(g + block, lens, 2, block)
    assert c.tables.size(1) * block <= 128
    q = _q(g, len(lens), 2 * g)
    _check_decode(c, q, _decode(c, q))
    assert _deverr() == 0


# More than half as many (row, kv head) pairs as SMs, a few tiles each: one CTA a pair.
@pytest.mark.parametrize("g", [1, 7, 8, 9, 12, 13, 16])
@pytest.mark.parametrize("share,Hk", [(0.51, 1), (0.86, 4), (1.0, 1), (1.0, 2)])
def test_one_cta_a_pair(cuda_lib, g, share, Hk):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rows = int(sms * share) // Hk
    lens = [(900, 0, 1, 130, 1200, 257, 64)[i % 7] for i in range(rows)]
    c = Cache(g + rows, lens, Hk, 64)
    q = _q(g, rows, Hk * g)
    _check_decode(c, q, _decode(c, q))
    assert _deverr() == 0
