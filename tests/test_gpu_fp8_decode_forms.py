"""GPU tests of every form in which nkv_paged_decode_fp8 launches: thread-block
clusters of one and of several CTAs a (row, kv head), and the split over the
SMs with its join. Outputs start as NaN, so a head that a form does not write
shows. The bound per element is derived in oracle/fp8_cache.py:
decode_fp8_ref."""

import pytest
import torch

from oracle.fp8_cache import decode_fp8_ref
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


# The split over the SMs and its join: more pairs than SMs, of up to 700 tokens,
# so that many are cut by a CTA's range; or few rows under a table so wide that a
# cluster would have too many tiles.
def _split_lens(Hk, wide):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    if wide:
        return [20001, 0, 129, 7000]
    return [(700, 0, 1, 130, 699, 257, 64, 512)[i % 8] for i in range(sms // Hk + 9)]


@pytest.mark.parametrize("g", range(1, 17))
@pytest.mark.parametrize("Hk,block", [(4, 64), (3, 16)])
@pytest.mark.parametrize("wide", [False, True])
def test_split_of_every_group_width(cuda_lib, g, Hk, block, wide):
    c = Cache(g, _split_lens(Hk, wide), Hk, block)
    q = _q(g, len(c.lens), Hk * g)
    _check_decode(c, q, _decode(c, q))
    assert _deverr() == 0


@pytest.mark.parametrize("Hq,Hk", [(8, 2), (4, 4), (12, 4), (9, 3), (24, 2), (16, 1)])
@pytest.mark.parametrize("spread,v_spread,sink", [(0.0, 0.0, False), (3.0, 0.5, False), (0.5, 12.0, False),
                                                  (0.5, 6.0, True)])
@pytest.mark.parametrize("wide", [False, True])
def test_split_of_row_scales_far_apart(cuda_lib, Hq, Hk, spread, v_spread, sink, wide):
    c = Cache(Hq, _split_lens(Hk, wide), Hk, 64, spread=spread, v_spread=v_spread, sink=sink)
    q = _q(6, len(c.lens), Hq)
    _check_decode(c, q, _decode(c, q))
    assert _deverr() == 0


@pytest.mark.parametrize("Hq,Hk", [(8, 2), (2, 2), (21, 3), (64, 4)])
@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** -20, 2.0 ** 12, 2.0 ** 60])
def test_split_of_queries_of_any_size(cuda_lib, Hq, Hk, factor):
    c = Cache(7, [20000, 3, 900], Hk, 64)
    shift = round(torch.tensor(factor).log2().item())
    for b, n in enumerate(c.lens):
        pos = torch.arange(n)
        c.ke[c.tables[b].long()[pos // 64], :, pos % 64] -= shift
    q = (_q(8, 3, Hq).float() * factor).to(torch.bfloat16)
    _check_decode(c, q, _decode(c, q))


@pytest.mark.parametrize("Hq,Hk,wide", [(8, 2, True), (8, 2, False), (6, 3, False), (26, 2, True), (4, 4, True)])
def test_split_with_nan_among_the_live_rows(cuda_lib, Hq, Hk, wide):
    """A NaN among a row's keys, values or queries, in any of the CTAs that share the row, is its heads' result alone."""
    g = Hq // Hk
    c = Cache(15, _split_lens(Hk, wide), Hk, 64)
    q = _q(15, len(c.lens), Hq)
    long = [b for b, n in enumerate(c.lens) if n > 600][:3]
    long = long if len(long) == 3 else [0, 3, 0]
    at = lambda b, t: (int(c.tables[b, t // 64]), t % 64)  # noqa: E731
    bad = torch.zeros(len(c.lens), Hq, 128, dtype=torch.bool, device=DEV)
    last = c.lens[long[0]] - 1
    c.k[(*at(long[0], last), 0, 3)] = 0x7F
    bad[long[0], :g] = True
    c.v[(*at(long[1], 7), Hk - 1, 5)] = 0xFF
    bad[long[1], -g:, 5] = True
    q[long[2], Hq - 1, 9] = float("nan")
    bad[long[2], Hq - 1] = True
    out = _decode(c, q)
    assert torch.equal(torch.isnan(out), bad)
    c.k[(*at(long[0], last), 0, 3)] = 0
    c.v[(*at(long[1], 7), Hk - 1, 5)] = 0
    good = ~bad.any(-1, keepdim=True).expand_as(bad)  # heads that no NaN reaches
    clean = torch.where(torch.isnan(q), torch.zeros_like(q), q)
    ref, bound = decode_fp8_ref(clean, *(t.to(DEV) for t in (c.k, c.v, c.ke, c.ve)), c.tables.to(DEV),
                                c.lens_t(), SCALE)
    assert bool(((out.double() - ref).abs() <= bound)[good].all())


@pytest.mark.parametrize("Hq,Hk", [(8, 2), (3, 3), (16, 1), (64, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_split_with_strides(cuda_lib, Hq, Hk, wide):
    """q heads apart in a wider tensor, rows of the output in one, the table a slice of a wider one."""
    c = Cache(9, _split_lens(Hk, wide), Hk, 128)
    B, mb = c.tables.shape
    q = _q(9, B, Hq)
    around = torch.full((B, Hq + 3, 256), float("nan"), dtype=torch.bfloat16, device=DEV)
    around[:, 2:2 + Hq, :128] = q
    out = torch.full((B, Hq + 2, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    table = torch.full((B, mb + 5), -1, dtype=torch.int32, device=DEV)
    table[:, :mb] = c.tables
    got = _ops().paged_decode_fp8(around[:, 2:2 + Hq, :128], *c.dev(), table[:, :mb], c.lens_t(), SCALE,
                                  out=out[:, 1:-1])
    _check_decode(c, q, got)
    assert bool(out[:, 0].isnan().all()) and bool(out[:, -1].isnan().all())
    assert _deverr() == 0


@pytest.mark.parametrize("Hq,Hk", [(8, 2), (4, 4), (9, 3), (16, 1), (64, 4)])
@pytest.mark.parametrize("wide", [False, True])
def test_split_is_the_same_every_time_and_for_any_workspace(cuda_lib, Hq, Hk, wide):
    ops = _ops()
    c = Cache(10, _split_lens(Hk, wide), Hk, 64)
    q = _q(10, len(c.lens), Hq)
    first = _decode(c, q)
    _check_decode(c, q, first)
    for fill in (0, 255, 127):  # 255: NaN in every partial result, and -1 in every record
        ws = torch.full((ops.decode_fp8_workspace_bytes(Hq, Hk),), fill, dtype=torch.uint8, device=DEV)
        assert torch.equal(_decode(c, q, workspace=ws), first)


@pytest.mark.parametrize("Hq,Hk", [(8, 2), (16, 1)])
def test_lengths_that_change_in_a_graph(cuda_lib, Hq, Hk):
    """Captured under a wide table (the split), replayed with short rows, empty ones and long ones."""
    c = Cache(11, [20000, 9000, 700, 20000], Hk, 64)
    q = _q(11, 4, Hq)
    lens, tables, dev = c.lens_t(), c.tables.to(DEV), c.dev()
    out = _nan_out(q)
    call = lambda: _ops().paged_decode_fp8(q, *dev, tables, lens, SCALE, out=out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for new in ([1, 0, 3, 2], [0, 0, 0, 0], [20000, 1, 0, 19999], [130, 9000, 700, 64]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        _check_decode(c, q, out, lens)
    assert _deverr() == 0
