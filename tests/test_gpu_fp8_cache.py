"""GPU tests of the 8-bit KV cache -- nkv_store_kvcache_fp8,
nkv_load_kvcache_fp8, nkv_paged_decode_fp8 -- against the 64-bit oracle.

Stored codes, exponent bytes and the rows read back are exact. The decode's
bound per element is derived in oracle/fp8_cache.py: decode_fp8_ref.
"""

import numpy as np
import pytest
import torch

from oracle.fp8_cache import (decode_fp8_ref, dequantise_ref, quantise_ref, sequence_ref,
                              store_fp8_ref)

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _ops():
    from nanokv_b200 import ops
    return ops


def _deverr():
    from nanokv_b200 import _lib
    return _lib.read_device_error(clear=True)


class Cache:
    """An 8-bit cache whose unused rows hold NaN codes and byte 255, and a
    shuffled block table over it."""

    def __init__(self, seed, lens, Hk, block, spare=2, spread=0.5, v_spread=0.5, sink=False):
        rng = np.random.default_rng(seed)
        self.lens, self.Hk, self.block = lens, Hk, block
        need = sum(-(-n // block) for n in lens)
        self.blocks = need + spare
        perm = rng.permutation(self.blocks)
        width = max(1, max(-(-n // block) for n in lens))
        table, at = [], 0
        for n in lens:
            m = -(-n // block)
            table.append(list(perm[at:at + m]) + [-1] * (width - m))
            at += m
        self.tables = torch.tensor(np.array(table), dtype=torch.int32)
        self.k, self.v = (torch.full((self.blocks, block, Hk, 128), 0x7F, dtype=torch.uint8) for _ in "kv")
        self.ke, self.ve = (torch.full((self.blocks, Hk, block), 255, dtype=torch.uint8) for _ in "kv")
        for codes, exps, s in ((self.k, self.ke, spread), (self.v, self.ve, v_spread)):
            for b, n in enumerate(lens):
                if n == 0:
                    continue
                c = rng.integers(0, 255, (n, Hk, 128), dtype=np.uint8)
                c[(c & 127) == 127] = 0  # no NaN among the live rows
                # scales near 2^-8: rows of norm about 1
                e = np.clip(np.rint(119 + s * rng.standard_normal((n, Hk))), 10, 246).astype(np.uint8)
                if sink:
                    e[0] = max(10, int(119 - 4 * s))  # a first token with a tiny value
                pos = np.arange(n)
                page = self.tables[b].numpy()[pos // block]
                codes[page, pos % block] = torch.from_numpy(c)
                exps[page, :, pos % block] = torch.from_numpy(e)

    def dev(self):
        f = torch.float8_e4m3fn
        return (self.k.to(DEV).view(f), self.v.to(DEV).view(f), self.ke.to(DEV), self.ve.to(DEV))

    def lens_t(self):
        return torch.tensor(self.lens, dtype=torch.int32, device=DEV)


def _q(seed, B, Hq, spread=0.5):
    g = torch.Generator().manual_seed(seed)
    # e4m3 codes are spread over [2^-9, 448]: queries that give scores of a few units
    x = torch.randn(B, Hq, 128, generator=g) * torch.exp(spread * torch.randn(B, Hq, 1, generator=g))
    return (x * 0.3).to(torch.bfloat16).to(DEV)


def _check_decode(c, q, out, lens=None):
    k, v, ke, ve = (t.to(DEV) for t in (c.k, c.v, c.ke, c.ve))
    lens = c.lens_t() if lens is None else lens
    ref, bound = decode_fp8_ref(q, k, v, ke, ve, c.tables.to(DEV), lens, SCALE)
    off = (out.double() - ref).abs()
    assert torch.isfinite(out.float()).all()
    worst = (off - bound).max().item()
    assert worst <= 0, f"{worst} over the bound, {(off > bound).float().mean().item():.4f} of the elements"


# ---------------------------------------------------------------- rows
ROWS = [(1, 1, 128), (7, 8, 16), (33, 2, 32), (130, 4, 64), (257, 8, 256), (65, 5, 384)]


def _rows(seed, T, Hk):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, Hk, 128), dtype=np.float32)
    x *= np.exp2(rng.integers(-60, 60, (T, Hk, 1))).astype(np.float32)
    x.reshape(-1)[rng.integers(0, x.size, 1 + x.size // 50)] = 0.0
    x = torch.from_numpy(x).to(torch.bfloat16)
    return x


@pytest.mark.parametrize("T,Hk,block", ROWS)
def test_store_and_load_are_exact(cuda_lib, T, Hk, block):
    ops = _ops()
    rng = np.random.default_rng(T)
    key, value = _rows(T, T, Hk), _rows(T + 1, T, Hk)
    # rows that are hard to scale: zeros, one huge, one tiny, borders of the scale
    edge = [0.0, 3.3895e38, 1e-40, 448.0, 449.0, 1.75, 1.7578125, 2.0 ** -120, 2.0 ** 127]
    for i, e in enumerate(edge[:T]):
        key[i, 0] = 0.0
        key[i, 0, i % 128] = e
    blocks = -(-T // block) + 1
    slots = torch.from_numpy(rng.permutation(blocks * block)[:T].astype(np.int32))
    if T > 3:
        slots[T // 2] = -1
    k0 = torch.full((blocks, block, Hk, 128), 3, dtype=torch.uint8)
    e0 = torch.full((blocks, Hk, block), 7, dtype=torch.uint8)
    ref = [k0.clone(), k0.clone(), e0.clone(), e0.clone()]
    store_fp8_ref(key, value, *ref, slots)
    f = torch.float8_e4m3fn
    got = [k0.to(DEV).view(f), k0.to(DEV).view(f), e0.to(DEV), e0.to(DEV)]
    # as slices of a wider projection output
    wide = torch.cat([torch.zeros(T, 128 * Hk), key.float().view(T, -1), value.float().view(T, -1)], 1)
    wide = wide.to(torch.bfloat16).to(DEV)
    ops.store_kvcache_fp8(wide[:, 128 * Hk:256 * Hk].view(T, Hk, 128),
                          wide[:, 256 * Hk:].view(T, Hk, 128), *got, slots.to(DEV))
    for a, b in zip(got, ref):
        assert torch.equal(a.view(torch.uint8).cpu(), b)
    # every slot read back as one sequence over all pages, in page order
    table = torch.arange(blocks, dtype=torch.int32, device=DEV).view(1, -1)
    cu = torch.tensor([0, blocks * block], dtype=torch.int32, device=DEV)
    k, v = ops.load_kvcache_fp8(*got, table, cu, blocks * block)
    for out, codes, exps in ((k, ref[0], ref[2]), (v, ref[1], ref[3])):
        want = dequantise_ref(codes, exps.transpose(1, 2)).reshape(-1, Hk, 128)
        live = (exps.transpose(1, 2).reshape(-1, Hk) != 7)
        assert torch.equal(out.cpu().double()[live], want[live])
    assert _deverr() == 0


def test_store_of_infinities_and_nan(cuda_lib):
    ops = _ops()
    x = torch.randn(4, 2, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    x[0, 0, 5] = float("inf")
    x[1, 1, 6] = float("-inf")
    x[2, 0, 7] = float("nan")
    x[3, 1] = float("nan")
    f = torch.float8_e4m3fn
    k, v = (torch.zeros(1, 16, 2, 128, dtype=torch.uint8, device=DEV) for _ in "kv")
    ke, ve = (torch.zeros(1, 2, 16, dtype=torch.uint8, device=DEV) for _ in "kv")
    slots = torch.arange(4, dtype=torch.int32, device=DEV)
    ops.store_kvcache_fp8(x.to(DEV), x.to(DEV), k.view(f), v.view(f), ke, ve, slots)
    codes, exps = quantise_ref(x)
    for c, e in ((k, ke), (v, ve)):
        assert torch.equal(c[0, :4].cpu(), codes) and torch.equal(e[0, :, :4].T.cpu(), exps)


def test_load_ragged_sequences_and_rows_behind(cuda_lib):
    ops = _ops()
    c = Cache(11, [0, 1, 300, 16, 0, 129, 15], 3, 16)
    cu = np.cumsum([0] + c.lens)
    total = int(cu[-1]) + 5  # five rows behind the last sequence
    outs = [torch.full((total, 2 * c.Hk, 128), 9.0, dtype=torch.bfloat16, device=DEV) for _ in "kv"]
    k, v = ops.load_kvcache_fp8(*c.dev(), c.tables.to(DEV),
                                torch.tensor(cu, dtype=torch.int32, device=DEV), total,
                                k_out=outs[0][:, c.Hk:], v_out=outs[1][:, :c.Hk])
    for b, n in enumerate(c.lens):
        for out, codes, exps in ((k, c.k, c.ke), (v, c.v, c.ve)):
            assert torch.equal(out[cu[b]:cu[b + 1]].cpu().double(), sequence_ref(codes, exps, c.tables[b], n))
    assert bool((outs[0][:, :c.Hk] == 9).all()) and bool((outs[1][:, c.Hk:] == 9).all())
    assert bool((k[int(cu[-1]):] == 9).all()) and bool((v[int(cu[-1]):] == 9).all())
    assert _deverr() == 0


def test_bad_slots_and_pages_are_flagged(cuda_lib):
    from nanokv_b200 import _lib

    ops = _ops()
    c = Cache(12, [40, 20], 2, 16, spare=0)
    dev = c.dev()
    before = [t.clone().view(torch.uint8) for t in dev]
    x = torch.ones(3, 2, 128, dtype=torch.bfloat16, device=DEV)
    ops.store_kvcache_fp8(x, x, *dev, torch.tensor([c.blocks * 16, -2, -1], dtype=torch.int32, device=DEV))
    assert _deverr() == _lib.DEVERR_STORE_SLOT
    for a, b in zip(dev, before):
        assert torch.equal(a.view(torch.uint8), b)
    tables = c.tables.clone()
    tables[0, 1] = c.blocks
    cu = torch.tensor([0, 40, 60], dtype=torch.int32, device=DEV)
    k, v = ops.load_kvcache_fp8(*dev, tables.to(DEV), cu, 60)
    assert _deverr() == _lib.DEVERR_DECODE_BLOCK
    assert bool((k[16:32] == 0).all()) and bool((v[16:32] == 0).all())
    # a sequence longer than its table
    cu = torch.tensor([0, 16 * c.tables.size(1) + 3], dtype=torch.int32, device=DEV)
    ops.load_kvcache_fp8(*dev, c.tables.to(DEV), cu, 16 * c.tables.size(1) + 3)
    assert _deverr() == _lib.DEVERR_PREFILL_RANGE
    lens = torch.tensor([16 * c.tables.size(1) + 100, 20], dtype=torch.int32, device=DEV)
    full = torch.randint(0, c.blocks, c.tables.shape, dtype=torch.int32, device=DEV)
    ops.paged_decode_fp8(_q(1, 2, 4), *dev, full, lens, SCALE)
    assert _deverr() == _lib.DEVERR_DECODE_BLOCK
    lens = torch.tensor([40, 20], dtype=torch.int32, device=DEV)
    out = ops.paged_decode_fp8(_q(1, 2, 4), *dev, tables.to(DEV), lens, SCALE)
    assert _deverr() == _lib.DEVERR_DECODE_BLOCK
    ref, bound = decode_fp8_ref(_q(1, 2, 4)[1:], c.k.to(DEV), c.v.to(DEV), c.ke.to(DEV), c.ve.to(DEV),
                                c.tables[1:].to(DEV), lens[1:], SCALE)
    assert bool(((out[1:].double() - ref).abs() <= bound).all())  # the other row is not touched by it


# ---------------------------------------------------------------- decode
DECODE = [
    # lens, Hq, Hk, block
    ([1], 1, 1, 128),
    ([0], 4, 2, 128),
    ([700], 16, 8, 256),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33], 4, 2, 16),
    ([127, 128, 129, 255, 256, 257, 0, 511], 32, 8, 256),
    ([64, 65, 1000, 63, 0, 0], 10, 2, 64),
    ([1, 300, 90], 16, 1, 32),
    ([3000, 7, 0, 1500], 64, 4, 512),
    ([33000], 4, 1, 256),
    ([20001, 0, 1, 5000, 129], 5, 1, 128),
    ([0, 0, 0, 0], 8, 8, 256),
    ([200] * 37, 24, 8, 384),
    (list(range(0, 300)), 2, 1, 128),
    ([128] * 400, 3, 3, 128),
    ([(37 * i) % 41 for i in range(4099)], 4, 2, 16),
    ([700, 0, 90000], 36, 4, 256),
]


@pytest.mark.parametrize("lens,Hq,Hk,block", DECODE, ids=[str(i) for i in range(len(DECODE))])
def test_decode_matches_64_bits(cuda_lib, lens, Hq, Hk, block):
    c = Cache(len(lens) + Hq, lens, Hk, block)
    q = _q(Hq, len(lens), Hq)
    out = _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE)
    _check_decode(c, q, out)
    assert _deverr() == 0


@pytest.mark.parametrize("g", range(1, 17))
def test_decode_every_group_width(cuda_lib, g):
    c = Cache(g, [333, 1, 128, 0, 2100], 2, 128)
    q = _q(g, 5, 2 * g)
    out = _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE)
    _check_decode(c, q, out)


# More (row, kv head) pairs than SMs, some long enough that the split cuts
# them: the join takes a pair's 5 to 16 q heads in one CTA.
@pytest.mark.parametrize("Hq,Hk,rows", [(64, 8, 24), (56, 8, 24), (40, 8, 24), (24, 8, 24), (32, 2, 80),
                                        (27, 3, 60), (24, 4, 50), (5, 1, 151)])
@pytest.mark.parametrize("long", [900, 5000])
def test_decode_many_split_pairs(cuda_lib, Hq, Hk, rows, long):
    lens = [(0, 1, 130, long, long - 77, 257, 64)[i % 7] for i in range(rows)]
    c = Cache(Hq + rows, lens, Hk, 64)
    q = _q(Hq, rows, Hq)
    out = _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE)
    _check_decode(c, q, out)
    assert _deverr() == 0


@pytest.mark.parametrize("spread,v_spread,sink", [(0.0, 0.0, False), (3.0, 0.5, False), (0.5, 12.0, False),
                                                  (0.5, 6.0, True)])
def test_decode_row_scales_far_apart(cuda_lib, spread, v_spread, sink):
    c = Cache(5, [900, 130, 4000], 2, 128, spread=spread, v_spread=v_spread, sink=sink)
    q = _q(6, 3, 8)
    out = _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE)
    _check_decode(c, q, out)


@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** -20, 2.0 ** 12, 2.0 ** 60])
def test_decode_queries_of_any_size(cuda_lib, factor):
    """Queries far outside 16-bit floats' middle range, the cache scaled the other way."""
    c = Cache(7, [500, 3], 2, 64)
    shift = int(np.log2(factor))
    for b, n in enumerate(c.lens):
        pos = torch.arange(n)
        page = c.tables[b].long()[pos // 64]
        c.ke[page, :, pos % 64] -= shift
    q = (_q(8, 2, 4).float() * factor).to(torch.bfloat16)
    out = _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE)
    _check_decode(c, q, out)


def test_decode_nan_and_infinity_among_the_live_rows(cuda_lib):
    """A NaN among a row's keys, values or queries is its heads' result, nobody else's."""
    c = Cache(15, [300, 300, 300, 40], 2, 64)
    q = _q(15, 4, 4)
    at = lambda b, t: (int(c.tables[b, t // 64]), t % 64)  # noqa: E731
    c.k[(*at(0, 250), 0, 3)] = 0x7F
    c.v[(*at(1, 7), 1, 5)] = 0xFF
    q[2, 3, 9] = float("nan")
    out = _ops().paged_decode_fp8(q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE)
    bad = torch.zeros(4, 4, 128, dtype=torch.bool, device=DEV)
    bad[0, :2] = True
    bad[1, 2:, 5] = True
    bad[2, 3] = True
    assert torch.equal(torch.isnan(out), bad)
    c.k[(*at(0, 250), 0, 3)] = 0
    c.v[(*at(1, 7), 1, 5)] = 0
    clean = torch.where(torch.isnan(q), torch.zeros_like(q), q)
    ref, bound = decode_fp8_ref(clean, *(t.to(DEV) for t in (c.k, c.v, c.ke, c.ve)), c.tables.to(DEV),
                                c.lens_t(), SCALE)
    good = ~bad.any(-1)  # heads that no NaN reaches
    assert bool(((out.double() - ref).abs() <= bound)[good].all())


def test_decode_without_tables(cuda_lib):
    """No page at all: every row is empty, or flagged and empty."""
    from nanokv_b200 import _lib

    c = Cache(16, [0, 0, 0], 2, 64)
    q = _q(16, 3, 4)
    tables = torch.empty(3, 0, dtype=torch.int32, device=DEV)
    out = torch.full((3, 4, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    _ops().paged_decode_fp8(q, *c.dev(), tables, c.lens_t(), SCALE, out=out)
    assert bool((out == 0).all()) and _deverr() == 0
    out.fill_(3.0)
    _ops().paged_decode_fp8(q, *c.dev(), tables, c.lens_t() + 5, SCALE, out=out)
    assert bool((out == 0).all()) and _deverr() == _lib.DEVERR_DECODE_BLOCK


def test_decode_strided_rows_and_outputs(cuda_lib):
    c = Cache(9, [300, 0, 77], 2, 128)
    q = _q(9, 3, 8)
    wide = torch.full((3, 20, 256), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 4:20:2, :128] = q
    qs = wide[:, 4:20:2, :128]  # head stride 512
    out = torch.full((3, 12, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    wide_table = torch.full((3, 9), -1, dtype=torch.int32, device=DEV)
    wide_table[:, :c.tables.size(1)] = c.tables
    got = _ops().paged_decode_fp8(qs, *c.dev(), wide_table[:, :c.tables.size(1)], c.lens_t(), SCALE,
                                  out=out[:, 2:10])
    _check_decode(c, q, got)
    assert bool((out[:, :2] == 5).all()) and bool((out[:, 10:] == 5).all())


def test_decode_is_the_same_every_time_and_for_any_workspace(cuda_lib):
    ops = _ops()
    c = Cache(10, [9000, 3, 700, 4097], 4, 256)
    q = _q(10, 4, 16)
    args = (q, *c.dev(), c.tables.to(DEV), c.lens_t(), SCALE)
    first = ops.paged_decode_fp8(*args)
    for fill in (0, 255, 127):
        ws = torch.full((ops.decode_fp8_workspace_bytes(16, 4),), fill, dtype=torch.uint8, device=DEV)
        assert torch.equal(ops.paged_decode_fp8(*args, workspace=ws), first)
    _check_decode(c, q, first)


def test_decode_of_a_cache_past_32_bits(cuda_lib):
    """Values past 4 GiB (the pages at the end of a 4.4 GiB cache): store, decode, read-back."""
    ops = _ops()
    Hk, block, blocks = 8, 256, 16900
    small = Cache(13, [600, 1, 257], Hk, block, spare=0)
    q = _q(13, 3, 16)
    first = blocks - small.blocks
    big = [torch.empty(blocks, block, Hk, 128, dtype=torch.uint8, device=DEV) for _ in "kv"]
    exps = [torch.empty(blocks, Hk, block, dtype=torch.uint8, device=DEV) for _ in "kv"]
    for b, s in zip(big + exps, (small.k, small.v, small.ke, small.ve)):
        b[first:] = s.to(DEV)
    assert big[0].numel() > 1 << 32
    f = torch.float8_e4m3fn
    tables = torch.where(small.tables >= 0, small.tables + first, small.tables).to(DEV)
    args = (big[0].view(f), big[1].view(f), *exps)
    out = ops.paged_decode_fp8(q, *args, tables, small.lens_t(), SCALE)
    _check_decode(small, q, out)
    x = _rows(14, 2, Hk).to(DEV)
    slot = blocks * block - 2
    ops.store_kvcache_fp8(x, x, *args, torch.tensor([slot, slot + 1], dtype=torch.int32, device=DEV))
    codes, e = quantise_ref(x.cpu())
    assert torch.equal(big[0][-1, -2:].cpu(), codes) and torch.equal(exps[1][-1, :, -2:].T.cpu(), e)
    cu = torch.tensor([0, 600], dtype=torch.int32, device=DEV)
    k, _ = ops.load_kvcache_fp8(*args, tables[:1], cu, 600)
    want = dequantise_ref(big[0][tables[0].long()], exps[0][tables[0].long()].transpose(1, 2))
    assert torch.equal(k.double(), want.reshape(-1, Hk, 128)[:600])
    assert _deverr() == 0


def test_decode_captured_replayed_and_on_two_streams(cuda_lib):
    ops = _ops()
    cs = [Cache(20 + i, [2500, 0, 130, 4000], 2, 128) for i in range(2)]
    qs = [_q(30 + i, 4, 8) for i in range(2)]
    devs = [c.dev() for c in cs]
    tables = [c.tables.to(DEV) for c in cs]
    lens = [c.lens_t() for c in cs]
    graphs, outs = [], []
    for i in range(2):
        ops.paged_decode_fp8(qs[i], *devs[i], tables[i], lens[i], SCALE)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_decode_fp8(qs[i], *devs[i], tables[i], lens[i], SCALE))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):  # both graphs at once, eager calls beside them
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = ops.paged_decode_fp8(qs[0], *devs[0], tables[0], lens[0], SCALE)
    torch.cuda.synchronize()
    for i in range(2):
        _check_decode(cs[i], qs[i], outs[i])
    assert torch.equal(eager, outs[0])
    # other lengths in the same graph
    lens[0].copy_(torch.tensor([2, 0, 0, 3999], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    _check_decode(cs[0], qs[0], outs[0], lens[0])


def test_store_then_decode_then_load_as_a_step(cuda_lib):
    """A prompt stored, then decode steps that each store their row first."""
    ops = _ops()
    Hk, Hq, block, L = 2, 8, 64, 190
    f = torch.float8_e4m3fn
    k, v = (torch.zeros(8, block, Hk, 128, dtype=torch.uint8, device=DEV) for _ in "kv")
    ke, ve = (torch.zeros(8, Hk, block, dtype=torch.uint8, device=DEV) for _ in "kv")
    cache = (k.view(f), v.view(f), ke, ve)
    table = torch.tensor([[5, 2, 7, 0]], dtype=torch.int32, device=DEV)
    slot = lambda t: int(table[0, t // block]) * block + t % block  # noqa: E731
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(2, L + 4, Hk, 128, generator=g).to(torch.bfloat16).to(DEV)
    ops.store_kvcache_fp8(rows[0, :L], rows[1, :L], *cache,
                          torch.tensor([slot(t) for t in range(L)], dtype=torch.int32, device=DEV))
    for t in range(L, L + 4):
        q = _q(t, 1, Hq)
        ops.store_kvcache_fp8(rows[0, t:t + 1], rows[1, t:t + 1], *cache,
                              torch.tensor([slot(t)], dtype=torch.int32, device=DEV))
        lens = torch.tensor([t + 1], dtype=torch.int32, device=DEV)
        out = ops.paged_decode_fp8(q, *cache, table, lens, SCALE)
        ref, bound = decode_fp8_ref(q, k, v, ke, ve, table, lens, SCALE)
        assert bool(((out.double() - ref).abs() <= bound).all())
    cu = torch.tensor([0, L + 4], dtype=torch.int32, device=DEV)
    back = ops.load_kvcache_fp8(*cache, table, cu, L + 4)
    for out, x in zip(back, rows):
        codes, exps = quantise_ref(x.cpu())
        assert torch.equal(out.cpu().double(), dequantise_ref(codes, exps))
