"""GPU tests of the page operators -- nkv_copy_pages, nkv_fork_pages,
nkv_free_pages, nkv_compact_pages -- against plain loops (oracle/cache_pages.py).
Everything is moved or counted, so every comparison is exact."""

from collections import Counter

import numpy as np
import pytest
import torch

from oracle.cache_pages import PageState, cache_bytes

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ops():
    from nanokv_b200 import ops
    return ops


def _lib():
    from nanokv_b200 import _lib
    return _lib


def _deverr():
    return _lib().read_device_error(clear=True)


def _caches(seed, kind, pages, block, Hk, layers=2):
    """(tensors on the device, page_dim) of a cache."""
    rng = np.random.default_rng(seed)

    def raw(*shape):
        return torch.from_numpy(rng.integers(0, 255, shape, dtype=np.uint8)).to(DEV)

    if kind == "stack":  # the whole model's bf16 cache in one tensor
        return [raw(2, layers, pages, block, Hk, 256).view(torch.bfloat16)], 2
    if kind == "views":  # K and V of every layer
        return [raw(pages, block, Hk, 256).view(torch.bfloat16) for _ in range(2 * layers)], 0
    f = torch.float8_e4m3fn  # an 8-bit cache with its exponent bytes
    if kind == "fp8":
        return [raw(pages, block, Hk, 128).view(f), raw(pages, block, Hk, 128).view(f),
                raw(pages, Hk, block), raw(pages, Hk, block)], 0
    return [raw(2, layers, pages, block, Hk, 128).view(f), raw(2, layers, pages, Hk, block)], 2


def _state(seed, lens, rows, pages, block, width):
    """A table whose used rows hold `lens`, over shuffled pages; every other used row shares its full pages with the one before."""
    rng = np.random.default_rng(seed)
    perm = list(rng.permutation(pages))
    tables = [[-1] * width for _ in range(rows)]
    row_lens = [0] * rows
    refs = [0] * pages
    used = list(rng.permutation(rows)[:len(lens)])
    for i, (row, n) in enumerate(zip(used, lens)):
        row, row_lens[row] = int(row), n
        for j in range(-(-n // block)):
            if i % 2 and j < min(n, lens[i - 1]) // block:
                p = tables[int(used[i - 1])][j]
            else:
                p = int(perm.pop())
            tables[row][j] = p
            refs[p] += 1
    return tables, row_lens, refs, [int(r) for r in used]


def _dev(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _same(ref, caches, page_dim, tables=None, lens=None, refs=None):
    for c, want in zip(caches, ref.caches):
        assert torch.equal(cache_bytes(c, page_dim).cpu(), want)
    if tables is not None:
        assert tables.cpu().tolist() == ref.tables
    if lens is not None:
        assert lens.cpu().tolist() == ref.lens
    if refs is not None:
        assert refs.cpu().tolist() == ref.refs


def _ref(tables, lens, refs, caches, page_dim, block):
    return PageState(tables, lens, refs, [cache_bytes(c, page_dim).cpu().clone() for c in caches], block)


KINDS = ["stack", "views", "fp8", "fp8_stack"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pages,block,Hk,n", [(3, 16, 1, 1), (40, 16, 3, 13), (9, 256, 8, 4), (70, 48, 2, 33)])
def test_copy_pages(cuda_lib, kind, pages, block, Hk, n):
    caches, pd = _caches(n, kind, pages, block, Hk)
    rng = np.random.default_rng(n)
    perm = [int(x) for x in rng.permutation(pages)]
    dst = perm[:n]
    src = [perm[n + int(i)] for i in rng.integers(0, pages - n, n)]  # pages may be read twice
    ref = _ref([], [], [], caches, pd, block)
    ref.copy_pages(src, dst)
    _ops().copy_pages(caches, _dev(src), _dev(dst), page_dim=pd)
    _same(ref, caches, pd)
    assert _deverr() == 0


def test_copy_pages_refuses_ambiguous_pairs(cuda_lib):
    caches, pd = _caches(1, "fp8", 12, 16, 2)
    src = [0, 1, 2, 3, -1, 4, 12, 5, -2]
    dst = [6, 7, 7, 0, -1, 12, 8, 5, 9]  # 7 twice; 0 is read; pages past the end; 5 onto itself
    ref = _ref([], [], [], caches, pd, 16)
    ref.copy_pages(src, dst)
    _ops().copy_pages(caches, _dev(src), _dev(dst), page_dim=pd)
    _same(ref, caches, pd)
    assert _deverr() == _lib().DEVERR_PAGES


FORKS = [
    # lens, rows, block, branches, spare pages
    ([700], 6, 256, 4, 6),
    ([1, 16, 17, 31, 0, 33, 48], 40, 16, 3, 30),
    ([128, 256, 64], 12, 64, 2, 0),
    ([5] * 90, 300, 32, 2, 200),
    ([200, 1500, 33, 100, 64, 65], 2000, 64, 5, 40),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,rows,block,branches,spare", FORKS, ids=[str(i) for i in range(len(FORKS))])
def test_fork_pages(cuda_lib, kind, lens, rows, block, branches, spare):
    ops = _ops()
    pages = sum(-(-n // block) for n in lens) + spare
    width = max(-(-n // block) for n in lens) + 2
    tables, row_lens, refs, used = _state(3, lens, rows, pages, block, width)
    caches, pd = _caches(4, kind, pages, block, 2)
    free_rows = [r for r in range(rows) if r not in used]
    src = [r for r in used for _ in range(branches)]
    dst = free_rows[::-1][:len(src)]
    ref = _ref(tables, row_lens, refs, caches, pd, block)
    t, n, r = _dev(tables), _dev(row_lens), _dev(refs)
    assert ref.fork(src, dst) == ops.fork_pages(caches, t, n, r, _dev(src), _dev(dst), block, page_dim=pd).tolist()
    _same(ref, caches, pd, t, n, r)
    # the branches replaced by forks of other rows, some of them padding
    src, dst = src[::-1], list(dst)
    src[0] = dst[0] = -1
    assert ref.fork(src, dst) == ops.fork_pages(caches, t, n, r, _dev(src), _dev(dst), block, page_dim=pd).tolist()
    _same(ref, caches, pd, t, n, r)
    assert _deverr() == 0
    # dropped: everything as it was before
    ref.free([d for d in dst if d >= 0], False)
    ops.free_pages(t, n, r, _dev(dst), block)
    _same(ref, caches, pd, t, n, r)
    assert _deverr() == 0


def test_fork_refusals_and_an_empty_pool(cuda_lib):
    ops = _ops()
    block, lens, rows = 16, [20, 5, 32, 40], 12
    pages = sum(-(-n // block) for n in lens)  # two of them free: the last row shares two
    tables, row_lens, refs, used = _state(5, lens, rows, pages, block, 4)
    caches, pd = _caches(6, "fp8", pages, block, 2)
    a, b, c, d = used
    f = [r for r in range(rows) if r not in used]
    # a target that is a source, one named twice, rows past the table; then three wants for two free pages
    src = [a, a, b, b, 12, a, a, c, b, d]
    dst = [b, f[0], f[1], f[1], f[2], -3, f[3], f[4], f[5], f[6]]
    ref = _ref(tables, row_lens, refs, caches, pd, block)
    t, n, r = _dev(tables), _dev(row_lens), _dev(refs)
    got = ops.fork_pages(caches, t, n, r, _dev(src), _dev(dst), block, page_dim=pd).tolist()
    assert got == ref.fork(src, dst)
    assert got.count(-2) == 7 and got[7] == -1
    _same(ref, caches, pd, t, n, r)
    assert _deverr() == _lib().DEVERR_PAGES


def test_fork_flags_a_page_that_nobody_holds(cuda_lib):
    caches, pd = _caches(7, "views", 5, 16, 1)
    t, n, r = _dev([[0, 3, -1], [-1, -1, -1]]), _dev([32, 0]), _dev([1, 1, 1, 0, 1])
    assert _ops().fork_pages(caches, t, n, r, _dev([0]), _dev([1]), 16, page_dim=pd).tolist() == [-1]
    assert _deverr() == _lib().DEVERR_PAGES


def test_fork_of_many_rows_and_a_large_pool(cuda_lib):
    """More forks and pages than the planning CTA has threads: 3,000 forks, the free pages past the first 16k."""
    ops = _ops()
    block, rows, width, pages = 16, 4000, 3, 21000
    lens = [5 + (i % 40) for i in range(900)]
    tables, row_lens, refs, used = _state(13, lens, rows, pages, block, width)
    for p in range(16500):  # the low pages are taken by others
        refs[p] = max(refs[p], 1)
    caches, pd = _caches(14, "fp8", pages, block, 1)
    free_rows = [r for r in range(rows) if r not in set(used)][:3000]
    src = [used[i % len(used)] for i in range(3000)]
    ref = _ref(tables, row_lens, refs, caches, pd, block)
    t, n, r = _dev(tables), _dev(row_lens), _dev(refs)
    # PageState counts repeats in a list: no repeats here, so its loops are kept short
    ref_out = _fork_without_checks(ref, src, free_rows)
    out = ops.fork_pages(caches, t, n, r, _dev(src), _dev(free_rows), block, page_dim=pd)
    assert out.tolist() == ref_out
    _same(ref, caches, pd, t, n, r)
    assert _deverr() == 0


def _fork_without_checks(ref, src, dst):
    """PageState.fork for targets that are distinct and no sources."""
    free = [p for p, r in enumerate(ref.refs) if r <= 0]
    out = []
    for s, d in zip(src, dst):
        full, tail = divmod(ref.lens[s], ref.block)
        page = free.pop(0) if tail else -1
        for j in range(full):
            ref.tables[d][j] = ref.tables[s][j]
            ref.refs[ref.tables[s][j]] += 1
        if tail:
            ref.tables[d][full], ref.refs[page] = page, 1
            ref.copy(ref.tables[s][full], page, tail)
        ref.lens[d] = ref.lens[s]
        out.append(page)
    return out


@pytest.mark.parametrize("trim", [False, True])
@pytest.mark.parametrize("n_rows,block,width", [(3, 16, 5), (400, 64, 30), (9, 256, 700)])
def test_free_pages(cuda_lib, n_rows, block, width, trim):
    ops = _ops()
    rng = np.random.default_rng(n_rows)
    lens = [int(x) for x in rng.integers(0, (width - 1) * block, n_rows)]
    pages = sum(-(-n // block) for n in lens) + 1
    tables, row_lens, refs, used = _state(7, lens, n_rows + 5, pages, block, width)
    if trim:  # the rows were shortened on the device
        row_lens = [int(n * rng.uniform(0, 1)) if n else 0 for n in row_lens]
    rows = used[::2] + [-1] + used[:1]  # padding, and one row twice
    ref = _ref(tables, row_lens, refs, [], 0, block)
    t, n, r = _dev(tables), _dev(row_lens), _dev(refs)
    ref.free(rows[:-1], trim)
    ops.free_pages(t, n, r, _dev(rows), block, trim=trim)
    _same(ref, [], 0, t, n, r)
    assert _deverr() == 0
    ref.free(used, trim)
    ops.free_pages(t, n, r, _dev(used), block, trim=trim)
    _same(ref, [], 0, t, n, r)
    assert _deverr() == 0


def test_free_pages_flags_bad_state(cuda_lib):
    ops = _ops()
    t, n, r = _dev([[0, 1], [0, 9], [2, -1]]), _dev([20, 20, 3]), _dev([1, 1, 0, 0])
    ops.free_pages(t, n, r, _dev([0, 1, 2, 3, -2]), 16)
    # page 0 is released twice, page 9 does not exist, page 2 was free, rows 3 and -2 do not exist
    assert _deverr() == _lib().DEVERR_PAGES
    assert r.tolist() == [0, 0, 0, 0] and n.tolist() == [0, 0, 0]
    assert t.tolist() == [[-1, -1]] * 3


COMPACT = [
    # pages, live, rows, block, Hk
    (1, 1, 1, 16, 1),
    (2, 1, 3, 16, 2),
    (50, 0, 2, 16, 1),
    (50, 50, 7, 16, 1),
    (96, 23, 16, 32, 3),
    (1025, 400, 64, 16, 1),
    (5000, 2600, 300, 16, 1),
    (40000, 17000, 500, 16, 1),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("pages,live,rows,block,Hk", COMPACT)
def test_compact_pages(cuda_lib, kind, in_place, pages, live, rows, block, Hk):
    ops = _ops()
    rng = np.random.default_rng(pages + live)
    width = -(-live // rows) + 2
    ids = [int(x) for x in rng.permutation(pages)[:live]]
    tables = [[-1] * width for _ in range(rows)]
    for i, p in enumerate(ids):
        tables[i % rows][i // rows] = p
        if i % 3 == 0:  # shared with another row
            tables[(i + 1) % rows][width - 1] = p
    held = Counter(p for row in tables for p in row)
    refs = [held[p] for p in range(pages)]
    caches, pd = _caches(8, kind, pages, block, Hk, layers=1)
    ref = _ref(tables, [], refs, caches, pd, block)
    t, r = _dev(tables), _dev(refs)
    outs = {} if in_place else {"out_block_tables": torch.empty_like(t), "out_ref_counts": torch.empty_like(r)}
    count = ops.compact_pages(caches, t, r, page_dim=pd, **outs)
    if not in_place:
        assert t.tolist() == tables and r.tolist() == refs  # the inputs stay
        t, r = outs["out_block_tables"], outs["out_ref_counts"]
    assert count.item() == ref.compact()
    _same(ref, caches, pd, t, None, r)
    assert _deverr() == 0


def test_compact_flags_entries_that_name_no_page_in_use(cuda_lib):
    caches, pd = _caches(9, "views", 6, 16, 1)
    t, r = _dev([[5, 3, 9]]), _dev([0, 1, 0, 0, 0, 1])
    _ops().compact_pages(caches, t, r, page_dim=pd)
    assert _deverr() == _lib().DEVERR_PAGES
    assert t.tolist() == [[0, 3, 9]] and r.tolist() == [1, 1, 0, 0, 0, 0]


def test_many_layer_views_in_one_call(cuda_lib):
    """36 layers of an 8-bit cache as per-layer views: 144 tensors."""
    ops = _ops()
    caches = [c for i in range(36) for c in _caches(i, "fp8", 10, 16, 1)[0]]
    tables, lens, refs, used = _state(2, [37], 3, 10, 16, 4)
    ref = _ref(tables, lens, refs, caches, 0, 16)
    t, n, r = _dev(tables), _dev(lens), _dev(refs)
    dst = [x for x in range(3) if x not in used]
    assert ref.fork(used * 2, dst) == ops.fork_pages(caches, t, n, r, _dev(used * 2), _dev(dst), 16).tolist()
    ref.free(used, False)
    ops.free_pages(t, n, r, _dev(used), 16)
    ref.compact()
    ops.compact_pages(caches, t, r)
    _same(ref, caches, 0, t, n, r)


def test_pages_past_32_bits(cuda_lib):
    """Pages whose offsets need more than 32 bits, forked and compacted."""
    ops = _ops()
    pages, block, Hk = 8400, 256, 8
    cache = torch.empty(pages, block, Hk, 128, dtype=torch.bfloat16, device=DEV)
    assert cache.numel() * 2 > 1 << 32
    mark = torch.arange(block * Hk * 128, device=DEV).view(block, Hk, 128).remainder(251).to(torch.bfloat16)
    for i, p in enumerate((8397, 8399)):
        cache[p] = mark + i
    t, n, r = _dev([[8397, 8399], [-1, -1]]), _dev([256 + 100, 0]), torch.ones(pages, dtype=torch.int32, device=DEV)
    r[8398] = 0
    cache[8398] = 7
    out = ops.fork_pages([cache], t, n, r, _dev([0]), _dev([1]), block)
    assert out.tolist() == [8398] and t.tolist() == [[8397, 8399], [8397, 8398]]
    assert torch.equal(cache[8398, :100], mark[:100] + 1) and bool((cache[8398, 100:] == 7).all())
    r = torch.zeros(pages, dtype=torch.int32, device=DEV)
    r[8397], r[8398], r[8399] = 2, 1, 1
    assert ops.compact_pages([cache], t, r).item() == 3
    assert t.tolist() == [[0, 2], [0, 1]]
    assert torch.equal(cache[0], mark) and torch.equal(cache[2], mark + 1)
    assert torch.equal(cache[1, :100], mark[:100] + 1)


def test_captured_calls_replay(cuda_lib):
    """A fork, a free and a compaction in one graph, replayed from the same state."""
    ops = _ops()
    block, lens = 32, [100, 40, 64]
    pages = 30
    tables, row_lens, refs, used = _state(11, lens, 9, pages, block, 5)
    caches, pd = _caches(12, "fp8_stack", pages, block, 2)
    dst = [x for x in range(9) if x not in used][:4]
    src = [used[0], used[1], used[2], used[0]]
    drop = [used[1], dst[0]]
    t, n, r = _dev(tables), _dev(row_lens), _dev(refs)
    s, d, f = _dev(src), _dev(dst), _dev(drop)
    keep = [x.clone() for x in (t, n, r, *caches)]

    def step():
        out = ops.fork_pages(caches, t, n, r, s, d, block, page_dim=pd)
        ops.free_pages(t, n, r, f, block)
        return out, ops.compact_pages(caches, t, r, page_dim=pd)

    step()
    torch.cuda.synchronize()
    for a, b in zip((t, n, r, *caches), keep):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, live = step()
    for _ in range(3):
        for a, b in zip((t, n, r, *caches), keep):
            a.copy_(b)
        ref = _ref(tables, row_lens, refs, caches, pd, block)
        graph.replay()
        torch.cuda.synchronize()
        assert out.tolist() == ref.fork(src, dst)
        ref.free(drop, False)
        assert live.item() == ref.compact()
        _same(ref, caches, pd, t, n, r)
    assert _deverr() == 0


def test_a_life_of_an_8_bit_cache(cuda_lib):
    """Prompt stored, forked, the branches decoding on their own, a row freed,
    the pool compacted: attention over the result as over the rows themselves."""
    from oracle.fp8_cache import decode_fp8_ref

    ops = _ops()
    Hq, Hk, block, L, pages = 8, 2, 32, 75, 20
    f = torch.float8_e4m3fn
    g = torch.Generator().manual_seed(2)
    k, v = (torch.zeros(pages, block, Hk, 128, dtype=torch.uint8, device=DEV) for _ in "kv")
    ke, ve = (torch.zeros(pages, Hk, block, dtype=torch.uint8, device=DEV) for _ in "kv")
    cache = [k.view(f), v.view(f), ke, ve]
    t, n = _dev([[9, 14, 3, -1], [11, -1, -1, -1], [-1] * 4, [-1] * 4]), _dev([L, 20, 0, 0])
    r = torch.zeros(pages, dtype=torch.int32, device=DEV)
    r[torch.tensor([9, 14, 3, 11], device=DEV)] = 1
    x = torch.randn(2, L + 20, Hk, 128, generator=g).to(torch.bfloat16).to(DEV)

    def slots(row, positions):
        table = t[row].tolist()
        return _dev([table[p // block] * block + p % block for p in positions])

    s = torch.cat([slots(0, range(L)), slots(1, range(20))])
    ops.store_kvcache_fp8(x[0], x[1], *cache, s)
    assert ops.fork_pages(cache, t, n, r, _dev([0, 0]), _dev([2, 3]), block).tolist() == [0, 1]
    new = torch.randn(2, 3, Hk, 128, generator=g).to(torch.bfloat16).to(DEV)
    n[torch.tensor([0, 2, 3], device=DEV)] += 1
    ops.store_kvcache_fp8(new[0], new[1], *cache, torch.cat([slots(i, [L]) for i in (0, 2, 3)]))
    ops.free_pages(t, n, r, _dev([1]), block)
    assert ops.compact_pages(cache, t, r).item() == 5
    assert sorted(set(t.flatten().tolist())) == [-1, 0, 1, 2, 3, 4]
    q = torch.randn(4, Hq, 128, generator=g).to(torch.bfloat16).to(DEV)
    out = ops.paged_decode_fp8(q, *cache, t, n, 128 ** -0.5)
    # the same rows in a cache without sharing
    k2, v2 = (torch.zeros(16, block, Hk, 128, dtype=torch.uint8, device=DEV) for _ in "kv")
    ke2, ve2 = (torch.zeros(16, Hk, block, dtype=torch.uint8, device=DEV) for _ in "kv")
    t2 = torch.arange(16, dtype=torch.int32, device=DEV).view(4, 4)
    for i, row in enumerate((0, 2, 3)):
        rows = torch.cat([x[:, :L], new[:, i:i + 1]], 1)
        at = torch.tensor([row * 4 * block + p for p in range(L + 1)], dtype=torch.int32, device=DEV)
        ops.store_kvcache_fp8(rows[0], rows[1], k2.view(f), v2.view(f), ke2, ve2, at)
    ref, bound = decode_fp8_ref(q, k2, v2, ke2, ve2, t2, n, 128 ** -0.5)
    assert bool(((out.double() - ref).abs() <= bound).all())
    assert _deverr() == 0
