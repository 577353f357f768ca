"""GPU tests of a compression step on rows that share pages (a forked row and
its branches), with the pages' reference counts in the Context: a row that
would rewrite a shared page is left as it is and flagged."""

import types

import numpy as np
import pytest
import torch

from oracle.inputs import bf16, make_paged_batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _counts(tables, pages):
    refs = [0] * pages
    for row in tables:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return refs


@pytest.mark.parametrize("on_device", [False, True])
@pytest.mark.parametrize("shared", [0, 1, 3, 4])
def test_periodic_step(cuda_lib, on_device, shared):
    """Rows of 1300 tokens in pages of 256: the window is pages 1 to 4, pages 1
    to 3 are rewritten (513 kept tokens and the tail's 20), 4 and 5 given up."""
    from nanokv_b200 import _lib
    from nanokv_b200.layers.attention import Attention
    from nanokv_b200.utils.context import get_context, reset_context, set_context

    L, Hq, Hk = 2, 16, 8
    pb = make_paged_batch(seed=41, lens=[1300, 1300, 1300, 90], Hq=Hq, Hk=Hk)
    tables = pb.block_tables.tolist()
    tables[2][shared] = tables[0][shared]
    pages = pb.k_cache.shape[0]
    refs = _counts(tables, pages)
    rewrites = shared in (1, 2, 3)
    cfg = types.SimpleNamespace(kv_compress_enabled=True, kv_compress_window_blocks=4,
                                kv_compress_keep_blocks=2, kv_compress_keep_extra_tokens=1)
    layers = []
    for _ in range(L):
        a = Attention(Hq, 128, SCALE, Hk, cfg, L)
        a.k_cache, a.v_cache = pb.k_cache.to(DEV), pb.v_cache.to(DEV)
        layers.append(a)
    cl, bt = pb.context_lens.to(DEV), _i32(tables)
    set_context(True, slot_mapping=pb.slot_mapping.to(DEV), context_lens=cl, block_tables=bt)
    ctx = get_context()
    ctx.is_compress_step = True
    ctx.page_ref_counts = _i32(refs)
    if on_device:
        ctx.compress_device_select, ctx.compress_topk = True, 2
        ctx.compress_selected_t = torch.empty(2, dtype=torch.int32, device=DEV)
        ctx.compress_base_context_lens = torch.empty_like(cl)
        ctx.compress_tail_uncompressed_t = _i32([1300, 1300, 0, 0])
        ctx.compress_selected_host = torch.empty(2, dtype=torch.int32).pin_memory()
    else:
        ctx.compress_selected_batch_indices = [0, 1]
        ctx.compress_base_context_lens = cl.clone()
    before = [(a.k_cache.clone(), a.v_cache.clone()) for a in layers]
    for i, a in enumerate(layers):
        a.forward(pb.q.to(DEV), pb.k_new.to(DEV), pb.v_new.to(DEV), i)
    torch.cuda.synchronize()
    reset_context()
    done = [1] if rewrites else [0, 1]
    assert _lib.read_device_error(clear=True) == (_lib.DEVERR_PAGES if rewrites else 0)
    assert cl.tolist() == [789 if b in done else n for b, n in enumerate((1300, 1300, 1300, 90))]
    for b in range(2):
        kept = tables[b][:4] + [-1, -1] + tables[b][6:] if b in done else tables[b]
        assert bt[b].tolist() == kept
    left = [list(row) for row in tables]
    for b in done:
        left[b][4] = left[b][5] = -1
    assert ctx.page_ref_counts.tolist() == _counts(left, pages)
    if on_device:
        assert sorted(x for x in ctx.compress_selected_host.tolist() if x >= 0) == done
    else:
        assert [e["batch_index"] for e in ctx.compression_events] == done
    # the row that shares the page keeps its tokens (its new one is the step's)
    new = int(pb.slot_mapping[2])
    for a, (k0, v0) in zip(layers, before):
        for now, then in ((a.k_cache, k0), (a.v_cache, v0)):
            at = torch.tensor(tables[2][:6], device=DEV)
            same = (now[at] == then[at]).flatten(2).all(-1).reshape(-1)
            assert bool(same[:1299].all()) and tables[2][5] == new // 256


@pytest.mark.parametrize("shared", [False, True])
def test_threshold_step(cuda_lib, shared):
    from nanokv_b200 import _lib
    from nanokv_b200.engine.query_window import QueryWindowManager
    from nanokv_b200.layers.kvchat import Attention
    from nanokv_b200.utils.context import get_context, reset_context, set_kvchat_context

    Hq, Hk, W, S, R = 16, 8, 50, 575, 321
    cfg = types.SimpleNamespace(kv_compress_enabled=True, kv_compress_N=4, kv_compress_S=S,
                                kv_compress_R=R, query_window_size=W)
    pb = make_paged_batch(seed=42, lens=[S, S, 200], Hq=Hq, Hk=Hk)
    tables = pb.block_tables.tolist()
    if shared:
        tables[2][0] = tables[0][0]
    qwm = QueryWindowManager(1, W, Hq, 128, device=DEV)
    qwm.ring.copy_(bf16(np.random.default_rng(3).standard_normal(qwm.ring.shape, dtype=np.float32)))
    for s in (10, 11):
        qwm.activate(s)
    a = Attention(Hq, 128, SCALE, Hk, cfg, 1)
    a.query_window_manager = qwm
    a.k_cache, a.v_cache = pb.k_cache.to(DEV), pb.v_cache.to(DEV)
    cl = pb.context_lens.to(DEV)
    slots = pb.slot_mapping.clone()
    slots[2] = -1
    set_kvchat_context(False, slot_mapping=slots.to(DEV), context_lens=cl, block_tables=_i32(tables))
    ctx = get_context()
    ctx.page_ref_counts = _i32(_counts(tables, pb.k_cache.shape[0]))
    ctx.compress_need_mask, ctx.compress_any, ctx.seq_ids = [True, True, False], True, [10, 11, 12]
    ctx.runtime_compress_S, ctx.runtime_compress_R = S, R
    page0 = a.k_cache[tables[0][0]].clone(), a.v_cache[tables[0][0]].clone()
    a.forward(pb.q.to(DEV), pb.k_new.to(DEV), pb.v_new.to(DEV), 0)
    torch.cuda.synchronize()
    reset_context()
    assert _lib.read_device_error(clear=True) == (_lib.DEVERR_PAGES if shared else 0)
    assert cl.tolist() == [S if shared else R, R, 200]
    assert [e["batch_index"] for e in ctx.compression_events] == ([1] if shared else [0, 1])
    same = torch.equal(a.k_cache[tables[0][0]], page0[0]) and torch.equal(a.v_cache[tables[0][0]], page0[1])
    assert same == shared
    assert not qwm.has(10) and not qwm.has(11)


def test_unshared_rows(cuda_lib):
    """Rows of every kind, in place and out of place, against plain loops."""
    from nanokv_b200 import _lib, ops

    rng = np.random.default_rng(9)
    rows, width, block = 300, 90, 16
    lens = [int(x) for x in rng.integers(0, width * block + 1, rows)]
    tables = rng.integers(-1, 6000, (rows, width)).tolist()
    counts = rng.choice([-1, 0, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 2], 6000).tolist()
    names = [int(x) for x in rng.permutation(rows)] + [-1]
    t, n, r = _i32(tables), _i32(lens), _i32(counts)
    for window, kept, use in ((4, 33, n), (70, 1100, n), (1, 1, n), (0, 40, None), (0, 1440, None)):
        want = []
        for b in names:
            first = lens[b] // block - window if use is not None else 0
            pages = tables[b][max(first, 0):max(first + -(-kept // block), 0)]
            want.append(-1 if b < 0 or any(p >= 0 and counts[p] > 1 for p in pages) else b)
        given = _i32(names)
        out = ops.unshared_rows(given, t, r, block, kept, lens=use, window_blocks=window)
        assert out.tolist() == want and given.tolist() == names
        assert 1 < sum(w >= 0 for w in want) < rows or kept > 500
        assert _lib.read_device_error(clear=True) == _lib.DEVERR_PAGES
        ops.unshared_rows(given, t, r, block, kept, lens=use, window_blocks=window, out=given)
        assert given.tolist() == want
        _lib.read_device_error(clear=True)
        assert ops.unshared_rows(given, t, r, block, kept, lens=use, window_blocks=window).tolist() == want
        assert _lib.read_device_error(clear=True) == 0
    assert ops.unshared_rows(_i32([rows, -2, -1]), t, r, block, 1).tolist() == [-1] * 3
    assert _lib.read_device_error(clear=True) == _lib.DEVERR_PAGES
