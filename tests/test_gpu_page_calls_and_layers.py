"""GPU tests of the layers' decode step right behind page operators that write
its tables, lengths and cache rows, eager and in one CUDA graph."""

import types

import numpy as np
import pytest
import torch

from oracle.attention import paged_decode_ref
from oracle.inputs import bf16, make_paged_batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("rows", [2, 40])
def test_fork_step_free_compact_step(cuda_lib, captured, rows):
    """Row 0 forked over all other rows, a step, the odd branches freed, the pool
    compacted, a step: no other kernel between them."""
    from nanokv_b200 import _lib, ops
    from nanokv_b200.layers.attention import Attention
    from nanokv_b200.utils.context import reset_context, set_context

    Hq, Hk, block, n = 16, 8, 256, 700
    pages = 3 * rows + 5
    pb = make_paged_batch(seed=7, lens=[n] + [5] * (rows - 1), Hq=Hq, Hk=Hk, num_blocks=pages)
    tables = torch.full((rows, 4), -1, dtype=torch.int32)
    tables[:, :pb.block_tables.size(1)] = pb.block_tables
    refs = [0] * pages
    for p in tables.flatten().tolist():
        if p >= 0:
            refs[p] += 1
    a = Attention(Hq, 128, SCALE, Hk, types.SimpleNamespace(kv_compress_enabled=False), 1)
    a.k_cache, a.v_cache = pb.k_cache.to(DEV), pb.v_cache.to(DEV)
    caches = [a.k_cache, a.v_cache]
    t, lens, r = tables.to(DEV), pb.context_lens.to(DEV), _i32(refs)
    src, dst = _i32([0] * (rows - 1)), _i32(list(range(1, rows)))
    odd = _i32(list(range(1, rows, 2)))
    q = bf16(np.random.default_rng(8).standard_normal((rows, Hq, 128), dtype=np.float32))
    k = torch.zeros(rows, Hk, 128, dtype=torch.bfloat16, device=DEV)
    qd, slots = q.to(DEV), _i32([-1] * rows)
    keep = [x.clone() for x in (t, lens, r, *caches)]
    set_context(True, slot_mapping=slots, context_lens=lens, block_tables=t)

    def step():
        new = ops.fork_pages(caches, t, lens, r, src, dst, block)
        first = a.forward(qd, k, k, 0)
        ops.free_pages(t, lens, r, odd, block)
        live = ops.compact_pages(caches, t, r)
        return new, first, live, a.forward(qd, k, k, 0)

    def restore():
        for x, y in zip((t, lens, r, *caches), keep):
            x.copy_(y)
        torch.cuda.synchronize()

    run = step
    if captured:
        step()
        restore()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()

        def run():
            graph.replay()
            return outs
    ref = paged_decode_ref(q, pb.k_cache, pb.v_cache, tables[:1].expand(rows, -1).contiguous(),
                           torch.full((rows,), n, dtype=torch.int32), SCALE)
    for _ in range(5):
        restore()
        new, first, live, second = run()
        torch.cuda.synchronize()
        assert bool((new >= 0).all()) and live.item() == 2 + 1 + (rows - 1) // 2
        assert (first[:, 0].float().cpu() - ref).abs().max().item() <= 2e-2
        got = second[:, 0].float().cpu()
        assert (got[::2] - ref[::2]).abs().max().item() <= 2e-2
        assert bool((got[1::2] == 0).all())
    reset_context()
    assert _lib.read_device_error(clear=True) == 0
