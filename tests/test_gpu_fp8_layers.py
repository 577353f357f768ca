"""GPU tests of the layers over an 8-bit cache (Attention.forward /
forward_qkv: prompt, prompt chunk over a cached prefix, mixed step, decode),
and of the pages a compression step frees on the device.

What the layer stores is exact; what it attends over is the stored rows, so
its outputs are held to the oracle's on those rows: decode to the bound of
oracle/fp8_cache.py, prefill to the prefill tests' tolerances (max-abs 2e-2,
relative 1e-2)."""

import types

import numpy as np
import pytest
import torch

from oracle.attention import varlen_attention_ref
from oracle.cache_pages import PageState
from oracle.fp8_cache import decode_fp8_ref, dequantise_ref, quantise_ref, sequence_ref, store_fp8_ref
from oracle.inputs import bf16, make_paged_batch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def _cfg(**kw):
    base = dict(kv_compress_enabled=False, kv_compress_window_blocks=4, kv_compress_keep_blocks=2,
                kv_compress_keep_extra_tokens=1)
    base.update(kw)
    return types.SimpleNamespace(**base)


class Layer:
    """An Attention over an empty 8-bit cache and the oracle's copy of it."""

    def __init__(self, Hq, Hk, blocks, block, **cfg):
        from nanokv_b200.layers.attention import Attention

        self.attn = Attention(Hq, 128, SCALE, Hk, _cfg(**cfg), 1)
        self.ref = [torch.zeros(blocks, block, Hk, 128, dtype=torch.uint8) for _ in "kv"] + \
                   [torch.zeros(blocks, Hk, block, dtype=torch.uint8) for _ in "kv"]
        k, v, ke, ve = (t.to(DEV) for t in self.ref)
        f = torch.float8_e4m3fn
        self.attn.k_cache, self.attn.v_cache, self.attn.k_exp, self.attn.v_exp = k.view(f), v.view(f), ke, ve

    def store_ref(self, k, v, slots):
        store_fp8_ref(k, v, *self.ref, slots)

    def check_cache(self):
        a = self.attn
        for t, want in zip((a.k_cache, a.v_cache, a.k_exp, a.v_exp), self.ref):
            assert torch.equal(t.view(torch.uint8).cpu(), want)


def _qkv(seed, T, Hq, Hk):
    rng = np.random.default_rng(seed)
    x = bf16(rng.standard_normal((T, (Hq + 2 * Hk) * 128), dtype=np.float32))
    d = x.to(DEV)
    parts = d.split([Hq * 128, Hk * 128, Hk * 128], dim=-1)
    return x, [p.view(T, -1, 128) for p in parts]


def _rows(x, Hq, Hk):
    T = x.shape[0]
    return (x[:, :Hq * 128].reshape(T, Hq, 128), x[:, Hq * 128:(Hq + Hk) * 128].reshape(T, Hk, 128),
            x[:, (Hq + Hk) * 128:].reshape(T, Hk, 128))


@pytest.mark.parametrize("block,Hq,Hk", [(256, 16, 8), (128, 8, 2)])
def test_prompt_then_chunk_then_decode(cuda_lib, block, Hq, Hk):
    from nanokv_b200.utils.context import get_context, reset_context, set_context

    layer = Layer(Hq, Hk, 14, block)
    tables = torch.tensor([[3, 7, 1, 12], [5, 0, 9, 2]], dtype=torch.int32)
    slot = lambda b, t: int(tables[b, t // block]) * block + t % block  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731

    # ---- two prompts, no cached prefix: attention over the step's own rows
    first = [200, 131]
    x, (q, k, v) = _qkv(1, sum(first), Hq, Hk)
    slots = [slot(b, t) for b in range(2) for t in range(first[b])]
    set_context(False, i32([0, 200, 331]), i32([0, 200, 331]), 200, 200, i32(slots))
    o = layer.attn.forward(q, k, v, 0)
    qr, kr, vr = _rows(x, Hq, Hk)
    layer.store_ref(kr, vr, torch.tensor(slots))
    layer.check_cache()
    ref = varlen_attention_ref(qr, kr, vr, torch.tensor([0, 200, 331]), torch.tensor([0, 200, 331]), SCALE, True)
    assert (o.float().cpu().view(ref.shape) - ref).abs().max().item() <= 2e-2

    # ---- the next chunk of the first, one decode row of the second: over the stored rows
    news, ends = [150, 1], [350, 132]
    x, (q, k, v) = _qkv(2, 151, Hq, Hk)
    slots = [slot(b, t) for b in range(2) for t in range(ends[b] - news[b], ends[b])]
    for total in (0, 482):  # read from the device, or given by the host
        set_context(False, i32([0, 150, 151]), i32([0, 350, 482]), 150, 350, i32(slots), None, tables.to(DEV))
        get_context().total_seqlen_k = total
        o = layer.attn.forward(q, k, v, 0)
        qr, kr, vr = _rows(x, Hq, Hk)
        layer.store_ref(kr, vr, torch.tensor(slots))
        layer.check_cache()
        rows = [torch.cat([sequence_ref(layer.ref[i], layer.ref[2 + i], tables[b], ends[b]) for b in range(2)])
                for i in range(2)]
        ref = varlen_attention_ref(qr, rows[0].to(torch.bfloat16), rows[1].to(torch.bfloat16),
                                   torch.tensor([0, 150, 151]), torch.tensor([0, 350, 482]), SCALE, True)
        got = o.float().cpu().view(ref.shape)
        assert (got - ref).abs().max().item() <= 2e-2
        assert ((got - ref).norm() / ref.norm()).item() <= 1e-2

    # ---- decode steps
    for step in range(3):
        lens = [351 + step, 133 + step]
        x, (q, k, v) = _qkv(3 + step, 2, Hq, Hk)
        slots = [slot(b, lens[b] - 1) for b in range(2)]
        set_context(True, slot_mapping=i32(slots), context_lens=i32(lens), block_tables=tables.to(DEV))
        o = layer.attn.forward(q, k, v, 0)
        qr, kr, vr = _rows(x, Hq, Hk)
        layer.store_ref(kr, vr, torch.tensor(slots))
        layer.check_cache()
        assert o.shape == (2, 1, Hq, 128)
        ref, bound = decode_fp8_ref(qr, *layer.ref, tables, torch.tensor(lens), SCALE)
        assert bool(((o.cpu().double().view(ref.shape) - ref).abs() <= bound).all())
    reset_context()


def test_forward_qkv_stores_the_rotated_rows(cuda_lib):
    from nanokv_b200.utils.context import reset_context, set_context
    from oracle.norm_rope import qk_norm_rope_store_ref, rope_cache

    Hq, Hk, block, T = 8, 2, 64, 3
    layer = Layer(Hq, Hk, 6, block)
    x, _ = _qkv(9, T, Hq, Hk)
    g = torch.Generator().manual_seed(1)
    qw, kw = ((1 + 0.1 * torch.randn(128, generator=g)).to(torch.bfloat16) for _ in "qk")
    pos, cs = torch.tensor([5, 70, 0]), rope_cache(128, 10000.0)
    tables = torch.tensor([[4, -1], [1, 3], [0, -1]], dtype=torch.int32)
    lens = torch.tensor([6, 71, 1], dtype=torch.int32)
    slots = torch.tensor([4 * 64 + 5, 3 * 64 + 6, 0], dtype=torch.int32)
    set_context(True, slot_mapping=slots.to(DEV), context_lens=lens.to(DEV), block_tables=tables.to(DEV))
    o = layer.attn.forward_qkv(x.to(DEV), pos.to(DEV), qw.to(DEV), kw.to(DEV), cs.to(DEV), 1e-6, 0)
    reset_context()
    q, k, _ = qk_norm_rope_store_ref(x, pos, cs, qw, kw, 1e-6, Hq, Hk, None, None, None)
    a = layer.attn
    for row, s in enumerate(slots.tolist()):
        # v is copied before it is quantised: exact; a rotated k element may be one bf16 step off,
        # which the quantisation may turn into one of its own steps
        codes, exps = quantise_ref(_rows(x, Hq, Hk)[2][row])
        assert torch.equal(a.v_cache.view(torch.uint8)[s // block, s % block].cpu(), codes)
        assert torch.equal(a.v_exp[s // block, :, s % block].cpu(), exps)
        got = dequantise_ref(a.k_cache.view(torch.uint8)[s // block, s % block].cpu(),
                             a.k_exp[s // block, :, s % block].cpu())
        top = k[row].double().abs().amax(-1, keepdim=True)
        step = 2.0 ** -4 * torch.maximum(k[row].double().abs(), top * 2.0 ** -13) * (1 + 2.0 ** -6) + 2.0 ** -7 * k[row].double().abs()
        assert bool(((got - k[row].double()).abs() <= step).all())
    ref, bound = decode_fp8_ref(q, *(t.view(torch.uint8).cpu() for t in (a.k_cache, a.v_cache, a.k_exp, a.v_exp)),
                                tables, lens, SCALE)
    # q too may be a bf16 step off in places: the bound of the rotated q's own rounding, 2^-7 of the scores
    assert (o.cpu().double().view(ref.shape) - ref).abs().max().item() <= bound.max().item() + 2e-2


def test_layer_refuses_compression_of_an_8_bit_cache(cuda_lib):
    from nanokv_b200 import ops
    from nanokv_b200.utils.context import get_context, reset_context, set_context

    layer = Layer(8, 2, 6, 128, kv_compress_enabled=True)
    _, (q, k, v) = _qkv(10, 1, 8, 2)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    set_context(True, slot_mapping=i32([0]), context_lens=i32([1]), block_tables=i32([[0]]))
    get_context().is_compress_step = True
    with pytest.raises(ValueError, match="bf16 cache"):
        layer.attn.forward(q, k, v, 0)
    reset_context()
    a = layer.attn
    with pytest.raises(AssertionError):  # the bf16 calls take no 8-bit cache
        ops.decode_step(q, k, v, a.k_cache, a.v_cache, i32([0]), i32([[0]]), i32([1]), SCALE)


def test_decode_step_of_several_layers_in_a_graph(cuda_lib):
    """Store + decode of three layers captured once and replayed with other rows and lengths."""
    from nanokv_b200.utils.context import reset_context, set_context

    Hq, Hk, block = 16, 4, 128
    layers = [Layer(Hq, Hk, 9, block) for _ in range(3)]
    rng = np.random.default_rng(5)
    tables = torch.tensor([[2, 4, 6, 8], [1, 3, 5, 7]], dtype=torch.int32)
    for layer in layers:  # something to attend to
        rows = bf16(rng.standard_normal((2, 9 * block, Hk, 128), dtype=np.float32))
        layer.store_ref(rows[0], rows[1], torch.arange(9 * block))
        for t, want in zip((layer.attn.k_cache, layer.attn.v_cache, layer.attn.k_exp, layer.attn.v_exp), layer.ref):
            t.view(torch.uint8).copy_(want.to(DEV))
    slots = torch.zeros(2, dtype=torch.int32, device=DEV)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    xs = [torch.zeros(2, (Hq + 2 * Hk) * 128, dtype=torch.bfloat16, device=DEV) for _ in layers]
    set_context(True, slot_mapping=slots, context_lens=lens, block_tables=tables.to(DEV))

    def step():
        outs = []
        for layer, x in zip(layers, xs):
            q, k, v = (p.view(2, -1, 128) for p in x.split([Hq * 128, Hk * 128, Hk * 128], dim=-1))
            outs.append(layer.attn.forward(q, k, v, 0))
        return outs

    slots.fill_(-1)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for n in ([300, 200], [301, 201], [512, 1]):
        where = [int(tables[b, (n[b] - 1) // block]) * block + (n[b] - 1) % block for b in range(2)]
        new = [_qkv(sum(n) + i, 2, Hq, Hk)[0] for i in range(3)]
        slots.copy_(torch.tensor(where, dtype=torch.int32))
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        for x, y in zip(xs, new):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for layer, x, o in zip(layers, new, outs):
            q, k, v = _rows(x, Hq, Hk)
            layer.store_ref(k, v, torch.tensor(where))
            layer.check_cache()
            ref, bound = decode_fp8_ref(q, *layer.ref, tables, torch.tensor(n), SCALE)
            assert bool(((o.cpu().double().view(ref.shape) - ref).abs() <= bound).all())
    reset_context()


@pytest.mark.parametrize("on_device", [False, True])
def test_compression_step_frees_its_pages_on_the_device(cuda_lib, on_device):
    from nanokv_b200.layers.attention import Attention
    from nanokv_b200.utils.context import get_context, reset_context, set_context

    L, Hq, Hk = 2, 16, 8
    lens = [1300, 2100, 700, 1800]
    pb = make_paged_batch(seed=70, lens=lens, Hq=Hq, Hk=Hk)
    layers = []
    for _ in range(L):
        a = Attention(Hq, 128, SCALE, Hk, _cfg(kv_compress_enabled=True), L)
        a.k_cache, a.v_cache = pb.k_cache.to(DEV), pb.v_cache.to(DEV)
        layers.append(a)
    refs = [0] * pb.k_cache.shape[0]
    for row in pb.block_tables.tolist():
        for p in row:
            if p >= 0:
                refs[p] += 1
    refs[pb.block_tables[1, 7]] += 1  # a page that another table shares
    ref = PageState(pb.block_tables.tolist(), [789, 1589, 700, 1289], refs, [], 256)  # its own counts
    ref.free([0, 1, 3], True)
    cl, bt = pb.context_lens.to(DEV), pb.block_tables.to(DEV)
    set_context(True, slot_mapping=pb.slot_mapping.to(DEV), context_lens=cl, block_tables=bt)
    ctx = get_context()
    ctx.is_compress_step = True
    ctx.page_ref_counts = torch.tensor(refs, dtype=torch.int32, device=DEV)
    if on_device:
        ctx.compress_device_select, ctx.compress_topk = True, 5
        ctx.compress_selected_t = torch.empty(5, dtype=torch.int32, device=DEV)
        ctx.compress_base_context_lens = torch.empty_like(cl)
        ctx.compress_tail_uncompressed_t = torch.tensor([1300, 2100, 0, 1800], dtype=torch.int32, device=DEV)
    else:
        ctx.compress_selected_batch_indices = [0, 1, 3]
        ctx.compress_base_context_lens = cl.clone()
    for i, a in enumerate(layers):
        a.forward(pb.q.to(DEV), pb.k_new.to(DEV), pb.v_new.to(DEV), i)
    torch.cuda.synchronize()
    reset_context()
    assert cl.tolist() == ref.lens
    assert bt.tolist() == ref.tables
    assert ctx.page_ref_counts.tolist() == ref.refs
