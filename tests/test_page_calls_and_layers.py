"""What the layers vouch for before and after the page operators, which write
tables, lengths and cache rows on the device. Host logic only: no GPU."""

import types

import numpy as np
import pytest
import torch

I32 = torch.int32


@pytest.fixture
def calls(monkeypatch):
    """ops with the launches taken out; the metadata_ready of every decode step."""
    from nanokv_b200 import build, ops
    from nanokv_b200.utils import context

    build.build()
    seen = []

    def decode_step(q, *args, metadata_ready=False, **kw):
        seen.append(metadata_ready)
        return q

    monkeypatch.setattr(ops, "decode_step", decode_step)
    monkeypatch.setattr(ops, "_one_device", lambda *a: 0)
    monkeypatch.setattr(ops, "_call", lambda *a: None)
    monkeypatch.setattr(context, "_PAGES_CALLED", False, raising=False)
    yield seen
    context.reset_context()


def _layer(kind):
    from nanokv_b200.layers import attention, kvchat

    cfg = types.SimpleNamespace(kv_compress_enabled=False, kv_compress_N=4, kv_compress_S=9, kv_compress_R=5)
    module = {"periodic": attention, "threshold": kvchat}[kind]
    a = module.Attention(4, 128, 0.1, 2, cfg, 1)
    a.k_cache = a.v_cache = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    return a


def _forward(a):
    a.forward(torch.zeros(2, 4, 128), torch.zeros(2, 2, 128), torch.zeros(2, 2, 128), 0)


def _page_calls():
    from nanokv_b200 import ops

    cache = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    t, n, r = torch.zeros(2, 1, dtype=I32), torch.zeros(2, dtype=I32), torch.ones(2, dtype=I32)
    return {"copy": lambda: ops.copy_pages([cache], n, n), "fork": lambda: ops.fork_pages([cache], t, n, r, n, n, 16),
            "free": lambda: ops.free_pages(t, n, r, n, 16), "compact": lambda: ops.compact_pages([cache], t, r)}


def _set_context():
    from nanokv_b200.utils.context import set_context

    set_context(True, slot_mapping=torch.zeros(2, dtype=I32), context_lens=torch.ones(2, dtype=I32),
                block_tables=torch.zeros(2, 1, dtype=I32))


def _upload():
    from nanokv_b200.engine.step_metadata import StepMetadata

    one, two = np.ones(2, dtype=np.int32), np.arange(3, dtype=np.int32)
    StepMetadata(input_ids=one, positions=one, cu_seqlens_q=two, cu_seqlens_k=two, max_seqlen_q=1,
                 max_seqlen_k=1, slot_mapping=one, context_lens=one, logits_indices=one,
                 block_tables=one.reshape(2, 1)).set_context(True, "cpu", pin=False)


@pytest.mark.parametrize("kind", ["periodic", "threshold"])
@pytest.mark.parametrize("name", ["copy", "fork", "free", "compact"])
def test_a_step_behind_a_page_call_does_not_vouch(calls, kind, name):
    a, page = _layer(kind), _page_calls()[name]
    _set_context()
    _forward(a)  # no page operator so far: as ever
    page()
    _forward(a)  # the same Context
    _set_context()
    _forward(a)  # a new one whose tensors may be the ones that the call wrote
    _upload()
    _forward(a)  # copied from the host after the call
    page()
    _forward(a)
    assert calls == [True, False, False, True, False]


def test_an_engine_may_say_where_its_metadata_comes_from(calls):
    from nanokv_b200.utils.context import get_context

    a, page = _layer("periodic"), _page_calls()["fork"]
    page()
    _set_context()
    get_context().metadata_from_host = True
    _forward(a)
    _set_context()
    get_context().metadata_from_host = False
    _forward(a)
    assert calls == [True, False]


@pytest.mark.parametrize("kw,status", [
    (dict(n=0), 0), (dict(n=-1), 1), (dict(rows=None), 1), (dict(out=None), 1), (dict(refs=None), 1),
    (dict(tables=None), 1), (dict(block=0), 1), (dict(mb=-1), 1), (dict(window=-1), 1), (dict(pages=-1), 1),
    (dict(pages=5), 1), (dict(num_rows=-1), 1), (dict(num_pages=-1), 1)])
def test_unshared_rows_refusals(kw, status):
    from nanokv_b200 import _lib, build

    build.build()
    a = dict(rows=16, n=1, tables=16, mb=4, num_rows=2, lens=16, refs=16, num_pages=8, block=16, window=2, pages=1,
             out=16)
    a.update(kw)
    assert _lib.load().nkv_unshared_rows(*a.values(), None) == status


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("entry", ["forward", "forward_qkv"])
def test_compression_of_an_8_bit_cache_is_refused_at_the_first_step(calls, monkeypatch, decode, entry):
    """Whatever the step is: not in the middle of serving, at the first that compresses."""
    from nanokv_b200 import ops
    from nanokv_b200.layers.attention import Attention
    from nanokv_b200.utils.context import set_context

    stored = []
    monkeypatch.setattr(ops, "store_kvcache_fp8", lambda *a: stored.append(a))
    monkeypatch.setattr(ops, "paged_decode_fp8", lambda q, *a: q)
    monkeypatch.setattr(ops, "flash_attn_varlen_func", lambda q, *a, **kw: q)
    q, k = torch.zeros(2, 4, 128), torch.zeros(2, 2, 128)
    monkeypatch.setattr(ops, "qk_norm_rope_store", lambda *a, **kw: (q, k, k))
    for enabled in (False, True):
        cfg = types.SimpleNamespace(kv_compress_enabled=enabled, kv_compress_window_blocks=4,
                                    kv_compress_keep_blocks=2, kv_compress_keep_extra_tokens=1)
        a = Attention(4, 128, 0.1, 2, cfg, 1)
        a.k_cache = a.v_cache = torch.zeros(2, 16, 2, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
        a.k_exp = a.v_exp = torch.zeros(2, 2, 16, dtype=torch.uint8)
        i = torch.zeros(2, dtype=I32)
        set_context(decode, i, i, 1, 1, i, i, None)

        def run():
            if entry == "forward":
                return a.forward(q, k, k, 0)
            return a.forward_qkv(torch.zeros(2, 8 * 128), i, None, None, None, 1e-6, 0)

        if enabled:
            with pytest.raises(ValueError, match="needs a bf16 cache"):
                run()
            assert len(stored) == 1
        else:
            run()
