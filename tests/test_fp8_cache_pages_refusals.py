"""Refusals of the 8-bit cache and page calls, and the oracle's rounding: no GPU."""

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle.fp8_cache import E4M3, dequantise_ref, quantise_ref, row_exponent


def _lib():
    from nanokv_b200 import _lib, build

    build.build()
    return _lib.load()


P = 16  # an aligned, non-null address that is never followed


def _store(lib, **kw):
    a = dict(key=P, ks=1024, value=P, vs=1024, k=P, v=P, ke=P, ve=P, blocks=4, block=256, slots=P, n=2,
             Hk=8, D=128)
    a.update(kw)
    return lib.nkv_store_kvcache_fp8(*a.values(), None)


def _load(lib, **kw):
    a = dict(k=P, v=P, ke=P, ve=P, blocks=4, block=256, bt=P, mb=2, cu=P, B=1, n=5, ko=P, kos=1024, vo=P,
             vos=1024, Hk=8, D=128)
    a.update(kw)
    return lib.nkv_load_kvcache_fp8(*a.values(), None)


def _decode(lib, **kw):
    a = dict(q=P, qs=4096, qh=128, k=P, v=P, ke=P, ve=P, blocks=4, bt=P, mb=2, cl=P, out=P, os=4096, B=2,
             Hq=32, Hk=8, D=128, block=256, scale=0.1, ws=P, wsb=1 << 30)
    a.update(kw)
    return lib.nkv_paged_decode_fp8(*a.values(), None)


BAD, UNSUPPORTED, WORKSPACE, ALIGN = 1, 2, 3, 4


@pytest.mark.parametrize("kw,status", [
    (dict(n=0), 0), (dict(blocks=0), 0), (dict(n=-1), BAD), (dict(key=None), BAD), (dict(slots=None), BAD),
    (dict(ke=None), BAD), (dict(D=64), UNSUPPORTED), (dict(block=48), UNSUPPORTED), (dict(block=0), BAD),
    (dict(block=200), UNSUPPORTED), (dict(blocks=1 << 23), UNSUPPORTED), (dict(key=24), ALIGN),
    (dict(ks=1028), ALIGN), (dict(ks=512), BAD), (dict(v=8), ALIGN), (dict(ve=1), ALIGN), (dict(Hk=0), BAD)])
def test_store_refusals(kw, status):
    assert _store(_lib(), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(n=0), 0), (dict(B=0), 0), (dict(n=-1), BAD), (dict(cu=None), BAD), (dict(bt=None), BAD),
    (dict(ko=None), BAD), (dict(kos=1000), BAD), (dict(vos=1025), ALIGN), (dict(vo=8), ALIGN),
    (dict(block=24), UNSUPPORTED), (dict(D=256), UNSUPPORTED)])
def test_load_refusals(kw, status):
    assert _load(_lib(), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(B=0), 0), (dict(B=-1), BAD), (dict(Hq=30), BAD), (dict(Hq=136), UNSUPPORTED), (dict(D=64), UNSUPPORTED),
    (dict(block=8), UNSUPPORTED), (dict(B=8193), UNSUPPORTED), (dict(q=None), BAD), (dict(cl=None), BAD),
    (dict(bt=None), BAD), (dict(scale=0.0), BAD), (dict(scale=math.inf), BAD), (dict(scale=math.nan), BAD),
    (dict(q=24), ALIGN), (dict(qh=132), ALIGN), (dict(os=4100), ALIGN), (dict(os=2048), BAD),
    (dict(qh=64), BAD), (dict(wsb=0), WORKSPACE), (dict(ws=None), WORKSPACE), (dict(ws=24), ALIGN)])
def test_decode_refusals(kw, status):
    assert _decode(_lib(), **kw) == status


def _regions(*rows):
    return (ctypes.c_int64 * (6 * len(rows)))(*[x for r in rows for x in r])


GOOD = (P, 2, 10 * 4096, 4096, 4096, 256)


@pytest.mark.parametrize("region,status", [
    ((0, 2, 40960, 4096, 4096, 256), BAD), ((P, -1, 40960, 4096, 4096, 256), BAD),
    ((P, 2, 100, 4096, 4096, 256), BAD), ((P, 2, 40960, 4096, 1000, 256), BAD),
    ((P, 2, 40960, 4096, 4096, 0), BAD), ((P, 2, 40960, 0, 4096, 256), BAD),
    ((P, 2, 40960, 4096, 2048, 256), BAD), ((8, 2, 40960, 4096, 4096, 256), ALIGN),
    ((P, 2, 40968, 4096, 4096, 256), ALIGN)])
def test_page_region_refusals(region, status):
    lib = _lib()
    r = _regions(GOOD, region)
    assert lib.nkv_fork_pages(r, 2, 10, 16, P, 4, 4, P, P, P, P, 1, P, P, 1 << 20, None) == status


def test_page_call_refusals():
    lib = _lib()
    r = _regions(GOOD)
    assert lib.nkv_copy_pages(r, 1, 10, P, P, 0, P, 1 << 20, None) == 0
    assert lib.nkv_copy_pages(r, 1, 10, None, P, 1, P, 1 << 20, None) == BAD
    assert lib.nkv_copy_pages(r, 1, 10, P, P, -1, P, 1 << 20, None) == BAD
    assert lib.nkv_copy_pages(r, 1, 10, P, P, 1, P, 8, None) == WORKSPACE
    assert lib.nkv_copy_pages(r, 1, 10, P, P, 1, 24, 1 << 20, None) == ALIGN
    assert lib.nkv_copy_pages(r, 257, 10, P, P, 1, P, 1 << 20, None) == UNSUPPORTED
    assert lib.nkv_copy_pages(None, 1, 10, P, P, 1, P, 1 << 20, None) == BAD
    fork = (P, 4, 4, P, P, P, P, 1, P, P, 1 << 20, None)
    assert lib.nkv_fork_pages(r, 1, 10, 0, *fork) == BAD
    assert lib.nkv_fork_pages(r, 1, 10, 16, None, *fork[1:]) == BAD
    assert lib.nkv_fork_pages(r, 1, 10, 16, P, 4, 1 << 30, *fork[3:]) == UNSUPPORTED
    assert lib.nkv_fork_pages(r, 1, 10, 16, *fork[:9], None, 1 << 20, None) == WORKSPACE
    assert lib.nkv_fork_pages(r, 1, 10, 16, *fork[:7], 4097, *fork[8:]) == UNSUPPORTED
    assert lib.nkv_free_pages(P, 4, 4, P, P, 10, 16, P, 0, 0, None) == 0
    assert lib.nkv_free_pages(P, 4, 4, P, None, 10, 16, P, 1, 0, None) == BAD
    assert lib.nkv_free_pages(P, 4, 4, P, P, 10, 0, P, 1, 0, None) == BAD
    assert lib.nkv_compact_pages(r, 1, 10, P, P, 4, P, P, None, P, 1 << 20, None) == BAD
    assert lib.nkv_compact_pages(r, 1, 10, None, P, 4, P, P, P, P, 1 << 20, None) == BAD
    assert lib.nkv_compact_pages(r, 1, 10, P, P, 4, P, P, P, P, 16, None) == WORKSPACE
    assert lib.nkv_compact_pages(r, 1, 0, P, P, 4, P, P, P, P, 1 << 20, None) == BAD
    assert lib.nkv_pages_workspace_size(-1, 0) == 0


def test_wrappers_reject_host_tensors():
    from nanokv_b200 import ops

    f = torch.float8_e4m3fn
    k = torch.zeros(2, 16, 1, 128, dtype=torch.uint8).view(f)
    e = torch.zeros(2, 1, 16, dtype=torch.uint8)
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    calls = [lambda: ops.store_kvcache_fp8(x, x, k, k, e, e, i),
             lambda: ops.load_kvcache_fp8(k, k, e, e, i.view(1, 1), torch.zeros(2, dtype=torch.int32), 1),
             lambda: ops.paged_decode_fp8(x, k, k, e, e, i.view(1, 1), i, 1.0),
             lambda: ops.copy_pages([k], i, i),
             lambda: ops.fork_pages([k], i.view(1, 1), i, i, i, i, 16),
             lambda: ops.free_pages(i.view(1, 1), i, i, i, 16),
             lambda: ops.compact_pages([k], i.view(1, 1), i)]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA tensors required"):
            call()


def test_oracle_rows_against_torch():
    """The oracle's codes are torch's e4m3 conversion of the scaled row, its values torch's."""
    x = torch.from_numpy(np.random.default_rng(1).standard_normal((50, 3, 128)) * 30).to(torch.bfloat16)
    x[0] = 0
    codes, exps = quantise_ref(x)
    k = exps.double() - 127
    back = dequantise_ref(codes, exps)
    want = (x.double() * 2.0 ** -k.unsqueeze(-1)).float().clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(want.view(torch.uint8) & 0x7F, codes & 0x7F)
    assert torch.equal(back, want.double() * 2.0 ** k.unsqueeze(-1))
    assert torch.equal(torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().nan_to_num(7.0),
                       E4M3.nan_to_num(7.0))
    # half a step of 3 fraction bits, 2^-4 of the value, or of the smallest normal number of the row
    floor = torch.exp2(k - 6).unsqueeze(-1)
    assert bool(((back - x.double()).abs() <= 2.0 ** -4 * torch.maximum(x.double().abs(), floor)).all())
    assert [row_exponent(a) for a in (0.0, 448.0, 449.0, 1.75, 1.76, 3e38)] == [-117, 0, 1, -8, -7, 119]
