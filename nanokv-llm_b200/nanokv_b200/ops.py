"""Torch-facing wrappers of the libnkv C ABI (include/nkv.h).

Every function here validates its tensors the way the reference does (the
same asserts as nanokvllm/layers/attention.py:33-40 for the store), passes raw
device pointers and the caller's current CUDA stream to the library, and
raises on a non-zero status. There is no CPU or Triton fallback: CPU tensors
are rejected.
"""

from __future__ import annotations

import math
import threading
from array import array
from functools import lru_cache

import torch

from . import _lib
from .utils.context import note_page_call

__all__ = [
    "store_kvcache",
    "flash_decode_with_kvcache",
    "paged_decode",
    "decode_step",
    "decode_workspace",
    "paged_prefill",
    "qk_norm_rope_store",
    "flash_attn_varlen_func",
    "window_compress",
    "window_select",
    "query_window_append",
    "threshold_compress",
    "store_kvcache_fp8",
    "load_kvcache_fp8",
    "paged_decode_fp8",
    "copy_pages",
    "fork_pages",
    "free_pages",
    "unshared_rows",
    "compact_pages",
]


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(name: str, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError(f"{name}: CUDA tensors required (libnkv has no CPU path)")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------- store
def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Writes key/value rows into their cache slots (slot == -1 is skipped).

    Same contract and asserts as the reference's store_kvcache
    (nanokvllm/layers/attention.py:33-40).
    """
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    assert slot_mapping.numel() == N
    if N == 0 or k_cache.numel() == 0:
        return
    _require_cuda("store_kvcache", key, value, k_cache, v_cache, slot_mapping)
    assert key.dtype == torch.bfloat16 and k_cache.dtype == torch.bfloat16
    assert slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous()
    num_slots = k_cache.numel() // D
    lib = _lib.load()
    _lib.check("nkv_store_kvcache", lib.nkv_store_kvcache(
        key.data_ptr(), key.stride(0), value.data_ptr(), value.stride(0),
        k_cache.data_ptr(), v_cache.data_ptr(), num_slots,
        slot_mapping.data_ptr(), N, num_heads, head_dim, _stream(key.device)))


# ---------------------------------------------------------------- decode
class _WorkspacePool:
    """One zero-initialised decode workspace per device, grown on demand.

    The decode kernel leaves its workspace zeroed after every call, so a
    single buffer serves every layer, step and captured graph. Call
    `decode_workspace(...)` with the largest shape before capturing a graph so
    the capture never allocates.
    """

    def __init__(self):
        self._bufs: dict[int, torch.Tensor] = {}
        self._lock = threading.Lock()

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor:
        idx = device.index if device.index is not None else torch.cuda.current_device()
        with self._lock:
            buf = self._bufs.get(idx)
            if buf is None or buf.numel() < nbytes:
                buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=torch.device("cuda", idx))
                self._bufs[idx] = buf
            return buf


_WS = _WorkspacePool()


def decode_workspace_bytes(batch: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                           max_blocks: int, block_size: int) -> int:
    return int(_lib.load().nkv_paged_decode_workspace_size(
        batch, num_q_heads, num_kv_heads, head_dim, max_blocks, block_size))


def decode_workspace(device: torch.device, batch: int, num_q_heads: int, num_kv_heads: int,
                     head_dim: int, max_blocks: int, block_size: int) -> torch.Tensor:
    nbytes = decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_blocks, block_size)
    return _WS.get(device, nbytes)


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_tables: torch.Tensor, context_lens: torch.Tensor, softmax_scale: float,
                 out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention for one query token per sequence over the paged cache.

    q: [B, Hq, D] bf16 (row stride free, head stride multiple of 8);
    k_cache/v_cache: [num_blocks, block_size, Hk, D]; block_tables [B, max_blocks]
    int32; context_lens [B] int32. Returns out [B, Hq, D] bf16.
    """
    _require_cuda("paged_decode", q, k_cache, v_cache, block_tables, context_lens)
    B, Hq, D = q.shape
    num_blocks, block_size, Hk, Dk = k_cache.shape
    assert Dk == D and v_cache.shape == k_cache.shape
    assert q.dtype == torch.bfloat16 and k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16
    assert q.stride(-1) == 1
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert block_tables.dtype == torch.int32 and context_lens.dtype == torch.int32
    assert block_tables.dim() == 2 and block_tables.size(0) >= B and block_tables.stride(1) == 1
    assert context_lens.numel() >= B and context_lens.is_contiguous()
    max_blocks = block_tables.size(1)
    if block_tables.stride(0) != max_blocks:
        block_tables = block_tables.contiguous()
    if out is None:
        out = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=q.device)
    assert out.stride(-1) == 1 and out.stride(1) == D
    if B == 0:
        return out
    if workspace is None:
        workspace = decode_workspace(q.device, B, Hq, Hk, D, max_blocks, block_size)
    lib = _lib.load()
    _lib.check("nkv_paged_decode", lib.nkv_paged_decode(
        q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), num_blocks,
        block_tables.data_ptr(), max_blocks, context_lens.data_ptr(), out.data_ptr(), out.stride(0),
        B, Hq, Hk, D, block_size, float(softmax_scale), workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), _stream(q.device)))
    return out


def decode_step(q: torch.Tensor, key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                v_cache: torch.Tensor, slot_mapping: torch.Tensor, block_tables: torch.Tensor,
                context_lens: torch.Tensor, softmax_scale: float, out: torch.Tensor | None = None,
                ring: torch.Tensor | None = None, layer_id: int = 0,
                ring_slot_of_row: torch.Tensor | None = None,
                ring_pos_of_row: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None,
                metadata_ready: bool = False) -> torch.Tensor:
    """One fused launch of store_kvcache(key, value, slot_mapping) [+ the
    KvChat query-window append] + paged_decode for a decode step (one new
    token per row, slot_mapping[b] = -1 or the slot of position
    context_lens[b] - 1).

    metadata_ready: the caller vouches that the kernel launched just before
    this call on the stream does not write block_tables, context_lens,
    slot_mapping or the ring indices (host copies and earlier kernels are
    fine), so the launch may read them before it waits for that kernel --
    true of a decode step's layers, whose metadata the engine copies from
    the host; not of a decode right after a compression kernel or a page
    operator (copy_pages, fork_pages, free_pages, compact_pages)."""
    _require_cuda("decode_step", q, key, value, k_cache, v_cache, slot_mapping, block_tables,
                  context_lens)
    B, Hq, D = q.shape
    num_blocks, block_size, Hk, Dk = k_cache.shape
    assert Dk == D and v_cache.shape == k_cache.shape
    assert key.shape == (B, Hk, D) and value.shape == (B, Hk, D)
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == D and value.stride(1) == D
    assert k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16
    assert q.stride(-1) == 1 and k_cache.is_contiguous() and v_cache.is_contiguous()
    assert slot_mapping.dtype == torch.int32 and slot_mapping.numel() == B
    assert block_tables.dtype == torch.int32 and context_lens.dtype == torch.int32
    max_blocks = block_tables.size(1)
    if block_tables.stride(0) != max_blocks:
        block_tables = block_tables.contiguous()
        metadata_ready = False  # the copy kernel just wrote it
    if out is None:
        out = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=q.device)
    if B == 0:
        return out
    if workspace is None:
        workspace = decode_workspace(q.device, B, Hq, Hk, D, max_blocks, block_size)
    if ring is not None:
        slots, layers, W, Hr, Dr = ring.shape
        assert Hr == Hq and Dr == D and ring.is_contiguous()
        ring_args = (ring.data_ptr(), slots, layers, W, layer_id, ring_slot_of_row.data_ptr(),
                     ring_pos_of_row.data_ptr())
    else:
        ring_args = (None, 0, 0, 0, 0, None, None)
    lib = _lib.load()
    _lib.check("nkv_decode_step", lib.nkv_decode_step(
        q.data_ptr(), q.stride(0), q.stride(1), key.data_ptr(), key.stride(0), value.data_ptr(),
        value.stride(0), slot_mapping.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        num_blocks, block_tables.data_ptr(), max_blocks, context_lens.data_ptr(), *ring_args,
        out.data_ptr(), out.stride(0), B, Hq, Hk, D, block_size, float(softmax_scale),
        1 if metadata_ready else 0,
        workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(q.device)))
    return out


def flash_decode_with_kvcache(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                              cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                              softmax_scale: float | None = None, causal: bool = True,
                              out: torch.Tensor | None = None) -> torch.Tensor:
    """Drop-in for the reference's flash_attn_with_kvcache decode call
    (nanokvllm/layers/attention.py:104-107): q is [B, 1, Hq, D], the result
    is [B, 1, Hq, D]. With one query token `causal` changes nothing."""
    assert q.dim() == 4 and q.size(1) == 1, "decode path: exactly one query token per sequence"
    if softmax_scale is None:
        softmax_scale = q.size(-1) ** -0.5
    o = paged_decode(q[:, 0], k_cache, v_cache, block_table, cache_seqlens, softmax_scale,
                     out=None if out is None else out[:, 0])
    return o.unsqueeze(1)


# ---------------------------------------------------------------- q/k norm + RoPE + store
def qk_norm_rope_store(qkv: torch.Tensor, positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                       q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, eps: float,
                       num_q_heads: int, num_kv_heads: int, k_cache: torch.Tensor | None = None,
                       v_cache: torch.Tensor | None = None,
                       slot_mapping: torch.Tensor | None = None,
                       q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """q_norm / k_norm + rotary_emb + store_kvcache of one layer in one launch
    (nkv_qk_norm_rope_store; the sequence at nanokvllm/models/qwen3.py:109-113
    and nanokvllm/layers/attention.py:72-73).

    qkv: [T, (Hq + 2 Hk) * 128] bf16 (the qkv projection output);
    positions: [T] int64; cos_sin_cache: the RotaryEmbedding module's fp32
    buffer ([max_pos, 1, 128] or [max_pos, 128]); norm weights [128] bf16.
    Returns (q [T, Hq, 128], v view [T, Hk, 128], k_out or None); k and v
    are written to the cache slots when k_cache is given.
    """
    _require_cuda("qk_norm_rope_store", qkv, positions, cos_sin_cache, q_norm_weight,
                  k_norm_weight, k_cache, v_cache, slot_mapping)
    T = qkv.size(0)
    D = 128
    assert qkv.dtype == torch.bfloat16 and qkv.stride(-1) == 1
    assert qkv.size(-1) == (num_q_heads + 2 * num_kv_heads) * D
    assert positions.dtype == torch.int64 and positions.is_contiguous() and positions.numel() == T
    cs = cos_sin_cache.reshape(-1, D)
    assert cs.dtype == torch.float32 and cs.is_contiguous()
    assert q_norm_weight.dtype == torch.bfloat16 and k_norm_weight.dtype == torch.bfloat16
    assert q_norm_weight.is_contiguous() and k_norm_weight.is_contiguous()
    if q_out is None:
        q_out = torch.empty(T, num_q_heads, D, dtype=torch.bfloat16, device=qkv.device)
    assert q_out.stride(-1) == 1 and q_out.stride(1) == D
    if k_out is not None:
        assert k_out.stride(-1) == 1 and k_out.stride(1) == D
    num_slots = 0
    if k_cache is not None:
        assert v_cache is not None and slot_mapping is not None
        assert k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16
        assert k_cache.is_contiguous() and v_cache.is_contiguous() and v_cache.shape == k_cache.shape
        assert slot_mapping.dtype == torch.int32 and slot_mapping.numel() == T
        num_slots = k_cache.numel() // (num_kv_heads * D)
    v = qkv[:, (num_q_heads + num_kv_heads) * D:].view(T, num_kv_heads, D)
    if T == 0:
        return q_out, v, k_out
    lib = _lib.load()
    _lib.check("nkv_qk_norm_rope_store", lib.nkv_qk_norm_rope_store(
        qkv.data_ptr(), qkv.stride(0), T, positions.data_ptr(), cs.data_ptr(), cs.size(0),
        q_norm_weight.data_ptr(), k_norm_weight.data_ptr(), float(eps), q_out.data_ptr(),
        q_out.stride(0), _ptr(k_out), 0 if k_out is None else k_out.stride(0), _ptr(k_cache),
        _ptr(v_cache), num_slots, _ptr(slot_mapping), num_q_heads, num_kv_heads, D,
        _stream(qkv.device)))
    return q_out, v, k_out


# ---------------------------------------------------------------- prefill
def paged_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                  cu_seqlens_k: torch.Tensor, max_seqlen_q: int, softmax_scale: float,
                  causal: bool = True, block_table: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Variable-length attention of a prefill / mixed batch (nkv_paged_prefill).

    q: [T, Hq, D] bf16. With block_table ([B, max_blocks] int32) k / v are the
    paged caches [num_blocks, block_size, Hk, D]; without it they are the
    step's rows [Tk, Hk, D] addressed through cu_seqlens_k. cu_seqlens_* are
    int32 [B + 1] device tensors; causal masks bottom-right aligned.
    Returns out [T, Hq, D] bf16.
    """
    _require_cuda("paged_prefill", q, k, v, cu_seqlens_q, cu_seqlens_k, block_table)
    T, Hq, D = q.shape
    assert q.dtype == torch.bfloat16 and k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16
    assert q.stride(-1) == 1 and k.stride(-1) == 1 and v.stride(-1) == 1
    assert cu_seqlens_q.dtype == torch.int32 and cu_seqlens_k.dtype == torch.int32
    assert cu_seqlens_q.is_contiguous() and cu_seqlens_k.is_contiguous()
    B = cu_seqlens_q.numel() - 1
    assert cu_seqlens_k.numel() == B + 1
    if block_table is not None:
        num_blocks, block_size, Hk, Dk = k.shape
        assert k.is_contiguous() and v.is_contiguous() and v.shape == k.shape
        assert block_table.dtype == torch.int32 and block_table.dim() == 2
        assert block_table.size(0) >= B
        if not block_table.is_contiguous():
            block_table = block_table.contiguous()
        rows, k_stride, v_stride = num_blocks * block_size, Hk * D, Hk * D
        max_blocks = block_table.size(1)
        bt_ptr = block_table.data_ptr()
    else:
        rows, Hk, Dk = k.shape
        assert v.shape == k.shape and k.stride(1) == D and v.stride(1) == D
        k_stride, v_stride = k.stride(0), v.stride(0)
        block_size = max_blocks = 0
        bt_ptr = None
    assert Dk == D
    if out is None:
        out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=q.device)
    assert out.stride(-1) == 1 and out.stride(1) == D and out.size(0) >= T
    if B <= 0 or T == 0 or max_seqlen_q <= 0:
        return out
    lib = _lib.load()
    _lib.check("nkv_paged_prefill", lib.nkv_paged_prefill(
        q.data_ptr(), q.stride(0), q.stride(1), T, k.data_ptr(), k_stride, v.data_ptr(), v_stride,
        rows, bt_ptr, max_blocks, block_size, cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), B,
        int(max_seqlen_q), 1 if causal else 0, out.data_ptr(), out.stride(0), Hq, Hk, D,
        float(softmax_scale), _stream(q.device)))
    return out


def flash_attn_varlen_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                           max_seqlen_q: int, max_seqlen_k: int,
                           softmax_scale: float | None = None, causal: bool = False,
                           block_table: torch.Tensor | None = None) -> torch.Tensor:
    """Drop-in for the reference's prefill / mixed-batch call of
    flash_attn_varlen_func (nanokvllm/layers/attention.py:96-102), with the
    keyword names and defaults of flash-attn's function. max_seqlen_k is
    accepted for the signature; the kernel reads each length from cu_seqlens_k.
    """
    del max_seqlen_k
    if softmax_scale is None:
        softmax_scale = q.size(-1) ** -0.5
    return paged_prefill(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, softmax_scale,
                         causal=causal, block_table=block_table)


def window_select(context_lens: torch.Tensor, tail_uncompressed: torch.Tensor, block_size: int,
                  window_blocks: int, topk: int, out_selected: torch.Tensor | None = None,
                  out_count: torch.Tensor | None = None,
                  out_base_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Device-side periodic-compression selection (nkv_window_select): the
    first `topk` eligible rows by the reference's rule (model_runner.py:
    305-321) into out_selected[topk], -1 padded. All tensors int32 on the
    device; nothing is read back, so the call can sit inside a CUDA graph."""
    _require_cuda("window_select", context_lens, tail_uncompressed, out_selected, out_count,
                  out_base_lens)
    B = context_lens.numel()
    assert context_lens.dtype == torch.int32 and tail_uncompressed.dtype == torch.int32
    assert context_lens.is_contiguous() and tail_uncompressed.is_contiguous()
    assert tail_uncompressed.numel() >= B
    if out_selected is None:
        out_selected = torch.empty(topk, dtype=torch.int32, device=context_lens.device)
    assert out_selected.dtype == torch.int32 and out_selected.numel() >= topk
    lib = _lib.load()
    _lib.check("nkv_window_select", lib.nkv_window_select(
        context_lens.data_ptr(), tail_uncompressed.data_ptr(), B, block_size, window_blocks, topk,
        out_selected.data_ptr(), _ptr(out_count), _ptr(out_base_lens), _stream(context_lens.device)))
    return out_selected


# ---------------------------------------------------------------- window compression
def window_compress(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_tables: torch.Tensor, base_context_lens: torch.Tensor,
                    context_lens: torch.Tensor, selected: torch.Tensor, window_blocks: int,
                    keep_tokens: int, obs_window: int = 1, softmax_scale: float | None = None,
                    out_keep_idx: torch.Tensor | None = None,
                    out_new_lens: torch.Tensor | None = None,
                    out_importance: torch.Tensor | None = None) -> None:
    """Periodic window compression of one layer (SnapKV scoring + compaction).

    `selected` is an int32 device tensor of batch indices; context_lens is
    updated in place. softmax_scale defaults to SnapKV's 1/sqrt(head_dim).
    out_importance (bf16 [m, window_blocks * block_size - obs_window]), if
    given, receives the importance SnapKV ranked.
    """
    _require_cuda("window_compress", q, k_cache, v_cache, block_tables, base_context_lens,
                  context_lens, selected)
    m = selected.numel()
    if m == 0:
        return
    num_blocks, block_size, Hk, D = k_cache.shape
    assert k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16
    Hq = q.size(1)
    assert q.stride(-1) == 1 and q.stride(1) == D
    assert selected.dtype == torch.int32 and selected.is_contiguous()
    assert block_tables.dtype == torch.int32 and block_tables.is_contiguous()
    assert base_context_lens.dtype == torch.int32 and context_lens.dtype == torch.int32
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    if out_importance is not None:
        assert out_importance.dtype == torch.bfloat16 and out_importance.is_contiguous()
        assert out_importance.shape == (m, window_blocks * block_size - obs_window)
    lib = _lib.load()
    _lib.check("nkv_window_compress", lib.nkv_window_compress(
        q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), num_blocks,
        block_tables.data_ptr(), block_tables.size(1), base_context_lens.data_ptr(),
        context_lens.data_ptr(), selected.data_ptr(), m, window_blocks, keep_tokens, obs_window,
        Hq, Hk, D, block_size, float(softmax_scale), _ptr(out_keep_idx), _ptr(out_new_lens),
        _ptr(out_importance), _stream(q.device)))


# ---------------------------------------------------------------- KvChat threshold path
def query_window_append(q: torch.Tensor, ring: torch.Tensor, layer_id: int,
                        batch_index: torch.Tensor, ring_slot: torch.Tensor,
                        ring_pos: torch.Tensor) -> None:
    """ring[ring_slot[j], layer_id, ring_pos[j]] = q[batch_index[j]] for every j."""
    _require_cuda("query_window_append", q, ring, batch_index, ring_slot, ring_pos)
    n = batch_index.numel()
    if n == 0:
        return
    slots, layers, W, Hq, D = ring.shape
    assert q.size(1) == Hq and q.size(2) == D and q.stride(-1) == 1 and q.stride(1) == D
    assert ring.is_contiguous()
    lib = _lib.load()
    _lib.check("nkv_query_window_append", lib.nkv_query_window_append(
        q.data_ptr(), q.stride(0), ring.data_ptr(), slots, layers, W, layer_id,
        batch_index.data_ptr(), ring_slot.data_ptr(), ring_pos.data_ptr(), n, Hq, D,
        _stream(q.device)))


def threshold_compress(ring: torch.Tensor, ring_slot_of_selected: torch.Tensor, layer_id: int,
                       k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                       context_lens: torch.Tensor, selected: torch.Tensor, S: int, R: int,
                       softmax_scale: float | None = None,
                       out_keep_idx: torch.Tensor | None = None,
                       out_importance: torch.Tensor | None = None) -> None:
    """KvChat threshold compression S -> R of one layer; context_lens[sel] = R.
    out_importance (bf16 [m, S - W]), if given, receives the importance
    SnapKV ranked."""
    _require_cuda("threshold_compress", ring, ring_slot_of_selected, k_cache, v_cache,
                  block_tables, context_lens, selected)
    m = selected.numel()
    if m == 0:
        return
    slots, layers, W, Hq, D = ring.shape
    num_blocks, block_size, Hk, Dk = k_cache.shape
    assert Dk == D and ring.is_contiguous() and block_tables.is_contiguous()
    assert k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    if out_importance is not None:
        assert out_importance.dtype == torch.bfloat16 and out_importance.is_contiguous()
        assert out_importance.shape == (m, S - W)
    lib = _lib.load()
    _lib.check("nkv_threshold_compress", lib.nkv_threshold_compress(
        ring.data_ptr(), slots, layers, W, layer_id, ring_slot_of_selected.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), num_blocks, block_tables.data_ptr(),
        block_tables.size(1), context_lens.data_ptr(), selected.data_ptr(), m, S, R, Hq, Hk, D,
        block_size, float(softmax_scale), _ptr(out_keep_idx), _ptr(out_importance),
        _stream(k_cache.device)))


# ---------------------------------------------------------------- 8-bit cache
# These calls are short, so their host side counts: one pass over the arguments,
# strides and shapes read once, the raw stream of the device.
def _one_device(name: str, *tensors: torch.Tensor | None) -> int:
    """The index of the CUDA device all tensors are on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name}: all tensors must be on one CUDA device")
    if index < 0:
        raise ValueError(f"{name}: CUDA tensors required (libnkv has no CPU path)")
    return index


def _call(device: int, name: str, *args) -> None:
    """Entry point `name` on the device's current stream, with that device current."""
    fn = getattr(_lib.load(), name)
    stream = torch._C._cuda_getCurrentRawStream(device)
    if device == torch._C._cuda_getDevice():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, stream)
    if status:
        _lib.check(name, status)


def _check_cache8(k_cache, v_cache, k_exp, v_exp) -> torch.Size:
    """(num_blocks, block_size, Hk, D) of an 8-bit cache."""
    shape = k_cache.shape
    num_blocks, block_size, Hk, _ = shape
    exp_shape = k_exp.shape
    assert v_cache.shape == shape and v_exp.shape == exp_shape
    assert exp_shape == (num_blocks, Hk, block_size)
    assert k_cache.dtype is _E4M3 and v_cache.dtype is _E4M3
    assert k_exp.dtype is torch.uint8 and v_exp.dtype is torch.uint8
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert k_exp.is_contiguous() and v_exp.is_contiguous()
    return shape


_E4M3 = torch.float8_e4m3fn
_BF16 = torch.bfloat16
_INT32 = torch.int32


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, k_exp: torch.Tensor, v_exp: torch.Tensor,
                      slot_mapping: torch.Tensor) -> None:
    """Writes key / value rows into the slots of an 8-bit cache (slot == -1 is
    skipped): e4m3 values with a power-of-two scale per (token, kv head) row.

    key / value: [N, Hk, 128] bf16, heads contiguous, row stride free (the
    slices of a qkv projection's output); k_cache / v_cache:
    [num_blocks, block_size, Hk, 128] float8_e4m3fn; k_exp / v_exp:
    [num_blocks, Hk, block_size] uint8, a row reads as
    e4m3 * 2^(exp - 127); slot_mapping: [N] int32.
    """
    device = _one_device("store_kvcache_fp8", key, value, k_cache, v_cache, k_exp, v_exp,
                         slot_mapping)
    num_blocks, block_size, Hk, D = _check_cache8(k_cache, v_cache, k_exp, v_exp)
    shape = key.shape
    N = shape[0]
    k_stride, v_stride = key.stride(), value.stride()
    assert shape == (N, Hk, D) and value.shape == shape
    assert key.dtype is _BF16 and value.dtype is _BF16
    assert k_stride[1:] == (D, 1) and v_stride[1:] == (D, 1)
    assert slot_mapping.dtype is _INT32 and slot_mapping.is_contiguous()
    assert slot_mapping.numel() == N
    if N == 0 or num_blocks == 0:
        return
    _call(device, "nkv_store_kvcache_fp8", key.data_ptr(), k_stride[0], value.data_ptr(),
          v_stride[0], k_cache.data_ptr(), v_cache.data_ptr(), k_exp.data_ptr(),
          v_exp.data_ptr(), num_blocks, block_size, slot_mapping.data_ptr(), N, Hk, D)


def load_kvcache_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_exp: torch.Tensor,
                     v_exp: torch.Tensor, block_tables: torch.Tensor, cu_seqlens: torch.Tensor,
                     num_tokens: int, k_out: torch.Tensor | None = None,
                     v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Whole sequences of an 8-bit cache as packed bf16 rows (exact), the k / v
    that paged_prefill takes without a block table.

    block_tables: [B, max_blocks] int32; cu_seqlens: [B + 1] int32 on the
    device; num_tokens: rows of the outputs, at least cu_seqlens[-1] (rows
    behind the last sequence are left as they are). Returns (k, v)
    [num_tokens, Hk, 128] bf16.
    """
    device = _one_device("load_kvcache_fp8", k_cache, v_cache, k_exp, v_exp, block_tables,
                         cu_seqlens, k_out, v_out)
    num_blocks, block_size, Hk, D = _check_cache8(k_cache, v_cache, k_exp, v_exp)
    B = cu_seqlens.numel() - 1
    assert cu_seqlens.dtype is _INT32 and cu_seqlens.is_contiguous() and B >= 0
    rows, max_blocks = block_tables.shape
    assert block_tables.dtype is _INT32 and rows >= B and num_tokens >= 0
    if not block_tables.is_contiguous():
        block_tables = block_tables.contiguous()
    if k_out is None:
        k_out = k_cache.new_empty((num_tokens, Hk, D), dtype=_BF16)
    if v_out is None:
        v_out = torch.empty_like(k_out, memory_format=torch.contiguous_format)
    k_stride, v_stride = k_out.stride(), v_out.stride()
    assert k_out.shape == (num_tokens, Hk, D) and v_out.shape == (num_tokens, Hk, D)
    assert k_out.dtype is _BF16 and v_out.dtype is _BF16
    if B == 0 or num_tokens == 0:
        return k_out, v_out
    assert k_stride[1:] == (D, 1) and v_stride[1:] == (D, 1)
    _call(device, "nkv_load_kvcache_fp8", k_cache.data_ptr(), v_cache.data_ptr(),
          k_exp.data_ptr(), v_exp.data_ptr(), num_blocks, block_size, block_tables.data_ptr(),
          max_blocks, cu_seqlens.data_ptr(), B, num_tokens, k_out.data_ptr(),
          k_stride[0], v_out.data_ptr(), v_stride[0], Hk, D)
    return k_out, v_out


def paged_decode_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     k_exp: torch.Tensor, v_exp: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, softmax_scale: float,
                     out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """paged_decode over an 8-bit cache: attention of one query token per
    sequence, split over the cached length and joined.

    q: [B, Hq, 128] bf16 (row and head strides multiples of 8); the cache as
    store_kvcache_fp8 writes it; block_tables [B, max_blocks] int32;
    context_lens [B] int32 (0 gives zeros; tokens whose table entry is no page
    count as zero keys and values, DEVERR_DECODE_BLOCK is set). workspace (uint8, at least
    decode_fp8_workspace_bytes) may hold anything; by default every call takes
    its own from torch's allocator, so calls on several streams and captured
    graphs share none. Returns out [B, Hq, 128] bf16.
    """
    device = _one_device("paged_decode_fp8", q, k_cache, v_cache, k_exp, v_exp, block_tables,
                         context_lens, out, workspace)
    q_shape, q_stride = q.shape, q.stride()
    B, Hq, D = q_shape
    num_blocks, block_size, Hk, Dk = _check_cache8(k_cache, v_cache, k_exp, v_exp)
    rows, max_blocks = block_tables.shape
    assert Dk == D and Hk > 0 and Hq % Hk == 0
    assert q.dtype is _BF16 and q_stride[2] == 1
    assert block_tables.dtype is _INT32 and context_lens.dtype is _INT32 and rows >= B
    assert context_lens.numel() >= B and context_lens.is_contiguous()
    if not block_tables.is_contiguous():
        block_tables = block_tables.contiguous()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_stride = Hq * D
    else:
        assert out.shape == q_shape and out.dtype is _BF16
        out_stride, *inner = out.stride()
        assert B == 0 or inner == [D, 1]
    if B == 0:
        return out
    if workspace is None:
        workspace = k_exp.new_empty(decode_fp8_workspace_bytes(Hq, Hk))
    assert workspace.is_contiguous()
    _call(device, "nkv_paged_decode_fp8", q.data_ptr(), q_stride[0], q_stride[1],
          k_cache.data_ptr(), v_cache.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), num_blocks,
          block_tables.data_ptr(), max_blocks, context_lens.data_ptr(), out.data_ptr(),
          out_stride, B, Hq, Hk, D, block_size, softmax_scale, workspace.data_ptr(),
          workspace.numel() * workspace.element_size())
    return out


@lru_cache(maxsize=None)
def decode_fp8_workspace_bytes(num_q_heads: int, num_kv_heads: int) -> int:
    return int(_lib.load().nkv_paged_decode_fp8_workspace_size(num_q_heads, num_kv_heads))


# ---------------------------------------------------------------- pages
def _page_regions(caches, page_dim: int, num_pages: int | None,
                  block_size: int | None) -> tuple[array | None, int | None, int, int | None]:
    """The caches as nkv_page_region records: (the records, their address, how
    many, num_pages).

    Each cache is contiguous, [*lead, num_pages, *page] with page_dim leading
    dims; with a block size a page is [block_size, Hk, D] (values) or
    [Hk, block_size] (exponent bytes)."""
    records = array("q")
    for c in caches:
        shape = c.shape
        assert c.is_contiguous() and 0 <= page_dim < len(shape)
        if num_pages is None:
            num_pages = shape[page_dim]
        assert shape[page_dim] == num_pages, "the caches differ in their number of pages"
        size = c.element_size()
        page = shape[page_dim + 1:]
        page_bytes = math.prod(page) * size
        if block_size is None:
            seg_bytes = token_bytes = page_bytes
        elif len(page) == 3:
            assert page[0] == block_size
            token_bytes = page[1] * page[2] * size
            seg_bytes = page_bytes
        else:
            assert len(page) == 2 and page[1] == block_size
            token_bytes = size
            seg_bytes = block_size * size
        records.extend((c.data_ptr(), math.prod(shape[:page_dim]), num_pages * page_bytes,
                        page_bytes, seg_bytes, token_bytes))
    if not caches:
        return None, None, 0, num_pages
    return records, records.buffer_info()[0], len(caches), num_pages


def _check_page_state(block_tables, *others) -> tuple[int, int]:
    """(rows, max_blocks) of a block table; every tensor int32 and contiguous."""
    rows, max_blocks = block_tables.shape
    assert block_tables.dtype is _INT32 and block_tables.is_contiguous()
    for t in others:
        assert t.dtype is _INT32 and t.is_contiguous()
    return rows, max_blocks


def _pages_workspace(like: torch.Tensor, n: int, num_pages: int) -> tuple[torch.Tensor, int]:
    """Scratch of one page call on the device of `like` (int32), from torch's
    allocator (stream-ordered, and a captured graph's own), and its size."""
    size = _pages_workspace_bytes(n, num_pages)
    return like.new_empty(size // 4), size


@lru_cache(maxsize=4096)
def _pages_workspace_bytes(n: int, num_pages: int) -> int:
    return int(_lib.load().nkv_pages_workspace_size(n, num_pages))


def copy_pages(caches, src: torch.Tensor, dst: torch.Tensor, page_dim: int = 0) -> None:
    """Copies page src[i] to page dst[i] in every cache tensor.

    caches: contiguous CUDA tensors [*lead, num_pages, *page] with page_dim
    leading dims (0 for one layer's view, 2 for kv_cache[2, layers, ...]);
    src / dst: int32 on the device. A page may be a source many times; a pair
    whose target is another pair's target or source, or outside the cache, is
    not copied and sets DEVERR_PAGES. Pairs (-1, -1) are padding.
    """
    device = _one_device("copy_pages", src, dst, *caches)
    n = src.numel()
    assert src.dtype is _INT32 and dst.dtype is _INT32 and dst.numel() == n
    assert src.is_contiguous() and dst.is_contiguous()
    _keep, regions, count, num_pages = _page_regions(caches, page_dim, None, None)
    if n == 0 or count == 0:
        return
    ws, size = _pages_workspace(src, n, 0)
    note_page_call()
    _call(device, "nkv_copy_pages", regions, count, num_pages, src.data_ptr(), dst.data_ptr(), n,
          ws.data_ptr(), size)


def fork_pages(caches, block_tables: torch.Tensor, context_lens: torch.Tensor,
               ref_counts: torch.Tensor, src_rows: torch.Tensor, dst_rows: torch.Tensor,
               block_size: int, page_dim: int = 0,
               out_pages: torch.Tensor | None = None) -> torch.Tensor:
    """Row dst_rows[i] becomes a copy of row src_rows[i]: full pages shared
    (ref_counts + 1), a partial last page copied -- its tokens only -- to the
    lowest free page (ref_counts <= 0); the pages dst_rows held are released
    first.

    block_tables [rows, max_blocks], context_lens [rows] and ref_counts
    [num_pages] (all int32) are updated in place; caches as copy_pages, each
    page [block_size, Hk, D] or, for exponent bytes, [Hk, block_size]. Shared
    pages are read only: do not compress a row while it shares some
    (unshared_rows). At most
    4096 forks per call. Returns out_pages int32 [n]: the page that was taken,
    -1 if none was needed, -2 if the fork was not made (a target that is named
    twice or is a source, a row out of range, no free page, a partial page that
    is none of the cache or that nobody holds: DEVERR_PAGES is set; or a
    (-1, -1) padding pair).
    """
    device = _one_device("fork_pages", block_tables, context_lens, ref_counts, src_rows, dst_rows,
                         out_pages, *caches)
    rows, max_blocks = _check_page_state(block_tables, context_lens, ref_counts, src_rows, dst_rows)
    n, num_pages = src_rows.numel(), ref_counts.numel()
    assert context_lens.numel() == rows and dst_rows.numel() == n
    _keep, regions, count, _ = _page_regions(caches, page_dim, num_pages, block_size)
    if out_pages is None:
        out_pages = src_rows.new_empty(n)
    assert out_pages.dtype is _INT32 and out_pages.is_contiguous() and out_pages.numel() == n
    if n == 0:
        return out_pages
    ws, size = _pages_workspace(src_rows, n, 0)
    note_page_call()
    _call(device, "nkv_fork_pages", regions, count, num_pages, block_size,
          block_tables.data_ptr(), max_blocks, rows, context_lens.data_ptr(),
          ref_counts.data_ptr(), src_rows.data_ptr(), dst_rows.data_ptr(), n,
          out_pages.data_ptr(), ws.data_ptr(), size)
    return out_pages


def free_pages(block_tables: torch.Tensor, context_lens: torch.Tensor, ref_counts: torch.Tensor,
               rows: torch.Tensor, block_size: int, trim: bool = False) -> None:
    """The named rows (int32 on the device, -1 is padding) give up their pages:
    ref_counts - 1, table entries -1. trim=False: all pages, and the row's
    length becomes 0; trim=True: the pages past context_lens, as after a
    compression that shortened the rows on the device."""
    device = _one_device("free_pages", block_tables, context_lens, ref_counts, rows)
    num_rows, max_blocks = _check_page_state(block_tables, context_lens, ref_counts, rows)
    n = rows.numel()
    assert context_lens.numel() == num_rows
    if n == 0:
        return
    note_page_call()
    _call(device, "nkv_free_pages", block_tables.data_ptr(), max_blocks, num_rows,
          context_lens.data_ptr(), ref_counts.data_ptr(), ref_counts.numel(), block_size,
          rows.data_ptr(), n, 1 if trim else 0)


def unshared_rows(rows: torch.Tensor, block_tables: torch.Tensor, ref_counts: torch.Tensor,
                  block_size: int, kept_tokens: int, lens: torch.Tensor | None = None,
                  window_blocks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """The named rows (int32 on the device, -1 stays) that a compression may
    rewrite in place: one that shares a page which the compression would write
    (the kept tokens' pages, from the window's first page on or, without lens,
    from the row's first) becomes -1 and sets DEVERR_PAGES."""
    device = _one_device("unshared_rows", rows, block_tables, ref_counts, lens, out)
    if out is None:
        out = torch.empty_like(rows, memory_format=torch.contiguous_format)
    num_rows, max_blocks = _check_page_state(block_tables, rows, ref_counts, out)
    n = rows.numel()
    assert out.numel() == n
    if lens is not None:
        assert lens.dtype is _INT32 and lens.is_contiguous()
        num_rows = min(num_rows, lens.numel())
    if n == 0:
        return out
    pages = min(-(-kept_tokens // block_size), max_blocks)
    _call(device, "nkv_unshared_rows", rows.data_ptr(), n, block_tables.data_ptr(), max_blocks,
          num_rows, _ptr(lens), ref_counts.data_ptr(), ref_counts.numel(), block_size,
          window_blocks, pages, out.data_ptr())
    return out


def compact_pages(caches, block_tables: torch.Tensor, ref_counts: torch.Tensor, page_dim: int = 0,
                  out_block_tables: torch.Tensor | None = None,
                  out_ref_counts: torch.Tensor | None = None,
                  out_num_live: torch.Tensor | None = None) -> torch.Tensor:
    """Brings the n pages in use (ref_counts > 0) to the first n of the cache:
    the i-th used page at or past n moves to the i-th free page before n in
    every cache tensor, and tables and counts follow (in place, or into the
    out tensors). Returns out_num_live, int32 [1]: n."""
    device = _one_device("compact_pages", block_tables, ref_counts, out_block_tables,
                         out_ref_counts, out_num_live, *caches)
    if out_block_tables is None:
        out_block_tables = block_tables
    if out_ref_counts is None:
        out_ref_counts = ref_counts
    if out_num_live is None:
        out_num_live = ref_counts.new_empty(1)
    rows, max_blocks = _check_page_state(block_tables, ref_counts, out_block_tables,
                                         out_ref_counts, out_num_live)
    num_pages = ref_counts.numel()
    assert out_block_tables.shape == (rows, max_blocks)
    assert out_ref_counts.numel() == num_pages and out_num_live.numel() == 1
    _keep, regions, count, _ = _page_regions(caches, page_dim, num_pages, None)
    ws, size = _pages_workspace(ref_counts, num_pages // 2, num_pages)
    note_page_call()
    _call(device, "nkv_compact_pages", regions, count, num_pages, block_tables.data_ptr(),
          out_block_tables.data_ptr(), rows * max_blocks, ref_counts.data_ptr(),
          out_ref_counts.data_ptr(), out_num_live.data_ptr(), ws.data_ptr(), size)
    return out_num_live
