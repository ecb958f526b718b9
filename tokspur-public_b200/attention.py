"""Harness objects over the attention entries of the C ABI: paged key / value cache, the rows of a step, head norm and rotation,
attention of drafted tokens. torch supplies device memory and streams only; every computation is a libtsp_moe.so kernel.

Row tensors are [rows, heads, head_dim], the heads of a row densely packed, rows any stride (in 16-byte steps) apart."""
from __future__ import annotations

import ctypes as C

import torch

from . import capi
from .layer import stream_ptr

TYPES = {"q8_0": capi.TYPE_Q8_0, "f16": capi.TYPE_F16}
STYLES = {"halves": capi.ROPE_HALVES, "pairs": capi.ROPE_PAIRS}


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _stride(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.stride(0) * t.element_size()


def _dtype(t: torch.Tensor) -> int:
    if t.dtype not in (torch.float32, torch.float16):
        raise TypeError(f"rows are float32 or float16, got {t.dtype}")
    return int(t.dtype == torch.float16)


def _rows(name: str, t: torch.Tensor | None, like: torch.Tensor | None = None, heads: int | None = None, dim: int | None = None, least: int = 0):
    """Checks what the library cannot see of a tensor of rows."""
    if t is None:
        return
    if t.dim() != 3 or t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != t.shape[2]):
        raise ValueError(f"{name}: rows are [rows, heads, head_dim] with densely packed heads")
    if (heads is not None and t.shape[1] != heads) or (dim is not None and t.shape[2] != dim) or t.shape[0] < least:
        raise ValueError(f"{name}: shape {tuple(t.shape)} does not hold {least} rows of {heads} heads of {dim}")
    if like is not None and t.dtype != like.dtype:
        raise TypeError(f"{name}: rows of {t.dtype} beside rows of {like.dtype}")


class KvCache:
    """A pool of pages (uint8 [pages, page stride]) and the page table (int32 [sequences, pages of a sequence]) that names them."""

    def __init__(self, pages: torch.Tensor, page_table: torch.Tensor, page_tokens: int, kv_heads: int, head_dim: int, type_: str):
        if pages.dtype != torch.uint8 or pages.dim() != 2 or pages.stride(1) != 1:
            raise ValueError("pages are uint8 [pages, page stride]")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1:
            raise ValueError("the page table is int32 [sequences, pages of a sequence]")
        if pages.shape[1] < page_bytes(type_, page_tokens, kv_heads, head_dim):
            raise ValueError("a page is smaller than its slots need")
        self.pages, self.page_table, self.kv_heads, self.head_dim, self.sequences = pages, page_table, kv_heads, head_dim, page_table.shape[0]
        # a row of the table may be part of a wider one: the stride is what the library walks by
        if page_table.shape[0] > 1 and page_table.stride(0) != page_table.shape[1]:
            raise ValueError("the page table is densely packed")
        self.struct = capi.KvCache(pages.data_ptr(), pages.stride(0), page_table.data_ptr(), page_table.shape[1], pages.shape[0], page_tokens, kv_heads,
                                   head_dim, TYPES[type_])
        self.ref = C.byref(self.struct)


def page_bytes(type_: str, page_tokens: int, kv_heads: int, head_dim: int) -> int:
    return int(capi.lib().tsp_kv_page_bytes(TYPES[type_], page_tokens, kv_heads, head_dim))


class KvBatch:
    """The rows of one step: int32 row offsets [sequences + 1] and cache lengths [sequences] on the device."""

    def __init__(self, row_offsets: torch.Tensor, lengths: torch.Tensor, rows: int):
        if row_offsets.dtype != torch.int32 or lengths.dtype != torch.int32 or row_offsets.numel() != lengths.numel() + 1 \
                or not row_offsets.is_contiguous() or not lengths.is_contiguous():
            raise ValueError("int32 row offsets of one more than the lengths")
        self.row_offsets, self.lengths, self.rows, self.sequences = row_offsets, lengths, rows, lengths.numel()
        self.struct = capi.KvBatch(row_offsets.data_ptr(), lengths.data_ptr(), lengths.numel(), rows)
        self.ref = C.byref(self.struct)


class QkNormRope:
    """Norm weights (float32 [head_dim] or None) and rotation of query and key heads."""

    def __init__(self, head_dim: int, rotary_dim: int, style: str, inv_freq: torch.Tensor | None, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6, magnitude: float = 1.0):
        for t, n in ((inv_freq, rotary_dim // 2), (q_norm, head_dim), (k_norm, head_dim)):
            if t is not None and (t.dtype != torch.float32 or t.numel() < n or not t.is_contiguous()):
                raise ValueError("norm weights and frequencies are dense float32")
        self.tensors, self.head_dim = (inv_freq, q_norm, k_norm), head_dim
        self.struct = capi.QkNormRope(_ptr(q_norm), _ptr(k_norm), _ptr(inv_freq), head_dim, rotary_dim, STYLES[style], eps, magnitude)
        self.ref = C.byref(self.struct)


def _check_batch(cache: KvCache, batch: KvBatch):
    if batch.sequences > cache.sequences:
        raise ValueError("the page table has fewer sequences than the batch")


def qk_norm_rope(turn: QkNormRope, q, k, positions, q_out, k_out, error):
    """q / k [rows, heads, head_dim] (either may be None) -> q_out / k_out of any of the two dtypes; positions int32 [rows]."""
    x = q if q is not None else k
    _rows("q", q, dim=turn.head_dim)
    _rows("k", k, like=q, dim=turn.head_dim, least=x.shape[0])
    o = q_out if q is not None else k_out
    for name, t, src in (("q_out", q_out, q), ("k_out", k_out, k)):
        if src is not None:
            _rows(name, t, like=o, heads=src.shape[1], dim=turn.head_dim, least=x.shape[0])
    if positions.dtype != torch.int32 or positions.numel() < x.shape[0] or not positions.is_contiguous():
        raise ValueError("positions are int32, one for each row")
    capi.call("tsp_qk_norm_rope", turn.ref, _ptr(q), _stride(q), _ptr(k), _stride(k), _dtype(x), positions.data_ptr(), x.shape[0],
              0 if q is None else q.shape[1], 0 if k is None else k.shape[1], _ptr(q_out), _stride(q_out), _ptr(k_out), _stride(k_out), _dtype(o),
              _ptr(error), stream_ptr())


def kv_cache_append(cache: KvCache, batch: KvBatch, k, v, error):
    _check_batch(cache, batch)
    _rows("k", k, heads=cache.kv_heads, dim=cache.head_dim, least=batch.rows)
    _rows("v", v, like=k, heads=cache.kv_heads, dim=cache.head_dim, least=batch.rows)
    capi.call("tsp_kv_cache_append", cache.ref, batch.ref, k.data_ptr(), _stride(k), v.data_ptr(), _stride(v), _dtype(k), _ptr(error), stream_ptr())


def qk_norm_rope_append(turn: QkNormRope, cache: KvCache, batch: KvBatch, q, k, v, positions, q_out, error):
    """Norm and rotation of q into q_out; of k into the cache, beside v."""
    _check_batch(cache, batch)
    _rows("q", q, dim=cache.head_dim, least=batch.rows)
    _rows("k", k, like=q, heads=cache.kv_heads, dim=cache.head_dim, least=batch.rows)
    _rows("v", v, like=q, heads=cache.kv_heads, dim=cache.head_dim, least=batch.rows)
    _rows("q_out", q_out, heads=q.shape[1], dim=cache.head_dim, least=batch.rows)
    if positions.dtype != torch.int32 or positions.numel() < batch.rows or not positions.is_contiguous():
        raise ValueError("positions are int32, one for each row")
    capi.call("tsp_qk_norm_rope_append", turn.ref, cache.ref, batch.ref, q.data_ptr(), _stride(q), k.data_ptr(), _stride(k), v.data_ptr(), _stride(v),
              _dtype(q), positions.data_ptr(), q.shape[1], q_out.data_ptr(), _stride(q_out), _dtype(q_out), _ptr(error), stream_ptr())


def kv_cache_read(cache: KvCache, batch: KvBatch, k_out, v_out, error):
    _check_batch(cache, batch)
    o = k_out if k_out is not None else v_out
    _rows("k_out", k_out, heads=cache.kv_heads, dim=cache.head_dim, least=batch.rows)
    _rows("v_out", v_out, like=o, heads=cache.kv_heads, dim=cache.head_dim, least=batch.rows)
    capi.call("tsp_kv_cache_read", cache.ref, batch.ref, _ptr(k_out), _stride(k_out), _ptr(v_out), _stride(v_out), _dtype(o), _ptr(error), stream_ptr())


def kv_cache_keep(cache: KvCache, batch: KvBatch, accepted, counts, error):
    """accepted int32 [rows] (a sequence's accepted nodes from its row offset on, ascending), counts int32 [sequences]."""
    _check_batch(cache, batch)
    for name, t, n in (("accepted", accepted, batch.rows), ("counts", counts, batch.sequences)):
        if t.dtype != torch.int32 or t.numel() < n or not t.is_contiguous():
            raise ValueError(f"{name}: int32, {n} of them")
    capi.call("tsp_kv_cache_keep", cache.ref, batch.ref, accepted.data_ptr(), counts.data_ptr(), _ptr(error), stream_ptr())


def tree_attention_scratch(device="cuda") -> torch.Tensor:
    """The workspace of tree_attention on `device`, as its first call wants it (zeros)."""
    with torch.cuda.device(device):
        return torch.zeros(int(capi.lib().tsp_tree_attention_scratch_bytes()), dtype=torch.uint8, device=device)


def tree_attention(cache: KvCache, batch: KvBatch, q, out, tree_mask, max_rows: int, scale: float, scratch, error):
    """q [rows, q_heads, head_dim] -> out, the same shape and dtype; tree_mask int64 [rows] (bit i: the row sees token i of its step) or None (chain)."""
    _check_batch(cache, batch)
    _rows("q", q, dim=cache.head_dim, least=batch.rows)
    _rows("out", out, like=q, heads=q.shape[1], dim=cache.head_dim, least=batch.rows)
    if tree_mask is not None and (tree_mask.dtype != torch.int64 or tree_mask.numel() < batch.rows or not tree_mask.is_contiguous()):
        raise ValueError("the tree's words are int64, one for each row")
    capi.call("tsp_tree_attention", cache.ref, batch.ref, q.data_ptr(), _stride(q), _ptr(tree_mask), q.shape[1], max_rows, scale, out.data_ptr(), _stride(out),
              _dtype(q), scratch.data_ptr(), scratch.numel(), _ptr(error), stream_ptr())
