"""Harness objects over the attention entries of the C ABI: paged key / value cache, the rows of a step, head norm and rotation,
attention of drafted tokens. torch supplies device memory and streams only; every computation is a libtsp_moe.so kernel.

Row tensors are [rows, heads, head_dim], the heads of a row densely packed, rows any stride (in 16-byte steps) apart."""
from __future__ import annotations

import ctypes as C

import torch

from . import capi

TYPES = {"q8_0": capi.TYPE_Q8_0, "f16": capi.TYPE_F16}
STYLES = {"halves": capi.ROPE_HALVES, "pairs": capi.ROPE_PAIRS}
SIZES = {torch.float32: 4, torch.float16: 2}   # of the row types; the library's dtype is 0 for four bytes, 1 for two


def _refuse(name, t, dtype, heads, dim, least):
    raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device} does not hold {least} rows of {heads} densely packed heads of {dim} {dtype}")


def _elsewhere(name, t, device):
    raise ValueError(f"{name}: on {t.device}, the call is for CUDA device {device}")


def _rows(name: str, t: torch.Tensor, dtype: torch.dtype, heads: int, dim: int, least: int, device: int) -> tuple[int, int]:
    """Pointer and row stride in bytes of [rows, heads, dim], after the checks that the library cannot make. A call of a few microseconds is
    in good part these lines: they ask each tensor as little as they can."""
    try:
        (rows, h, d), (step, between, one) = t.shape, t.stride()
        size = SIZES[dtype]
    except (ValueError, KeyError):
        _refuse(name, t, dtype, heads, dim, least)
    if rows < least or h != heads or d != dim or one != 1 or (between != dim and h != 1) or t.dtype is not dtype:
        _refuse(name, t, dtype, heads, dim, least)
    if t.get_device() != device:
        _elsewhere(name, t, device)
    return t.data_ptr(), step * size


def _words(name: str, t: torch.Tensor, dtype: torch.dtype, least: int, device: int) -> int:
    if t is None or t.dtype is not dtype or t.numel() < least or not t.is_contiguous():
        raise ValueError(f"{name}: {least} dense values of {dtype}")
    if t.get_device() != device:
        _elsewhere(name, t, device)
    return t.data_ptr()


_entries: dict = {}
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
# the current stream's handle without a Stream object around it (a microsecond less a call), where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _call(name: str, device: int, error: torch.Tensor | None, *args) -> None:
    """The library's entry on a device, on torch's current stream there."""
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = getattr(capi.lib(), name)
    if error is not None:
        if error.dtype is not torch.int32 or error.numel() < 1:
            raise ValueError("error word: one int32")
        if error.get_device() != device:
            _elsewhere("error word", error, device)
    if device < 0:
        raise ValueError(f"{name}: tensors in host memory")
    if device != _current_device():
        with torch.cuda.device(device):
            return _call(name, device, error, *args)
    rc = entry(*args, None if error is None else error.data_ptr(), _raw_stream(device))
    if rc:
        capi.check(rc)


class KvCache:
    """A pool of pages (uint8 [pages, page stride]) and the page table (int32 [sequences, pages of a sequence]) that names them."""

    def __init__(self, pages: torch.Tensor, page_table: torch.Tensor, page_tokens: int, kv_heads: int, head_dim: int, type_: str):
        if pages.dtype != torch.uint8 or pages.dim() != 2 or pages.stride(1) != 1:
            raise ValueError("pages are uint8 [pages, page stride]")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1:
            raise ValueError("the page table is int32 [sequences, pages of a sequence]")
        if pages.shape[1] < page_bytes(type_, page_tokens, kv_heads, head_dim):
            raise ValueError("a page is smaller than its slots need")
        self.device = pages.get_device()
        if page_table.get_device() != self.device:
            _elsewhere("page table", page_table, self.device)
        self.pages, self.page_table, self.kv_heads, self.head_dim, self.sequences = pages, page_table, kv_heads, head_dim, page_table.shape[0]
        # The library has one number for the words between two rows and for the pages of a sequence: columns of a wider table would pass for pages of this one
        if page_table.shape[0] > 1 and page_table.stride(0) != page_table.shape[1]:
            raise ValueError("the rows of the page table are not next to one another")
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
        self.device = lengths.get_device()
        if row_offsets.get_device() != self.device:
            _elsewhere("row offsets", row_offsets, self.device)
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
        devices = {t.get_device() for t in self.tensors if t is not None}
        if len(devices) > 1:
            raise ValueError(f"norm weights and frequencies on devices {sorted(devices)}")
        self.device = devices.pop() if devices else None
        self.struct = capi.QkNormRope(*(None if t is None else t.data_ptr() for t in (q_norm, k_norm, inv_freq)), head_dim, rotary_dim, STYLES[style], eps, magnitude)
        self.ref = C.byref(self.struct)


def _check_batch(cache: KvCache, batch: KvBatch) -> int:
    """The device of both."""
    if batch.sequences > cache.sequences:
        raise ValueError("the page table has fewer sequences than the batch")
    if batch.device != cache.device:
        _elsewhere("row offsets", batch.row_offsets, cache.device)
    return cache.device


def _check_turn(turn: QkNormRope, device: int):
    if turn.device is not None and turn.device != device:
        raise ValueError(f"norm weights and frequencies on devices {[turn.device]}, the call is for CUDA device {device}")


def _positions(turn: QkNormRope, positions, rows: int, device: int):
    return None if positions is None and not turn.struct.rotary_dim else _words("positions", positions, torch.int32, rows, device)


def qk_norm_rope(turn: QkNormRope, q, k, positions, q_out, k_out, error):
    """q / k [rows, heads, head_dim] (one may be None) -> q_out / k_out of any of the two dtypes; positions int32 [rows], None where nothing is rotated."""
    x, o, dim = (q, q_out, turn.head_dim) if q is not None else (k, k_out, turn.head_dim)
    if x is None or o is None or (q is not None and k is not None and k_out is None):
        raise ValueError("qk_norm_rope: rows of queries, keys or both, and as many outputs")
    rows, dt, ot = x.shape[0], x.dtype, o.dtype
    device = x.get_device()
    _check_turn(turn, device)
    hq = hk = qs = ks = qos = kos = 0
    qp = kp = qop = kop = None
    if q is not None:
        hq = q.shape[1]
        qp, qs = _rows("q", q, dt, hq, dim, rows, device)
        qop, qos = _rows("q_out", q_out, ot, hq, dim, rows, device)
    if k is not None:
        hk = k.shape[1]
        kp, ks = _rows("k", k, dt, hk, dim, rows, device)
        kop, kos = _rows("k_out", k_out, ot, hk, dim, rows, device)
    _call("tsp_qk_norm_rope", device, error, turn.ref, qp, qs, kp, ks, int(dt is torch.float16), _positions(turn, positions, rows, device), rows, hq, hk, qop, qos,
          kop, kos, int(ot is torch.float16))


def kv_cache_append(cache: KvCache, batch: KvBatch, k, v, error):
    device = _check_batch(cache, batch)
    dt = k.dtype
    kp, ks = _rows("k", k, dt, cache.kv_heads, cache.head_dim, batch.rows, device)
    vp, vs = _rows("v", v, dt, cache.kv_heads, cache.head_dim, batch.rows, device)
    _call("tsp_kv_cache_append", device, error, cache.ref, batch.ref, kp, ks, vp, vs, int(dt is torch.float16))


def qk_norm_rope_append(turn: QkNormRope, cache: KvCache, batch: KvBatch, q, k, v, positions, q_out, error):
    """Norm and rotation of q into q_out; of k into the cache, beside v."""
    device = _check_batch(cache, batch)
    _check_turn(turn, device)
    dt, ot, dim, heads, rows = q.dtype, q_out.dtype, cache.head_dim, q.shape[1], batch.rows
    qp, qs = _rows("q", q, dt, heads, dim, rows, device)
    kp, ks = _rows("k", k, dt, cache.kv_heads, dim, rows, device)
    vp, vs = _rows("v", v, dt, cache.kv_heads, dim, rows, device)
    op, os = _rows("q_out", q_out, ot, heads, dim, rows, device)
    _call("tsp_qk_norm_rope_append", device, error, turn.ref, cache.ref, batch.ref, qp, qs, kp, ks, vp, vs, int(dt is torch.float16),
          _positions(turn, positions, rows, device), heads, op, os, int(ot is torch.float16))


def kv_cache_read(cache: KvCache, batch: KvBatch, k_out, v_out, error):
    """Either of k_out and v_out may be None."""
    device = _check_batch(cache, batch)
    x = k_out if k_out is not None else v_out
    if x is None:
        raise ValueError("kv_cache_read: no rows to read into")
    kp, ks = (None, 0) if k_out is None else _rows("k_out", k_out, x.dtype, cache.kv_heads, cache.head_dim, batch.rows, device)
    vp, vs = (None, 0) if v_out is None else _rows("v_out", v_out, x.dtype, cache.kv_heads, cache.head_dim, batch.rows, device)
    _call("tsp_kv_cache_read", device, error, cache.ref, batch.ref, kp, ks, vp, vs, int(x.dtype is torch.float16))


def kv_cache_keep(cache: KvCache, batch: KvBatch, accepted, counts, error):
    """accepted int32 [rows] (a sequence's accepted nodes from its row offset on, ascending), counts int32 [sequences]."""
    device = _check_batch(cache, batch)
    _call("tsp_kv_cache_keep", device, error, cache.ref, batch.ref, _words("accepted", accepted, torch.int32, batch.rows, device), _words("counts", counts, torch.int32, batch.sequences, device))


def tree_attention_scratch(device="cuda") -> torch.Tensor:
    """The workspace of tree_attention on `device`, as its first call wants it (zeros)."""
    with torch.cuda.device(device):
        return torch.zeros(int(capi.lib().tsp_tree_attention_scratch_bytes()), dtype=torch.uint8, device=device)


def tree_attention(cache: KvCache, batch: KvBatch, q, out, tree_mask, max_rows: int, scale: float, scratch, error):
    """q [rows, q_heads, head_dim] -> out, the same shape and dtype; tree_mask int64 [rows] (bit i: the row sees token i of its step) or None (chain)."""
    device = _check_batch(cache, batch)
    dt, heads, dim, rows = q.dtype, q.shape[1], cache.head_dim, batch.rows
    qp, qs = _rows("q", q, dt, heads, dim, rows, device)
    op, os = _rows("out", out, dt, heads, dim, rows, device)
    workspace = _words("scratch", scratch, torch.uint8, 1, device)   # dense: its size is what the library may write
    _call("tsp_tree_attention", device, error, cache.ref, batch.ref, qp, qs, None if tree_mask is None else _words("tree words", tree_mask, torch.int64, rows, device), heads, max_rows,
          scale, op, os, int(dt is torch.float16), workspace, scratch.numel())
