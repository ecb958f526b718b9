"""CPU-only checks of the attention operators: sizes of the cache, and every refusal that happens before a launch."""
import ctypes as C

import numpy as np
import pytest
import torch

import attention_ref as R
from tokspur_public_b200 import attention as A
from tokspur_public_b200 import capi


def test_page_bytes():
    lib = capi.lib()
    for type_, name in ((capi.TYPE_Q8_0, "q8_0"), (capi.TYPE_F16, "f16")):
        for dim in (64, 128, 256):
            for page in (16, 32, 64, 128, 256):
                assert lib.tsp_kv_page_bytes(type_, page, 3, dim) == 3 * (page // 16) * 2 * R.half_bytes(dim, name)
    for bad in ((12, 64, 8, 128), (8, 48, 8, 128), (8, 512, 8, 128), (8, 8, 8, 128), (8, 64, 0, 128), (8, 64, 257, 128), (8, 64, 8, 96)):
        assert lib.tsp_kv_page_bytes(*bad) == 0


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_layout_tables_are_permutations(type_, dim):
    """Every byte of a group's part has one value."""
    k, v, scale = R.places(dim, type_)
    step = 1 if type_ == "q8_0" else 2
    for at in (k, v):
        assert np.array_equal(np.sort(at.ravel()), np.arange(16 * dim) * step)
    if scale is not None:
        assert np.array_equal(np.sort(scale.ravel()), 16 * dim + 2 * np.arange(dim // 2))


def test_host_model_of_the_cache_gives_back_what_it_took():
    rng = np.random.default_rng(3)
    for type_ in ("q8_0", "f16"):
        p = R.Pages(rng, type_, 32, 2, 64, [70])
        k, v = rng.normal(size=(70, 2, 64)), rng.normal(size=(70, 2, 64))
        for i in range(70):
            p.put(0, i, k[i], v[i])
        for i in range(70):
            a, b = p.get(0, i)
            assert np.array_equal(a, R.cached(k[i], type_)) and np.array_equal(b, R.cached(v[i], type_))


class Call:
    """Arguments of every entry that would be accepted but for the device; the pointers are never followed."""

    def __init__(self):
        self.cache = capi.KvCache(1 << 32, capi.lib().tsp_kv_page_bytes(8, 64, 8, 128), 1 << 20, 16, 64, 64, 8, 128, 8)
        self.batch = capi.KvBatch(1 << 21, 1 << 22, 4, 32)
        self.turn = capi.QkNormRope(1 << 23, 1 << 23, 1 << 24, 128, 128, 0, 1e-6, 1.0)
        self.q, self.k, self.v, self.out, self.kout = 1 << 40, 2 << 40, 3 << 40, 4 << 40, 5 << 40
        self.qs, self.ks, self.vs, self.os, self.kos = 16384, 4096, 4096, 16384, 4096
        self.dtype, self.out_dtype, self.q_heads, self.kv_heads, self.rows, self.max_rows, self.scale = 0, 0, 32, 8, 32, 8, 0.1
        self.positions, self.mask, self.scratch, self.scratch_bytes = 1 << 25, 1 << 26, 6 << 40, 1 << 30
        self.accepted, self.counts = 1 << 27, 1 << 28

    def norm(self):
        return capi.lib().tsp_qk_norm_rope(C.byref(self.turn), self.q, self.qs, self.k, self.ks, self.dtype, self.positions, self.rows, self.q_heads,
                                           self.kv_heads, self.out, self.os, self.kout, self.kos, self.out_dtype, None, None)

    def fused(self):
        return capi.lib().tsp_qk_norm_rope_append(C.byref(self.turn), C.byref(self.cache), C.byref(self.batch), self.q, self.qs, self.k, self.ks, self.v,
                                                  self.vs, self.dtype, self.positions, self.q_heads, self.out, self.os, self.out_dtype, None, None)

    def append(self):
        return capi.lib().tsp_kv_cache_append(C.byref(self.cache), C.byref(self.batch), self.k, self.ks, self.v, self.vs, self.dtype, None, None)

    def read(self):
        return capi.lib().tsp_kv_cache_read(C.byref(self.cache), C.byref(self.batch), self.k, self.ks, self.v, self.vs, self.dtype, None, None)

    def keep(self):
        return capi.lib().tsp_kv_cache_keep(C.byref(self.cache), C.byref(self.batch), self.accepted, self.counts, None, None)

    def attend(self):
        return capi.lib().tsp_tree_attention(C.byref(self.cache), C.byref(self.batch), self.q, self.qs, self.mask, self.q_heads, self.max_rows, self.scale,
                                             self.out, self.os, self.dtype, self.scratch, self.scratch_bytes, None, None)


def refused(entry, code=capi.E_ARG, **change):
    c = Call()
    for name, value in change.items():
        target, _, field = name.partition("__")
        setattr(getattr(c, target) if field else c, field or target, value)
    assert getattr(c, entry)() == code, (entry, change, capi.last_error())


CACHE = ["fused", "append", "read", "keep", "attend"]


@pytest.mark.parametrize("entry", CACHE)
def test_refusals_of_the_cache_and_the_batch(entry):
    for change in (dict(cache__d_pages=None), dict(cache__d_pages=(1 << 32) + 8), dict(cache__d_page_table=None), dict(cache__d_page_table=(1 << 20) + 2),
                   dict(cache__page_stride_bytes=1024), dict(cache__page_stride_bytes=(1 << 20) + 8), dict(cache__table_stride=0), dict(cache__table_stride=1 << 25),
                   dict(cache__pages=0), dict(cache__pages=1 << 31), dict(cache__page_tokens=48), dict(cache__page_tokens=512), dict(cache__kv_heads=0),
                   dict(cache__kv_heads=257), dict(batch__d_row_offsets=None), dict(batch__d_lengths=None), dict(batch__d_lengths=(1 << 22) + 1),
                   dict(batch__sequences=0), dict(batch__sequences=1025), dict(batch__rows=0), dict(batch__rows=(1 << 20) + 1)):
        refused(entry, **change)
    refused(entry, capi.E_TYPE, cache__type=12)
    refused(entry, capi.E_TYPE, cache__head_dim=96)


def test_refusals_of_rows():
    for entry in ("norm", "fused", "attend"):
        for change in (dict(q=None), dict(q=(1 << 40) + 8), dict(qs=16376), dict(qs=8192), dict(out=None), dict(os=16368), dict(dtype=2), dict(q=4 << 40, qs=32768)):
            refused(entry, **change)
    for entry in ("norm", "fused", "append", "read"):
        for change in (dict(k=(2 << 40) + 4), dict(ks=2048), dict(ks=4104)):
            refused(entry, **change)
    for entry in ("fused", "append"):
        for change in (dict(k=None), dict(v=None), dict(vs=4000), dict(v=1 << 32), dict(k=(1 << 32) - 4096)):
            refused(entry, **change)
    refused("fused", q_heads=0)
    refused("fused", out=1 << 32)
    refused("fused", out=2 << 40)
    refused("fused", out_dtype=1, out=1 << 40)          # in place, of another type
    refused("norm", out=2 << 40)
    refused("norm", kout=4 << 40)
    refused("norm", q_heads=0, kv_heads=0)
    refused("norm", rows=0)
    refused("norm", positions=None)
    refused("read", k=None, v=None)
    refused("read", v=2 << 40)
    refused("read", k=1 << 32)
    refused("keep", accepted=None)
    refused("keep", counts=None)
    refused("keep", counts=(1 << 28) + 2)


def test_refusals_of_norm_and_rotation():
    for entry in ("norm", "fused"):
        for change in (dict(turn__rotary_dim=130), dict(turn__rotary_dim=4), dict(turn__rotary_dim=136), dict(turn__style=2), dict(turn__eps=-1.0),
                       dict(turn__eps=float("nan")), dict(turn__magnitude=float("inf")), dict(turn__d_inv_freq=None), dict(turn__d_q_norm=(1 << 23) + 1)):
            refused(entry, **change)
    refused("norm", capi.E_TYPE, turn__head_dim=80)
    refused("fused", turn__head_dim=64)                  # not the cache's


def test_refusals_of_attention():
    for change in (dict(q_heads=33), dict(q_heads=8 * 65, qs=1 << 20, os=1 << 20), dict(max_rows=0), dict(max_rows=65), dict(scale=float("inf")), dict(mask=(1 << 26) + 4),
                   dict(scratch=None), dict(scratch=(6 << 40) + 8), dict(scratch_bytes=0), dict(out=1 << 40), dict(out=1 << 32), dict(scratch=1 << 40),
                   dict(scratch=4 << 40), dict(scratch=1 << 32)):
        refused("attend", **change)


def test_accepted_arguments_reach_the_device():
    """Nothing of the calls above is refused for another reason than the one changed: without a device they end in a CUDA error."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("would follow the pointers")
    for entry in ["norm"] + CACHE:
        assert getattr(Call(), entry)() == capi.E_CUDA, (entry, capi.last_error())


def test_tensors_of_another_device_are_refused():
    """Host memory beside a cache on a GPU (only its device index is set here): the library would follow the pointer on the wrong device."""
    rows, heads, dim = 3, 2, 64
    cache = A.KvCache(torch.zeros(4, A.page_bytes("q8_0", 16, heads, dim), dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), 16, heads, dim, "q8_0")
    batch = A.KvBatch(torch.tensor([0, rows], dtype=torch.int32), torch.zeros(1, dtype=torch.int32), rows)
    turn = A.QkNormRope(dim, dim, "halves", torch.ones(dim // 2))
    k, words = torch.zeros(rows, heads, dim), torch.zeros(rows, dtype=torch.int32)
    cache.device = 0
    with pytest.raises(ValueError, match="row offsets: on cpu"):
        A.kv_cache_append(cache, batch, k, k, None)
    batch.device = 0
    with pytest.raises(ValueError, match="k: on cpu"):
        A.kv_cache_append(cache, batch, k, k, None)
    with pytest.raises(ValueError, match="k_out: on cpu"):
        A.kv_cache_read(cache, batch, k, None, None)
    with pytest.raises(ValueError, match="accepted: on cpu"):
        A.kv_cache_keep(cache, batch, words, words, None)
    with pytest.raises(ValueError, match="frequencies on devices"):
        A.qk_norm_rope_append(turn, cache, batch, k, k, k, words, k, None)
    with pytest.raises(ValueError, match="q: on cpu"):
        A.tree_attention(cache, batch, k, k, None, rows, 1.0, torch.zeros(1, dtype=torch.uint8), None)
    with pytest.raises(ValueError, match="no rows"):
        A.kv_cache_read(cache, batch, None, None, None)
    k16 = k.to(torch.bfloat16)
    with pytest.raises(ValueError, match="bfloat16"):
        A.kv_cache_append(cache, batch, k16, k16, None)
