"""Head norm and rotation, the paged cache and the attention of drafted tokens against 64-bit restatements (attention_ref.py).

Tolerances, set before the first run. u16 = 2^-11, u32 = 2^-24 (half a step of binary16 / FP32 relative to the value).
  norm and rotation, FP32: a sum of dim squares, a square root, a division, four products, one rotation of two products with sin / cos good to 2
      units and angles to 2^-22: under 2^-19 of the head's largest value; binary16 rows add u16 of the value (2^-25 below 2^-14).
  cache: exact.
  attention, FP32 rows: a score is a sum of dim terms with FP32 rounding each, e = (dim + 8) u32 * sum|q_i k_i| scale; a weight changes by 2e at most,
      its normalisation by as much; the sum over the slots in FP32, slots u32 at worst: |v|max (4 e + (slots + 64) u32).
  attention, binary16 rows: products of binary16 parts, e = (u16 + (dim + 8) u32) sum|q_i k_i| scale for a key value rounded to binary16; weights and
      value products rounded to binary16: |v|max (4 e + 4 u16), and u16 of the result for its own rounding.
  Beside these bounds of the worst case, the 2-norm over all rows: errors of independent roundings, 5e-6 (FP32) and 2e-3 (binary16) of the result's.
"""
import numpy as np
import pytest

import attention_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tokspur_public_b200 import attention as A  # noqa: E402
from tokspur_public_b200 import capi  # noqa: E402

U16, U32 = 2.0 ** -11, 2.0 ** -24
NP = {"f32": np.float32, "f16": np.float16}


def dev(a):
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint32:
        a = a.view(np.int32)
    if a.dtype == np.uint64:
        a = a.view(np.int64)
    return torch.from_numpy(a).cuda()


def error_word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def check_turned(got, want, dtype):
    got = got.astype(np.float64)
    top = np.abs(want).max(-1, keepdims=True)
    tol = top * 2.0 ** -19 + (np.abs(want) * U16 + 2.0 ** -25 if dtype == "f16" else 0)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / (tol + 1e-300)).max())


def inv_freq(rotary, theta=1e6):
    return (theta ** (-np.arange(rotary // 2) / max(1, rotary // 2))).astype(np.float32)


# ---- norm and rotation -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,rotary,style", [(64, 64, "halves"), (64, 8, "pairs"), (128, 128, "halves"), (128, 128, "pairs"), (128, 64, "halves"), (128, 40, "halves"),
                                              (256, 256, "halves"), (256, 64, "pairs"), (256, 192, "halves"), (128, 0, "halves")])
@pytest.mark.parametrize("dtypes", [("f32", "f32"), ("f16", "f16"), ("f32", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("rows,hq,hk", [(1, 1, 1), (3, 7, 2), (17, 32, 8)])
def test_norm_and_rotation(dim, rotary, style, dtypes, rows, hq, hk):
    rng = np.random.default_rng(dim + rotary + rows)
    q, k = (rng.normal(size=(rows, h, dim)).astype(NP[dtypes[0]]) for h in (hq, hk))
    pos = rng.integers(0, 1 << 32, rows).astype(np.uint32)
    pos[0] = 0
    wq, wk = ((1 + 0.2 * rng.normal(size=dim)).astype(np.float32) for _ in range(2))
    f = inv_freq(rotary)
    turn = A.QkNormRope(dim, rotary, style, dev(f) if rotary else None, dev(wq), dev(wk), eps=1e-5, magnitude=1.25)
    qo, ko = (torch.full((rows + 1, h, dim), 7.0, dtype=getattr(torch, "float32" if dtypes[1] == "f32" else "float16"), device="cuda") for h in (hq, hk))
    err = error_word()
    A.qk_norm_rope(turn, dev(q), dev(k), dev(pos), qo, ko, err)
    assert int(err) == 0
    for x, w, o in ((q, wq, qo), (k, wk, ko)):
        check_turned(o[:rows].cpu().numpy(), R.turned(x, w, pos, f, rotary, style, 1e-5, 1.25), dtypes[1])
        assert (o[rows:] == 7).all()


def test_norm_and_rotation_of_parts_of_a_fused_row_in_place_and_one_side_alone():
    rng = np.random.default_rng(5)
    rows, hq, hk, dim = 9, 6, 2, 128
    x = rng.normal(size=(rows, hq + 2 * hk, dim)).astype(np.float32)
    pos, f, w = rng.integers(0, 5000, rows).astype(np.uint32), inv_freq(dim), (1 + 0.1 * rng.normal(size=dim)).astype(np.float32)
    turn = A.QkNormRope(dim, dim, "halves", dev(f), dev(w), None)
    t, err = dev(x), error_word()
    q, k = t[:, :hq], t[:, hq:hq + hk]
    A.qk_norm_rope(turn, q, k, dev(pos), q, k, err)
    got = t.cpu().numpy()
    check_turned(got[:, :hq], R.turned(x[:, :hq], w, pos, f, dim, "halves", 1e-6), "f32")
    check_turned(got[:, hq:hq + hk], R.turned(x[:, hq:hq + hk], None, pos, f, dim, "halves", 1e-6), "f32")
    assert np.array_equal(got[:, hq + hk:], x[:, hq + hk:])
    only = torch.empty(rows, hk, dim, device="cuda")
    A.qk_norm_rope(turn, None, dev(x[:, :hk]), dev(pos), None, only, err)
    check_turned(only.cpu().numpy(), R.turned(x[:, :hk], None, pos, f, dim, "halves", 1e-6), "f32")
    assert int(err) == 0


def test_norm_and_rotation_of_rows_that_are_not_finite_or_zero():
    dim, f = 128, inv_freq(128)
    x = np.random.default_rng(1).normal(size=(4, 2, dim)).astype(np.float32)
    x[1, 1, 5], x[2, 0, 100], x[3, 1] = np.nan, np.inf, 0
    turn = A.QkNormRope(dim, dim, "halves", dev(f), dev(np.ones(dim, np.float32)), None)
    out, err = torch.full((4, 2, dim), 3.0, device="cuda"), error_word()
    pos = np.arange(4).astype(np.uint32)
    A.qk_norm_rope(turn, dev(x), None, dev(pos), out, None, err)
    assert int(err) == capi.ERR_NONFINITE
    want = R.turned(np.where(np.isfinite(x), x, 0), np.ones(dim), pos, f, dim, "halves", 1e-6)
    want[1, 1] = want[2, 0] = 0
    check_turned(out.cpu().numpy(), want, "f32")
    big = np.full((1, 1, dim), 7e4, np.float32)     # fits FP32, not binary16
    err.zero_()
    o16 = torch.ones(1, 1, dim, dtype=torch.float16, device="cuda")
    A.qk_norm_rope(A.QkNormRope(dim, 0, "halves", None), dev(big), None, dev(pos), o16, None, err)
    assert int(err) == capi.ERR_NONFINITE and (o16 == 0).all()


# ---- the cache -----------------------------------------------------------------------------------------------------------------
def make_batch(counts, lengths, rows=None):
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)
    return A.KvBatch(dev(off), dev(np.array(lengths, np.uint32)), int(off[-1]) if rows is None else rows), off


def make_cache(p):
    return A.KvCache(dev(p.data), dev(p.table), p.page, p.heads, p.dim, p.type)


SHAPES = [([1], [0]), ([1], [16]), ([3, 0, 5], [15, 4, 62]), ([40, 1, 17, 64], [7, 0, 100, 33]), ([1] * 37, list(range(0, 74, 2)))]


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 3), (128, 64, 2), (128, 32, 8), (256, 256, 1)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_append_writes_its_slots_alone_and_read_gives_them_back(type_, dim, page, heads, dtype, shape):
    counts, lengths = SHAPES[shape]
    rng = np.random.default_rng(dim + page + shape)
    p = R.Pages(rng, type_, page, heads, dim, [a + b for a, b in zip(counts, lengths)], pad=48)
    cache, (batch, off) = make_cache(p), make_batch(counts, lengths)
    rows = batch.rows
    k, v = (rng.normal(size=(rows, heads, dim)).astype(NP[dtype]) for _ in range(2))
    err = error_word()
    A.kv_cache_append(cache, batch, dev(k), dev(v), err)
    assert int(err) == 0
    for s in range(len(counts)):
        for j in range(counts[s]):
            p.put(s, lengths[s] + j, k[off[s] + j].astype(np.float64), v[off[s] + j].astype(np.float64))
    assert np.array_equal(cache.pages.cpu().numpy(), p.data)     # every byte of the pool: the written slots and all others
    ko, vo = (torch.full((rows + 2, heads, dim), 9.0, dtype=torch.float32 if dtype == "f32" else torch.float16, device="cuda") for _ in range(2))
    A.kv_cache_read(cache, batch, ko, vo, err)
    assert int(err) == 0 and (ko[rows:] == 9).all() and (vo[rows:] == 9).all()
    for got, x in ((ko, k), (vo, v)):
        want = R.cached(x, type_).astype(np.float32).astype(NP[dtype])
        assert np.array_equal(got[:rows].cpu().numpy(), want)
    ko.fill_(9)
    A.kv_cache_read(cache, batch, ko, None, err)
    assert np.array_equal(ko[:rows].cpu().numpy(), R.cached(k, type_).astype(np.float32).astype(NP[dtype]))


def test_quantiser_at_its_borders():
    """Ties of the exact quotient go to the even code; scales at and below binary16's smallest values; signed zeros."""
    dim, heads = 128, 1
    x = np.zeros((6, heads, dim), np.float32)
    x[0, 0, :32] = (np.arange(32) + 0.5) * 2.0 ** -3                  # scale set by the next value: 127 / 8
    x[0, 0, 31] = 127 * 2.0 ** -3
    x[0, 0, 32:64] = -x[0, 0, :32]
    x[0, 0, 64:96] = np.nextafter(x[0, 0, :32], np.float32(1e9))      # just off the tie
    x[0, 0, 95] = 127 * 2.0 ** -3
    x[0, 0, 96:] = np.nextafter(x[0, 0, :32], np.float32(-1e9))
    x[0, 0, 127] = 127 * 2.0 ** -3
    x[1] = np.linspace(-1, 1, dim) * 127 * 2.0 ** -24                 # the smallest scale
    x[2] = np.linspace(-1, 1, dim) * 127 * 1.4 * 2.0 ** -24           # rounds down to it: codes are clamped
    x[3] = np.linspace(-1, 1, dim) * 127 * 0.4 * 2.0 ** -24           # no scale is left: zeros
    x[4] = -0.0
    x[5] = np.linspace(-1, 1, dim) * 127 * 65000.0                    # the largest
    rng = np.random.default_rng(0)
    p = R.Pages(rng, "q8_0", 16, heads, dim, [6])
    cache, (batch, _) = make_cache(p), make_batch([6], [0])
    err = error_word()
    A.kv_cache_append(cache, batch, dev(x), dev(x[::-1]), err)
    for j in range(6):
        p.put(0, j, x[j].astype(np.float64), x[5 - j].astype(np.float64))
    assert int(err) == 0 and np.array_equal(cache.pages.cpu().numpy(), p.data)


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
def test_append_of_rows_that_are_not_finite(type_):
    rng = np.random.default_rng(2)
    k, v = (rng.normal(size=(5, 2, 64)).astype(np.float32) for _ in range(2))
    k[1, 0, 3], v[2, 1, 60], k[3, 1, 0], v[4, 0, 7] = np.nan, np.inf, -np.inf, 3e38     # the last has no binary16 scale or value
    p = R.Pages(rng, type_, 16, 2, 64, [5])
    cache, (batch, _) = make_cache(p), make_batch([5], [0])
    err = error_word()
    A.kv_cache_append(cache, batch, dev(k), dev(v), err)
    assert int(err) == capi.ERR_NONFINITE
    k[1, 0], v[2, 1], k[3, 1], v[4, 0] = 0, 0, 0, 0
    for j in range(5):
        p.put(0, j, k[j].astype(np.float64), v[j].astype(np.float64))
    assert np.array_equal(cache.pages.cpu().numpy(), p.data)


def test_slots_without_a_page_and_rows_of_the_padding():
    rng = np.random.default_rng(4)
    counts, lengths = [4, 20, 3], [14, 10, 0]
    p = R.Pages(rng, "q8_0", 16, 2, 64, [18, 30, 3])
    p.table[1, 1] = 0xfffffff0          # slots 16..29 of sequence 1 have no page
    cache = make_cache(p)
    batch, off = make_batch(counts, lengths, rows=32)                 # five rows of padding
    k, v = (rng.normal(size=(32, 2, 64)).astype(np.float32) for _ in range(2))
    k[27:], v[27:] = np.nan, np.nan
    err = error_word()
    A.kv_cache_append(cache, batch, dev(k), dev(v), err)
    assert int(err) == capi.ERR_INDEX
    for s in range(3):
        for j in range(counts[s]):
            if not (s == 1 and lengths[s] + j >= 16):
                p.put(s, lengths[s] + j, k[off[s] + j].astype(np.float64), v[off[s] + j].astype(np.float64))
    assert np.array_equal(cache.pages.cpu().numpy(), p.data)
    out, err = torch.full((32, 2, 64), 5.0, device="cuda"), error_word()
    A.kv_cache_read(cache, batch, out, None, err)
    got = out.cpu().numpy()
    assert int(err) == capi.ERR_INDEX and (got[27:] == 5).all() and (got[off[1] + 6:off[2]] == 5).all()
    assert np.array_equal(got[off[2]:27], R.cached(k[off[2]:27], "q8_0").astype(np.float32))
    # a slot behind the table's last column, and offsets that descend
    err.zero_()
    A.kv_cache_append(cache, make_batch([4], [60])[0], dev(k[:4]), dev(v[:4]), err)
    assert int(err) == capi.ERR_INDEX and np.array_equal(cache.pages.cpu().numpy(), p.data)
    err.zero_()
    bad = A.KvBatch(dev(np.array([0, 3, 2, 4], np.uint32)), dev(np.array([0, 0, 0], np.uint32)), 4)
    A.kv_cache_read(cache, bad, torch.empty(4, 2, 64, device="cuda"), None, err)
    assert int(err) & capi.ERR_INDEX


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("dim,rotary,style,dtype", [(64, 64, "halves", "f32"), (128, 128, "pairs", "f16"), (128, 32, "halves", "f32"), (256, 64, "halves", "f16")])
def test_fused_norm_rotation_and_append(type_, dim, rotary, style, dtype):
    rng = np.random.default_rng(dim)
    counts, lengths, heads, hq = [5, 0, 33, 1], [100, 3, 14, 0], 2, 6
    p = R.Pages(rng, type_, 32, heads, dim, [a + b for a, b in zip(counts, lengths)])
    cache, (batch, off) = make_cache(p), make_batch(counts, lengths, rows=41)
    x = rng.normal(size=(41, hq + 2 * heads, dim)).astype(NP[dtype])
    pos = rng.integers(0, 20000, 41).astype(np.uint32)
    wq, wk, f = (1 + 0.1 * rng.normal(size=dim)).astype(np.float32), (1 + 0.1 * rng.normal(size=dim)).astype(np.float32), inv_freq(rotary)
    turn = A.QkNormRope(dim, rotary, style, dev(f), dev(wq), dev(wk))
    t, err = dev(x), error_word()
    q_out = torch.full((41, hq, dim), 3.0, dtype=t.dtype, device="cuda")
    A.qk_norm_rope_append(turn, cache, batch, t[:, :hq], t[:, hq:hq + heads], t[:, hq + heads:], dev(pos), q_out, err)
    assert int(err) == 0 and (q_out[39:] == 3).all()
    check_turned(q_out[:39].cpu().numpy(), R.turned(x[:39, :hq], wq, pos[:39], f, rotary, style, 1e-6), dtype)
    want = R.turned(x[:39, hq:hq + heads], wk, pos[:39], f, rotary, style, 1e-6)
    before = p.data.copy()
    for s in range(4):
        for j in range(counts[s]):
            p.put(s, lengths[s] + j, want[off[s] + j], x[off[s] + j, hq + heads:].astype(np.float64))
    got = cache.pages.cpu().numpy()
    # both sides round values of 64 bits that differ in their last places: a code or scale differs only where one lies within 2^-40 of a border
    assert np.array_equal(got, p.data), int((got != p.data).sum())
    assert not np.array_equal(got, before)


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("dim,page,heads", [(64, 16, 2), (128, 64, 8), (256, 32, 1)])
def test_keep_moves_the_accepted_slots(type_, dim, page, heads):
    rng = np.random.default_rng(dim)
    counts, lengths = [24, 64, 1, 7, 5], [11, 33, 0, 16, 60]
    accepted = [[0, 1, 5, 6, 23], sorted(rng.choice(64, 40, replace=False)), [0], [], [4]]
    p = R.Pages(rng, type_, page, heads, dim, [a + b for a, b in zip(counts, lengths)])
    for s in range(5):
        for j in range(counts[s]):
            p.put(s, lengths[s] + j, rng.normal(size=(heads, dim)), rng.normal(size=(heads, dim)))
    cache, (batch, off) = make_cache(p), make_batch(counts, lengths)
    acc = np.full(batch.rows, 77, np.uint32)
    for s, a in enumerate(accepted):
        acc[off[s]:off[s] + len(a)] = a
    err = error_word()
    A.kv_cache_keep(cache, batch, dev(acc), dev(np.array([len(a) for a in accepted], np.uint32)), err)
    assert int(err) == 0
    old = {(s, a): p.get(s, lengths[s] + a) for s in range(5) for a in accepted[s]}
    for s, path in enumerate(accepted):
        for j, a in enumerate(path):
            t0, t1 = (lengths[s] + a) % 16, (lengths[s] + j) % 16
            for h in range(heads):      # bit for bit, scales too
                for part, src, at in zip(p.part(s, lengths[s] + j, h), [x.copy() for x in saved(p, old, s, a, h, lengths)], (p.k_at, p.v_at)):
                    for o in range(1 if type_ == "q8_0" else 2):
                        part[at[t1] + o] = src[at[t0] + o]
                    if type_ == "q8_0":
                        for o in range(2):
                            part[p.scale_at[t1] + o] = src[p.scale_at[t0] + o]
    assert np.array_equal(cache.pages.cpu().numpy(), p.data)


def saved(p, old, s, a, h, lengths):
    """The parts of a source slot. Destinations are filled in ascending order and never above their source, so it still holds what it did."""
    k, v = p.get(s, lengths[s] + a)
    assert np.array_equal(k, old[s, a][0]) and np.array_equal(v, old[s, a][1])
    return p.part(s, lengths[s] + a, h)


def test_keep_refuses_paths_that_are_none():
    rng = np.random.default_rng(0)
    p = R.Pages(rng, "q8_0", 16, 2, 64, [20, 20, 20, 20])
    cache, (batch, off) = make_cache(p), make_batch([8, 8, 8, 8], [4, 4, 4, 4])
    for path, n in (([1, 1], 2), ([3, 2], 2), ([8], 1), ([0, 1, 2, 3, 4, 5, 6, 7, 8], 9)):
        acc = np.zeros(32, np.uint32)
        acc[8:8 + min(8, len(path))] = path[:8]
        acc[16:18] = [0, 1]     # its neighbour's path is the identity
        err = error_word()
        A.kv_cache_keep(cache, batch, dev(acc), dev(np.array([0, n, 2, 0], np.uint32)), err)
        assert int(err) == capi.ERR_INDEX and np.array_equal(cache.pages.cpu().numpy(), p.data), path


# ---- attention -------------------------------------------------------------------------------------------------------------------
class Step:
    """A batch with a filled cache. Slots that nothing wrote hold NaN (scales and binary16 values of all ones)."""

    def __init__(self, seed, type_, dim, page, heads, group, counts, lengths, dtype, tree, pad_rows=0, grow=0.3):
        rng = np.random.default_rng(seed)
        self.counts, self.lengths, self.dtype, self.heads, self.hq, self.dim = counts, lengths, dtype, heads, heads * group, dim
        total = [a + b for a, b in zip(counts, lengths)]
        self.p = p = R.Pages(rng, type_, page, heads, dim, total, fill=255)
        self.k, self.v = [], []
        for s, n in enumerate(total):
            x, y = rng.normal(size=(n, heads, dim)), rng.normal(size=(n, heads, dim))
            x[:n // 2] *= 1 + grow      # later maxima are not the first ones
            for j in range(n):
                p.put(s, j, x[j], y[j])
            self.k.append(R.cached(x, type_))
            self.v.append(R.cached(y, type_))
        off = np.concatenate([[0], np.cumsum(counts)])
        self.off, self.rows = off, int(off[-1])
        self.q = rng.normal(size=(self.rows + pad_rows, self.hq, dim)).astype(NP[dtype])
        self.mask = None
        if tree:
            self.mask = rng.integers(0, 1 << 63, self.rows + pad_rows, dtype=np.uint64) | (rng.integers(0, 2, self.rows + pad_rows).astype(np.uint64) << np.uint64(63))
        self.scale = 1.0 / np.sqrt(dim)
        self.batch, _ = make_batch(counts, lengths, rows=self.rows + pad_rows)
        self.most = max(1, max(counts))

    def visible(self, s, j):
        L, T = self.lengths[s], self.counts[s]
        w = (2 << j) - 1 if self.mask is None else int(self.mask[self.off[s] + j])
        return np.array([True] * L + [bool(w >> i & 1) for i in range(T)], bool)

    def run(self, cache=None, scratch=None, err=None, q=None, most=None):
        cache = cache or make_cache(self.p)
        q = dev(self.q) if q is None else q
        out = torch.full_like(q.contiguous(), 11.0)
        err = error_word() if err is None else err
        A.tree_attention(cache, self.batch, q, out, None if self.mask is None else dev(self.mask), most or self.most, self.scale,
                         A.tree_attention_scratch() if scratch is None else scratch, err)
        return out, int(err)

    def check(self, out, skip=()):
        out = out.cpu().numpy().astype(np.float64)
        assert (out[self.rows:] == 11).all()
        num = den = 0.0
        for s in range(len(self.counts)):
            for j in range(self.counts[s]):
                if s in skip:
                    continue
                r, vis = self.off[s] + j, self.visible(s, j)
                want, spread, vmax = R.attended(self.q[r], self.k[s], self.v[s], vis, self.scale)
                if not vis.any():
                    assert (out[r] == 0).all()
                    continue
                e = ((self.dim + 8) * U32 + (U16 if self.dtype == "f16" else 0)) * spread
                tol = vmax * (4 * e + (4 * U16 if self.dtype == "f16" else (len(vis) + 64) * U32)) + (U16 * np.abs(want) if self.dtype == "f16" else 0)
                d = np.abs(out[r] - want)
                assert (d <= tol).all(), (s, j, float(d.max()), float(np.max(tol)))
                num, den = num + float((d * d).sum()), den + float((want * want).sum())
        assert den == 0 or np.sqrt(num / den) <= (2e-3 if self.dtype == "f16" else 5e-6), np.sqrt(num / den)


CONTEXTS = [([1], [0]), ([1], [15]), ([1], [16]), ([1], [31]), ([2], [127]), ([1], [700]), ([1, 0, 3, 8], [33, 5, 0, 64]), ([64, 1], [90, 300]), ([5] * 9, [1, 17, 40, 0, 63, 64, 65, 128, 200])]


@pytest.mark.parametrize("shape", range(len(CONTEXTS)))
@pytest.mark.parametrize("type_,dim,page,heads,group", [("q8_0", 128, 64, 2, 4), ("q8_0", 64, 16, 3, 1), ("q8_0", 256, 32, 1, 8), ("f16", 128, 16, 1, 3), ("f16", 64, 256, 2, 8),
                                                        ("f16", 256, 64, 2, 2)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("tree", [False, True])
def test_attention(shape, type_, dim, page, heads, group, dtype, tree):
    counts, lengths = CONTEXTS[shape]
    s = Step(shape * 31 + dim, type_, dim, page, heads, group, counts, lengths, dtype, tree, pad_rows=shape % 3)
    out, err = s.run()
    assert err == 0
    s.check(out)


@pytest.mark.parametrize("type_,dim,heads,group,counts,lengths", [("q8_0", 128, 1, 16, [40], [2500]), ("q8_0", 128, 2, 4, [30, 64, 33], [1300, 70, 0]), ("q8_0", 64, 2, 12, [11, 22], [640, 513]),
                                                                  ("q8_0", 256, 1, 6, [64, 25], [333, 1024]), ("f16", 128, 2, 8, [64, 17], [1000, 129]), ("f16", 64, 1, 64, [5, 64], [200, 77]),
                                                                  ("f16", 256, 1, 32, [7], [999])])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_many_rows_per_head(type_, dim, heads, group, counts, lengths, dtype, tree):
    s = Step(7, type_, dim, 64, heads, group, counts, lengths, dtype, tree)
    out, err = s.run()
    assert err == 0
    s.check(out)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("group", [2, 16])
def test_rows_that_see_nothing_and_slots_that_hold_nothing(dtype, type_, group):
    """Words of zero, contexts of zero, and drafted slots of NaN or infinity that some rows see and others do not."""
    s = Step(3, type_, 128, 16, 2, group, [6, 6, 6], [0, 40, 0], dtype, True)
    s.mask[:] = np.arange(18, dtype=np.uint64) % 5
    s.mask[6:12] |= np.uint64(0xffffffffffffffc0)      # bits behind the sequence's rows say nothing
    s.p.poke_scale(1, 40 + 5, np.nan)                  # token 5: no row sees it
    s.p.poke_scale(0, 4, np.inf, which=(1,))
    out, err = s.run()
    assert err == 0
    s.check(out)
    s.p.poke_scale(2, 1, np.nan, which=(1,))           # token 1 of sequence 2: rows whose word has bit 1
    out, err = s.run()
    assert err == capi.ERR_NONFINITE
    s.check(out, skip=(2,))
    got = out.cpu().numpy().astype(np.float64)
    for j in range(6):
        if int(s.mask[12 + j]) & 2:
            assert (got[12 + j] == 0).all()
        else:
            want, _, _ = R.attended(s.q[12 + j], s.k[2], s.v[2], s.visible(2, j), s.scale)
            assert np.abs(got[12 + j] - want).max() <= 0.02 * max(1.0, np.abs(want).max())


def test_large_scores_and_large_values():
    """Scores far apart (weights of exactly one and zero), values near binary16's limits and far below one."""
    for dtype in ("f32", "f16"):
        for type_ in ("q8_0", "f16"):
            for at in (2e4, 1e-4):
                s = Step(5, type_, 128, 16, 1, 4, [4], [90], dtype, False)
                for j in range(94):
                    k, v = s.k[0][j] * 30, s.v[0][j] * (at / 6)
                    s.p.put(0, j, k, v)
                    s.k[0][j], s.v[0][j] = R.cached(k, type_), R.cached(v, type_)
                out, err = s.run()
                assert err == 0
                got = out.cpu().numpy().astype(np.float64)
                for j in range(4):
                    want, spread, vmax = R.attended(s.q[j], s.k[0], s.v[0], s.visible(0, j), s.scale)
                    e = (136 * U32 + (U16 if dtype == "f16" else 0)) * spread
                    tol = vmax * (4 * e + (4 * U16 if dtype == "f16" else 160 * U32)) + (U16 * np.abs(want) + 2.0 ** -25 if dtype == "f16" else 0)
                    assert (np.abs(got[j] - want) <= tol).all(), (dtype, type_, at)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("group", [2, 16])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-12])
def test_scales_of_zero_below_zero_and_close_to_it(dtype, group, scale):
    s = Step(13, "q8_0", 128, 16, 2, group, [3, 2], [37, 0], dtype, True)
    s.mask[1] = 0
    s.scale = scale
    out, err = s.run()
    assert err == 0
    s.check(out)


def test_sequences_out_of_range_are_zeros_and_leave_the_others():
    s = Step(9, "q8_0", 128, 16, 2, 4, [3, 9, 4, 2], [50, 20, 70, 8], "f16", False)
    out, err = s.run(most=8)                           # sequence 1 has more rows than the call says
    assert err == capi.ERR_INDEX and (out[3:12] == 0).all()
    s.check(out, skip=(1,))
    s.p.table[2, 2] = 0x7fffffff                       # a page that does not exist
    out, err = s.run()
    assert err & capi.ERR_INDEX and (out[12:16] == 0).all()
    s.check(out, skip=(2,))
    s.batch.lengths[3] = 5000                          # slots that the table does not hold
    out, err = s.run()
    assert err & capi.ERR_INDEX and (out[16:18] == 0).all() and (out[12:16] == 0).all()
    s.check(out, skip=(2, 3))


def test_strided_rows_other_streams_and_repeats():
    s = Step(11, "q8_0", 128, 32, 2, 8, [4, 1, 16], [500, 900, 40], "f16", True)
    cache, scratch = make_cache(s.p), A.tree_attention_scratch()
    out, err = s.run(cache, scratch)
    assert err == 0
    s.check(out)
    wide = torch.zeros(s.rows, s.hq + 5, 128, dtype=torch.float16, device="cuda")
    wide[:, 2:2 + s.hq] = dev(s.q)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(5):                             # the workspace is left as the next call wants it; the same bits every time
            again, err = s.run(cache, scratch, q=wide[:, 2:2 + s.hq])
            assert err == 0 and torch.equal(again, out)
    stream.synchronize()


def test_captured_step_follows_its_batch():
    """append, attention and keep in one graph; lengths, tokens and tree change between replays."""
    dim, heads, hq, T, page = 128, 2, 8, 5, 16
    rng = np.random.default_rng(21)
    p = R.Pages(rng, "q8_0", page, heads, dim, [400, 400], fill=255)
    cache, scratch, err = make_cache(p), A.tree_attention_scratch(), error_word()
    batch, off = make_batch([T, T], [0, 0])
    q, out = torch.zeros(2 * T, hq, dim, device="cuda"), torch.zeros(2 * T, hq, dim, device="cuda")
    k, v = torch.zeros(2 * T, heads, dim, device="cuda"), torch.zeros(2 * T, heads, dim, device="cuda")
    mask, acc, cnt = (torch.zeros(2 * T, dtype=torch.int64, device="cuda"), torch.zeros(2 * T, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))

    def step():
        A.kv_cache_append(cache, batch, k, v, err)
        A.tree_attention(cache, batch, q, out, mask, T, dim ** -0.5, scratch, err)
        A.kv_cache_keep(cache, batch, acc, cnt, err)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    kept = [([], []), ([], [])]
    length = [0, 0]
    for turn in range(40):
        hk, hv = rng.normal(size=(2 * T, heads, dim)).astype(np.float32), rng.normal(size=(2 * T, heads, dim)).astype(np.float32)
        hqv = rng.normal(size=(2 * T, hq, dim)).astype(np.float32)
        words = rng.integers(0, 32, 2 * T).astype(np.int64)
        paths = [sorted(rng.choice(T, rng.integers(0, T + 1), replace=False)) for _ in range(2)]
        hacc = np.zeros(2 * T, np.int32)
        for s in range(2):
            hacc[s * T:s * T + len(paths[s])] = paths[s]
        for t, h in ((k, hk), (v, hv), (q, hqv), (mask, words), (acc, hacc), (cnt, np.array([len(x) for x in paths], np.int32)), (batch.lengths, np.array(length, np.int32))):
            t.copy_(torch.from_numpy(h))
        graph.replay()
        got = out.cpu().numpy().astype(np.float64)
        assert int(err) == 0
        for s in range(2):
            ck = np.array(kept[s][0] + list(R.cached(hk[s * T:s * T + T], "q8_0"))).reshape(-1, heads, dim)
            cv = np.array(kept[s][1] + list(R.cached(hv[s * T:s * T + T], "q8_0"))).reshape(-1, heads, dim)
            for j in range(T):
                vis = np.array([True] * length[s] + [bool(int(words[s * T + j]) >> i & 1) for i in range(T)], bool)
                want, spread, vmax = R.attended(hqv[s * T + j], ck, cv, vis, dim ** -0.5)
                assert np.abs(got[s * T + j] - want).max() <= vmax * (4 * 136 * U32 * spread + (len(vis) + 64) * U32)
            for a in paths[s]:
                kept[s][0].append(ck[length[s] + a])
                kept[s][1].append(cv[length[s] + a])
            length[s] += len(paths[s])


def test_pages_behind_four_gigabytes():
    """Byte offsets of a page that do not fit 32 bits."""
    dim, heads, page = 128, 8, 256
    stride = capi.lib().tsp_kv_page_bytes(capi.TYPE_Q8_0, page, heads, dim)
    pages = (5 << 30) // stride
    pool = torch.empty(pages, stride, dtype=torch.uint8, device="cuda")
    table = np.array([[pages - 1, 0], [pages - 2, pages // 2]], np.uint32)
    cache = A.KvCache(pool, dev(table), page, heads, dim, "q8_0")
    counts, lengths = [300, 280], [0, 0]
    batch, off = make_batch(counts, lengths)
    rng = np.random.default_rng(0)
    k, v = (rng.normal(size=(580, heads, dim)).astype(np.float32) for _ in range(2))
    err, ko, vo = error_word(), torch.empty(580, heads, dim, device="cuda"), torch.empty(580, heads, dim, device="cuda")
    A.kv_cache_append(cache, batch, dev(k), dev(v), err)
    A.kv_cache_read(cache, batch, ko, vo, err)
    assert np.array_equal(ko.cpu().numpy(), R.cached(k, "q8_0").astype(np.float32)) and np.array_equal(vo.cpu().numpy(), R.cached(v, "q8_0").astype(np.float32))
    q = rng.normal(size=(2, 16, dim)).astype(np.float32)
    out = torch.empty(2, 16, dim, device="cuda")
    one, _ = make_batch([1, 1], [299, 279])
    A.tree_attention(cache, one, dev(q), out, None, 1, dim ** -0.5, A.tree_attention_scratch(), err)
    assert int(err) == 0
    for s in range(2):
        ck, cv = R.cached(k[off[s]:off[s + 1]], "q8_0"), R.cached(v[off[s]:off[s + 1]], "q8_0")
        want, spread, vmax = R.attended(q[s], ck, cv, np.ones(counts[s], bool), dim ** -0.5)
        assert np.abs(out[s].cpu().numpy() - want).max() <= vmax * (4 * 136 * U32 * spread + (counts[s] + 64) * U32)


@pytest.mark.parametrize("type_,dim,heads,group,counts,lengths", [("q8_0", 128, 8, 4, [17, 32], [9000, 3001]), ("q8_0", 128, 4, 4, [64], [30011]), ("f16", 128, 4, 8, [5, 33, 2], [12007, 4095, 64]),
                                                                  ("q8_0", 64, 8, 8, [9], [20000]), ("f16", 64, 8, 3, [6, 21], [16000, 9999]), ("q8_0", 256, 4, 2, [4, 1], [14000, 8000]),
                                                                  ("q8_0", 128, 8, 1, [1] * 24, [100 * i for i in range(24)]), ("f16", 128, 2, 6, [2], [40000])])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_long_runs(type_, dim, heads, group, counts, lengths, dtype):
    """Contexts that give every block more units than its stages hold, of several items or of one; the cache is written and read back by its own
    operators, and torch in 64 bits attends over what it holds."""
    g = torch.Generator(device="cuda").manual_seed(dim + len(counts))
    page, total = 64, [a + b for a, b in zip(counts, lengths)]
    need = [-(-n // page) for n in total]
    table = np.full((len(total), max(need)), 0xffffffff, np.uint32)
    order, at = np.random.default_rng(1).permutation(sum(need) + 1), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    pool = torch.full((sum(need) + 1, A.page_bytes(type_, page, heads, dim)), 255, dtype=torch.uint8, device="cuda")
    cache, err = A.KvCache(pool, dev(table), page, heads, dim, type_), error_word()
    everything, off = make_batch(total, [0] * len(total))
    k, v = (torch.randn(sum(total), heads, dim, generator=g, device="cuda") for _ in range(2))
    A.kv_cache_append(cache, everything, k, v, err)
    A.kv_cache_read(cache, everything, k, v, err)
    rows = sum(counts)
    q = torch.randn(rows, heads * group, dim, generator=g, device="cuda").to(torch.float32 if dtype == "f32" else torch.float16)
    batch, first = make_batch(counts, lengths)
    out, scratch = torch.empty_like(q), A.tree_attention_scratch()
    for _ in range(3):
        out.fill_(11)
        A.tree_attention(cache, batch, q, out, None, max(counts), dim ** -0.5, scratch, err)
    assert int(err) == 0
    num = den = 0.0
    for s in range(len(counts)):
        n, L = counts[s], lengths[s]
        kk, vv = (x[off[s]:off[s + 1]].double().permute(1, 0, 2).repeat_interleave(group, 0) for x in (k, v))
        x = q[first[s]:first[s + 1]].double().permute(1, 0, 2) @ kk.transpose(1, 2) * dim ** -0.5
        visible = torch.arange(L + n, device="cuda")[None] <= L + torch.arange(n, device="cuda")[:, None]
        want = (torch.softmax(x.masked_fill(~visible, -np.inf), -1) @ vv).permute(1, 0, 2)
        d = out[first[s]:first[s + 1]].double() - want
        num, den = num + float((d * d).sum()), den + float((want * want).sum())
    assert np.sqrt(num / den) <= (2e-3 if dtype == "f16" else 5e-6)


# ---- more than 48 binary16 rows per key / value head: the tiles of 128 rows, at the same edges

@pytest.mark.parametrize("type_,dim", [("q8_0", 128), ("q8_0", 64), ("f16", 128), ("f16", 64)])
@pytest.mark.parametrize("rows", [47, 48, 49, 64])
def test_rows_at_the_change_of_tiles(type_, dim, rows):
    s = Step(rows + dim, type_, dim, 16, 2, 1, [rows, 3], [200, 1027], "f16", True)
    out, err = s.run()
    assert err == 0
    s.check(out)


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-12])
def test_wide_tiles_scales(type_, dim, scale):
    s = Step(17, type_, dim, 16, 2, 16, [5, 2], [237, 0], "f16", True)
    s.mask[1] = 0
    s.scale = scale
    out, err = s.run()
    assert err == 0
    s.check(out)


@pytest.mark.parametrize("dim", [64, 128])
def test_wide_tiles_sequences_out_of_range(dim):
    s = Step(19, "q8_0", dim, 16, 2, 4, [3, 40, 20, 2], [50, 20, 170, 8], "f16", False)
    out, err = s.run(most=32)                          # sequence 1 has more rows than the call says
    assert err == capi.ERR_INDEX and (out[3:43] == 0).all()
    s.check(out, skip=(1,))
    s.p.table[2, 2] = 0x7fffffff                       # a page that does not exist
    out, err = s.run()
    assert err & capi.ERR_INDEX and (out[43:63] == 0).all()
    s.check(out, skip=(2,))
    s.batch.lengths[3] = 5000                          # slots that the table does not hold
    out, err = s.run()
    assert err & capi.ERR_INDEX and (out[63:65] == 0).all() and (out[43:63] == 0).all()
    s.check(out, skip=(2, 3))


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("at", [2e4, 1e-4])
def test_wide_tiles_large_scores_and_values(type_, at):
    """Scores far apart, values near binary16's limits and far below one; a scale that grows and falls from slot to slot."""
    s = Step(23, type_, 128, 16, 1, 4, [16], [190], "f16", False)
    for j in range(206):
        k, v = s.k[0][j] * (30 if j % 3 else 0.01), s.v[0][j] * (at / 6) * (1 if j % 5 else 1 / 64)
        s.p.put(0, j, k, v)
        s.k[0][j], s.v[0][j] = R.cached(k, type_), R.cached(v, type_)
    out, err = s.run()
    assert err == 0
    got = out.cpu().numpy().astype(np.float64)
    for j in range(16):
        want, spread, vmax = R.attended(s.q[j], s.k[0], s.v[0], s.visible(0, j), s.scale)
        e = (136 * U32 + U16) * spread
        # weights, the low parts' and the result's rounding; 2^-25: half of binary16's smallest step
        tol = vmax * (4 * e + 4 * U16) + U16 * np.abs(want) + 2.0 ** -25
        assert (np.abs(got[j] - want) <= tol).all(), (type_, at, j)


# ---- the cache write's other splits: many sequences (a warp for a whole head's values), more rows than two blocks an SM (four slots a key block)

@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("counts", [[1] * 250, [1, 0, 2] * 133, [90, 7, 0, 260]])
def test_append_of_many_rows_or_sequences(type_, counts):
    dim, heads, page = 128, 8, 16
    lengths = [(5 * i) % 23 for i in range(len(counts))]
    rng = np.random.default_rng(len(counts))
    p = R.Pages(rng, type_, page, heads, dim, [a + b for a, b in zip(counts, lengths)])
    cache, (batch, off) = make_cache(p), make_batch(counts, lengths, rows=sum(counts) + 2)
    k, v = (rng.normal(size=(batch.rows, heads, dim)).astype(np.float32) for _ in range(2))
    k[3, 1, 7] = np.inf                                # one head of one row: zeros
    v[5, 2, 9] = np.nan
    err = error_word()
    A.kv_cache_append(cache, batch, dev(k), dev(v), err)
    assert int(err) == capi.ERR_NONFINITE
    k[3, 1], v[5, 2] = 0, 0
    for s in range(len(counts)):
        for j in range(counts[s]):
            p.put(s, lengths[s] + j, k[off[s] + j].astype(np.float64), v[off[s] + j].astype(np.float64))
    assert np.array_equal(cache.pages.cpu().numpy(), p.data)


@pytest.mark.parametrize("type_", ["q8_0", "f16"])
@pytest.mark.parametrize("dim,rotary,style,dtype", [(64, 64, "pairs", "f16"), (128, 128, "halves", "f32"), (256, 128, "halves", "f32")])
def test_fused_norm_rotation_and_append_of_many_rows(type_, dim, rotary, style, dtype):
    rng = np.random.default_rng(dim + 1)
    counts, lengths, heads, hq = [100, 0, 257, 1], [9, 3, 14, 0], 2, 4
    rows = sum(counts)
    p = R.Pages(rng, type_, 64, heads, dim, [a + b for a, b in zip(counts, lengths)])
    cache, (batch, off) = make_cache(p), make_batch(counts, lengths, rows=rows + 3)
    x = rng.normal(size=(rows + 3, hq + 2 * heads, dim)).astype(NP[dtype])
    pos = rng.integers(0, 20000, rows + 3).astype(np.uint32)
    wq, wk, f = (1 + 0.1 * rng.normal(size=dim)).astype(np.float32), (1 + 0.1 * rng.normal(size=dim)).astype(np.float32), inv_freq(rotary)
    t, err = dev(x), error_word()
    q_out = torch.full((rows + 3, hq, dim), 3.0, dtype=t.dtype, device="cuda")
    A.qk_norm_rope_append(A.QkNormRope(dim, rotary, style, dev(f), dev(wq), dev(wk)), cache, batch, t[:, :hq], t[:, hq:hq + heads], t[:, hq + heads:], dev(pos), q_out, err)
    assert int(err) == 0 and (q_out[rows:] == 3).all()
    check_turned(q_out[:rows].cpu().numpy(), R.turned(x[:rows, :hq], wq, pos[:rows], f, rotary, style, 1e-6), dtype)
    want = R.turned(x[:rows, hq:hq + heads], wk, pos[:rows], f, rotary, style, 1e-6)
    for s in range(4):
        for j in range(counts[s]):
            p.put(s, lengths[s] + j, want[off[s] + j], x[off[s] + j, hq + heads:].astype(np.float64))
    assert np.array_equal(cache.pages.cpu().numpy(), p.data)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_stages_of_halves_without_a_page(dtype):
    """256 dims of binary16: keys and values arrive one after the other; a unit without a page passes both."""
    s = Step(29, "f16", 256, 16, 2, 3, [5, 9, 2], [700, 350, 40], dtype, True)
    out, err = s.run()
    assert err == 0
    s.check(out)
    s.p.table[1, 3] = 0x7fffffff
    out, err = s.run()
    assert err & capi.ERR_INDEX and (out[5:14] == 0).all()
    s.check(out, skip=(1,))


# ---- calls that the documentation allows: the most sequences, none at all, two at once

@pytest.mark.parametrize("group,dtype", [(2, "f32"), (4, "f16"), (64, "f16")])
def test_the_most_sequences(group, dtype):
    n = capi.KV_MAX_SEQUENCES
    s = Step(31, "q8_0", 64, 16, 1, group, [1] * (n - 3) + [0, 2, 3], [i % 19 for i in range(n)], dtype, True)
    out, err = s.run()
    assert err == 0
    s.check(out)


@pytest.mark.parametrize("group,dtype", [(2, "f32"), (32, "f16")])
def test_a_step_without_rows(group, dtype):
    """Three sequences, none with a token, in buffers of four rows: nothing is touched."""
    s = Step(33, "q8_0", 128, 16, 2, group, [0, 0, 0], [5, 0, 40], dtype, False, pad_rows=4)
    cache = make_cache(s.p)
    before, err = cache.pages.clone(), error_word()
    out, code = s.run(cache, most=4)
    assert code == 0 and (out == 11).all()
    k = torch.ones(s.batch.rows, 2, 128, device="cuda")
    A.kv_cache_append(cache, s.batch, k, k, err)
    A.kv_cache_keep(cache, s.batch, torch.zeros(s.batch.rows, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), err)
    q = torch.full((s.batch.rows, 4, 128), 2.0, device="cuda")
    A.qk_norm_rope_append(A.QkNormRope(128, 0, "halves", None), cache, s.batch, q, k, k, torch.zeros(s.batch.rows, dtype=torch.int32, device="cuda"), q, err)
    A.kv_cache_read(cache, s.batch, k, None, err)
    assert int(err) == 0 and torch.equal(cache.pages, before) and (k == 1).all() and (q == 2).all()


@pytest.mark.parametrize("group", [4, 32])
def test_two_captured_calls_at_once_with_a_workspace_each(group):
    steps = [Step(seed, "q8_0", 128, 32, 2, group, [3, 2], [1900, 700], "f16", True) for seed in (35, 36)]
    wants, graphs, outs, errs, keep = [], [], [], [], []
    for s in steps:
        want, err = s.run()
        assert err == 0
        s.check(want)
        wants.append(want)
        cache, q, mask, scratch, err, out = make_cache(s.p), dev(s.q), dev(s.mask), A.tree_attention_scratch(), error_word(), torch.full_like(want, 11.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(8):
                A.tree_attention(cache, s.batch, q, out, mask, s.most, s.scale, scratch, err)
        graphs.append(graph); outs.append(out); errs.append(err); keep.append((cache, q, mask, scratch))
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(6):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for want, out, err in zip(wants, outs, errs):
        assert int(err) == 0 and torch.equal(out, want)
