"""The attention operators where buffers, scales and sizes meet their edges, against 64-bit restatements (attention_ref.py). Tolerances are those of
test_gpu_attention.py, derived there."""
import os
import subprocess

import numpy as np
import pytest

import attention_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import U16, U32, Step, check_turned, dev, error_word, make_cache  # noqa: E402
from tokspur_public_b200 import attention as A  # noqa: E402
from tokspur_public_b200 import capi  # noqa: E402


@pytest.mark.parametrize("type_,dim,group,dtype", [("q8_0", 128, 4, "f16"), ("q8_0", 128, 4, "f32"), ("f16", 256, 8, "f32"), ("f16", 64, 8, "f16"), ("q8_0", 128, 32, "f16")])
def test_many_refills_give_the_same_bits(type_, dim, group, dtype):
    """Rings that go round dozens of times in every warp, 200 calls: a stage that is refilled under its reader shows as another result."""
    s = Step(41, type_, dim, 64, 4, group, [2, 1], [9000, 7000], dtype, False)
    cache, scratch, err, q = make_cache(s.p), A.tree_attention_scratch(), error_word(), dev(s.q)
    want, code = s.run(cache, scratch)
    assert code == 0
    s.check(want)
    outs = [torch.empty_like(want) for _ in range(20)]
    differing = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(10):
        for out in outs:
            A.tree_attention(cache, s.batch, q, out, None, s.most, s.scale, scratch, err)
        for out in outs:
            differing += (out != want).sum()
    assert int(differing) == 0 and int(err) == 0


# ---- slots that a row does not see: finite or not, large or not, they cost it nothing

def check_row(s, out, r, seq, j, k, v):
    """Step.check's bound for one row over the slots k, v of its sequence; returns the squares of error and value."""
    vis = s.visible(seq, j)
    want, spread, vmax = R.attended(s.q[r], k, v, vis, s.scale)
    e = ((s.dim + 8) * U32 + (U16 if s.dtype == "f16" else 0)) * spread
    tol = vmax * (4 * e + (4 * U16 if s.dtype == "f16" else (len(vis) + 64) * U32)) + (U16 * np.abs(want) + 2.0 ** -25 if s.dtype == "f16" else 0)
    d = np.abs(out[r] - want)
    assert (d <= tol).all(), (seq, j, float((d / tol).max()), float(d.max()))
    return float((d * d).sum()), float((want * want).sum())


def poked(s, hidden, which, value):
    """Rewrites the scales (binary16 cache: the values) of token `hidden[seq]` of every sequence's step."""
    for seq, token in enumerate(hidden):
        s.p.poke_scale(seq, s.lengths[seq] + token, value, which=which)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("type_,dim,group", [("q8_0", 128, 2), ("q8_0", 64, 3), ("q8_0", 256, 2), ("f16", 128, 2), ("q8_0", 128, 32), ("q8_0", 64, 32), ("f16", 64, 32)])
@pytest.mark.parametrize("which,value", [((1,), 6e4), ((1,), 512.0), ((0,), 6e4), ((0,), np.inf), ((0,), np.nan), ((1,), -np.inf), ((0, 1), 6e4)])
@pytest.mark.parametrize("small", [1.0, 2.0 ** -6])
def test_hidden_slots_cost_the_other_rows_nothing(dtype, type_, dim, group, which, value, small):
    """Token 1 of every step holds a scale (binary16: values) far above the others', or none that is finite; rows whose word hides it have the bounds of a
    step without it. The third step's tokens span units of both kernels, and units behind the token's own."""
    s = Step(43, type_, dim, 16, 2, group, [6, 12, 40], [0, 57, 300], dtype, True)
    if small != 1:                                     # the other slots' values and keys; the same scores
        s.q = (s.q.astype(np.float64) / small).astype(s.q.dtype)
        for seq in range(3):
            for j in range(len(s.k[seq])):
                k, v = s.k[seq][j] * small, s.v[seq][j] * small
                s.p.put(seq, j, k, v)
                s.k[seq][j], s.v[seq][j] = R.cached(k, type_), R.cached(v, type_)
    s.mask |= np.uint64(1)                             # a row of a short step sees something
    s.mask[::2] &= ~np.uint64(2)
    poked(s, [1, 1, 1], which, value)
    out, err = s.run()
    assert np.isfinite(value) or err == capi.ERR_NONFINITE
    got = out.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    num = den = 0.0
    for seq in range(3):
        for j in range(s.counts[seq]):
            r = s.off[seq] + j
            if not int(s.mask[r]) & 2:
                x, y = check_row(s, got, r, seq, j, s.k[seq], s.v[seq])
                num, den = num + x, den + y
    assert np.sqrt(num / den) <= (2e-3 if dtype == "f16" else 5e-6), np.sqrt(num / den)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("group", [2, 32])
@pytest.mark.parametrize("which,value", [((1,), 512.0), ((0,), 64.0), ((0, 1), 256.0)])
def test_rows_that_see_such_a_slot(dtype, group, which, value):
    """The rows on the other side, against sums over what the cache then holds (finite scales, results within binary16's range)."""
    s = Step(47, "q8_0", 128, 16, 2, group, [6, 12, 40], [0, 57, 300], dtype, True)
    s.mask |= np.uint64(3)
    for seq in range(3):                               # codes small enough that binary16 holds the results
        at = s.lengths[seq] + 1
        k, v = s.k[seq][at], np.clip(s.v[seq][at], -0.5, 0.5)
        s.p.put(seq, at, k, v)
    poked(s, [1, 1, 1], which, value)
    for seq in range(3):
        s.k[seq][s.lengths[seq] + 1], s.v[seq][s.lengths[seq] + 1] = s.p.get(seq, s.lengths[seq] + 1)
    out, err = s.run()
    got = out.cpu().numpy().astype(np.float64)
    limit = 65504 if dtype == "f16" else np.inf
    for seq in range(3):
        for j in range(s.counts[seq]):
            r = s.off[seq] + j
            want, _, _ = R.attended(s.q[r], s.k[seq], s.v[seq], s.visible(seq, j), s.scale)
            fits = [h for h in range(s.hq) if np.abs(want[h]).max() < 0.9 * limit]
            vis = s.visible(seq, j)
            for h in fits:
                w, spread, vmax = R.attended(s.q[r][h:h + 1], s.k[seq][:, h // group][:, None], s.v[seq][:, h // group][:, None], vis, s.scale)
                e = ((s.dim + 8) * U32 + (U16 if dtype == "f16" else 0)) * spread
                tol = vmax * (4 * e + (4 * U16 if dtype == "f16" else (len(vis) + 64) * U32)) + (U16 * np.abs(w[0]) + 2.0 ** -25 if dtype == "f16" else 0)
                assert (np.abs(got[r][h] - w[0]) <= tol).all(), (seq, j, h, float((np.abs(got[r][h] - w[0]) / tol).max()))


# ---- norm and rotation

def inv_freq(rotary):
    return (1e4 ** (-np.arange(rotary // 2) / max(1, rotary // 2))).astype(np.float32)


@pytest.mark.parametrize("dim,hq,hk", [(64, 1, 1), (64, 7, 2), (64, 3, 6), (128, 1, 1), (128, 7, 3), (256, 3, 2)])
@pytest.mark.parametrize("sides", ["q", "k", "none", "both"])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 700])
def test_norm_of_one_side_where_a_warp_holds_heads_of_both(dim, hq, hk, sides, dtype, rows):
    rng = np.random.default_rng(dim + hq)
    q, k = (rng.normal(size=(rows, h, dim)).astype(np.float32 if dtype == "f32" else np.float16) for h in (hq, hk))
    pos, f = rng.integers(0, 9000, rows).astype(np.uint32), inv_freq(dim)
    wq, wk = ((1 + 0.2 * rng.normal(size=dim)).astype(np.float32) if sides in (s, "both") else None for s in ("q", "k"))
    turn = A.QkNormRope(dim, dim, "halves", dev(f), None if wq is None else dev(wq), None if wk is None else dev(wk), eps=1e-5)
    qo, ko, err = torch.empty_like(dev(q)), torch.empty_like(dev(k)), error_word()
    A.qk_norm_rope(turn, dev(q), dev(k), dev(pos), qo, ko, err)
    assert int(err) == 0
    for x, w, o in ((q, wq, qo), (k, wk, ko)):
        check_turned(o.cpu().numpy(), R.turned(x, w, pos, f, dim, "halves", 1e-5), dtype)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-6])
@pytest.mark.parametrize("rows", [3, 600])
def test_norms_of_heads_whose_squares_leave_fp32(dim, eps, rows):
    """Finite heads around 1e19 and up (their squares overflow) and down to 1e-38 (they vanish); beside them heads of ordinary size, in the same warp."""
    rng = np.random.default_rng(dim)
    x = rng.normal(size=(rows, 7, dim))
    at = np.array([1.0, 1e19, 1e-20, 3e37, 1e-24, 1e-37, 1e30])
    x = (x * at[None, :, None]).astype(np.float32)
    x[1, 2] = 0
    x[1, 2, 5] = 1e-40                                 # one subnormal value
    if eps == 0:
        x[2, 4, :] = 0
        x[2, 4, 0] = -3e38                             # one value, near the largest
    pos, f, w = rng.integers(0, 9000, rows).astype(np.uint32), inv_freq(dim), (1 + 0.2 * rng.normal(size=dim)).astype(np.float32)
    t, err = dev(x), error_word()
    qo, ko = torch.empty_like(t[:, :4]), torch.empty_like(t[:, 4:])
    A.qk_norm_rope(A.QkNormRope(dim, dim, "halves", dev(f), dev(w), dev(w), eps=eps), t[:, :4], t[:, 4:], dev(pos), qo, ko, err)
    assert int(err) == 0
    want = R.turned(x, w, pos, f, dim, "halves", eps)
    got = np.concatenate([qo.cpu().numpy(), ko.cpu().numpy()], 1)
    # 2^-19 of the head's largest value as elsewhere; 2^-149: where values themselves are subnormal
    top = np.abs(want).max(-1, keepdims=True)
    assert (np.abs(got.astype(np.float64) - want) <= top * 2.0 ** -19 + 2.0 ** -149).all()


def test_the_key_in_the_cache_and_the_query_of_one_row_agree_on_large_heads():
    """The fused call: query rows normed in FP32, the same values as keys in 64 bits on their way into the cache."""
    dim = 128
    x = (np.random.default_rng(8).normal(size=(5, 3, dim)) * 1e19).astype(np.float32)
    p = R.Pages(np.random.default_rng(0), "f16", 16, 1, dim, [5])
    cache, err = make_cache(p), error_word()
    batch = A.KvBatch(dev(np.array([0, 5], np.uint32)), dev(np.zeros(1, np.uint32)), 5)
    t, q = dev(x), torch.empty(5, 1, dim, device="cuda")
    w, pos = np.ones(dim, np.float32), np.arange(5, dtype=np.uint32)
    A.qk_norm_rope_append(A.QkNormRope(dim, dim, "halves", dev(inv_freq(dim)), dev(w), dev(w)), cache, batch, t[:, :1], t[:, :1], dev(x[:, 2:] / np.float32(1e19)), dev(pos), q, err)
    k = torch.empty_like(q)
    A.kv_cache_read(cache, batch, k, None, err)
    assert int(err) == 0
    check_turned(q.cpu().numpy(), R.turned(x[:, :1], w, pos, inv_freq(dim), dim, "halves", 1e-6), "f32")
    check_turned(k.cpu().numpy(), R.turned(x[:, :1], w, pos, inv_freq(dim), dim, "halves", 1e-6), "f16")


@pytest.mark.parametrize("type_,dim,group", [("q8_0", 128, 4), ("f16", 64, 16), ("f16", 256, 2)])
@pytest.mark.parametrize("scale,at", [(1e-30, 1e29), (1e-37, 1e36), (-3e-34, 1e33), (1e-30, 1.0), (4e3, 1e-5), (1e30, 1e-31)])
def test_scales_far_from_one_with_rows_that_make_up_for_them(type_, dim, group, scale, at):
    """FP32 rows: any finite scale, and the scores are what they are."""
    s = Step(53, type_, dim, 16, 2, group, [5, 2], [200, 0], "f32", True)
    s.q = (s.q * np.float32(at)).astype(np.float32)
    s.scale = float(np.float32(scale))
    out, err = s.run()
    assert err == 0
    s.check(out)


# ---- the C++ host layer

def test_the_host_layer_refuses_before_it_launches():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    binary = os.path.join(root, "tokspur-public_b200", "native", "tests", "test_attention_refusals")
    if not os.path.exists(binary):
        subprocess.run(["make", "-s", "-C", os.path.dirname(os.path.dirname(binary))], check=True)
    r = subprocess.run([binary], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "attention refusal checks passed" in r.stdout


def test_rows_without_rotation_need_no_positions():
    x, w = np.random.default_rng(1).normal(size=(4, 3, 64)).astype(np.float32), np.ones(64, np.float32)
    out, err = torch.empty(4, 3, 64, device="cuda"), error_word()
    A.qk_norm_rope(A.QkNormRope(64, 0, "halves", None, dev(w)), dev(x), None, None, out, None, err)
    assert int(err) == 0
    check_turned(out.cpu().numpy(), R.turned(x, w, np.zeros(4), np.ones(1), 0, "halves", 1e-6), "f32")
