"""The attention half of a decode / verify step as cases that can be timed and compared: norm and rotation of query and key heads,
the paged key / value cache (quantised as it is written, read back, compacted after a verify) and the attention of drafted tokens
over it.

A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one pass: with `own` through the
library's public entry points, otherwise in elementary torch operations. Kinds:

  turn     `tsp_qk_norm_rope`: per-head norm and rotation of query and key rows.
  write    `tsp_qk_norm_rope_append`, then `tsp_kv_cache_read` of the same rows: a step's rows normed, rotated and quantised into
           the cache, and what the cache then holds of them.
  keep     `tsp_kv_cache_append` of drafted rows, `tsp_kv_cache_keep` of the accepted ones, `tsp_kv_cache_read` of the draft zone.
  read     `tsp_kv_cache_read` of whole sequences.
  attend   `tsp_tree_attention`: the drafted tokens of every sequence over its context and over each other.

A cache page holds `page_tokens` slots of every key / value head: [head][group of 16 slots][K values | K scales | V values | V scales].
Group of 16 slots, q8_0 (stored byte = code + 128, a binary16 scale per 32 dims):
  K values [64 dims][slot][8 dims of the first 32 | 8 of the second, four times over], V values [32 dims][8][4][4][4] with byte (g, t, i, e) =
  dim 8i + g of slot 2t + (e & 1) + 8 (e >> 1), scales [32 dims][slot].
f16: K values [32 dims][slot][32], V values [32 dims][2][8][4][2][4] with (m, g, t, i, e) = dim 8 (2m + i) + g of that slot; no scales.
"""
from __future__ import annotations

import math

import torch

own = False

GROUP = 16


# ---- cases -------------------------------------------------------------------------------------------------------------------
def _heads(q_heads=32, kv_heads=8, dim=128):
    return {"q_heads": q_heads, "kv_heads": kv_heads, "dim": dim}


def listed():
    return [
        # the few rows of one verify pass: bound by the launch
        {"name": "turn_8_f32", "kind": "turn", "rows": 8, "dtype": "f32", "style": "halves", "rotary": 128, "far": 1 << 20, **_heads()},
        # a prompt's rows
        {"name": "turn_4096_f16", "kind": "turn", "rows": 4096, "dtype": "f16", "style": "halves", "rotary": 128, "far": 32768, **_heads()},
        # a ragged batch of drafts written into the cache, FP32 rows as the host layer passes them, part of a head rotated
        {"name": "write_draft_f32", "kind": "write", "sequences": 6, "most": 8, "length": 5000, "dtype": "f32", "cache": "q8_0", "page": 64, "style": "halves",
         "rotary": 64, **_heads()},
        # three prompts
        {"name": "write_prompts_f16", "kind": "write", "sequences": 3, "most": 1500, "length": 0, "dtype": "f16", "cache": "q8_0", "page": 64, "style": "pairs",
         "rotary": 128, **_heads()},
        # the accepted path of one tree
        {"name": "keep_tree_f32", "kind": "keep", "sequences": 1, "most": 24, "length": 3001, "dtype": "f32", "cache": "q8_0", "page": 64, **_heads()},
        # a full batch of short drafts, pages that end inside a draft
        {"name": "keep_batch_f16", "kind": "keep", "sequences": 64, "most": 16, "length": 2000, "dtype": "f16", "cache": "q8_0", "page": 16, **_heads()},
        # long contexts as plain rows
        {"name": "read_long_f16", "kind": "read", "sequences": 2, "most": 32768, "dtype": "f16", "cache": "q8_0", "page": 64, **_heads()},
        # one user generating: the smallest call
        {"name": "attend_one", "kind": "attend", "sequences": 1, "most": 1, "length": 4096, "tree": False, "dtype": "f16", "cache": "q8_0", "page": 64, **_heads()},
        # a full decode batch of ragged contexts
        {"name": "attend_batch", "kind": "attend", "sequences": 64, "most": 1, "length": 8192, "tree": False, "dtype": "f16", "cache": "q8_0", "page": 64, **_heads()},
        # verify rows of a draft chain: FP32 rows, wide heads, a binary16 cache
        {"name": "attend_chain_f32", "kind": "attend", "sequences": 6, "most": 8, "length": 6000, "tree": False, "dtype": "f32", "cache": "f16", "page": 16,
         **_heads(16, 2, 256)},
        # drafted trees of a few users
        {"name": "attend_trees", "kind": "attend", "sequences": 4, "most": 32, "length": 20000, "tree": True, "dtype": "f16", "cache": "q8_0", "page": 64, **_heads()},
        # the widest tree over a long context
        {"name": "attend_long", "kind": "attend", "sequences": 1, "most": 64, "length": 131072, "tree": True, "dtype": "f16", "cache": "q8_0", "page": 256, **_heads()},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    kind = rng.choice(["turn", "write", "keep", "read", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    c = {"kind": kind, "dtype": rng.choice(["f16", "f32"]), **_heads(kv * rng.choice([1, 2, 3, 4, 6, 8]), kv, dim)}
    if kind in ("turn", "write"):
        c.update(style=rng.choice(["halves", "pairs"]), rotary=rng.choice([dim, dim, dim // 2, dim // 4]))
    if kind == "turn":
        c.update(rows=log(1, 4096), far=log(100, 1 << 20))
        return c
    c.update(cache=rng.choice(["q8_0", "q8_0", "f16"]), page=rng.choice([16, 32, 64, 128, 256]))
    if kind == "read":
        c.update(sequences=log(1, 32))
        c.update(most=log(1, 32768 // c["sequences"]))
    elif kind == "write":
        c.update(sequences=log(1, 64), length=log(1, 20000))
        c.update(most=log(1, max(2, 4096 // c["sequences"])))
    elif kind == "keep":
        c.update(sequences=log(1, 64), most=log(2, 64), length=log(1, 20000))
    else:
        c.update(sequences=log(1, 64), most=rng.choice([1, 1, log(2, 64), log(2, 16)]), tree=rng.choice([False, True]))
        rows, values = c["sequences"] * c["q_heads"] * max(1, c["most"] // 4), c["sequences"] * kv * dim
        c.update(length=log(1, max(2, min(65536, (1 << 24) // rows, (1 << 28) // values))))
    return c


def _counts(case):
    """Rows of every sequence: ragged between half of `most` (at least one) and `most`, the first sequence the fullest."""
    most, n = case["most"], case["sequences"]
    return [most if s == 0 else most - (s * 7919) % (most // 2 + 1) for s in range(n)]


def _lengths(case):
    """Slots of every sequence that were there before: ragged between an eighth of `length` and `length`."""
    full, n = case.get("length", 0), case["sequences"]
    return [full if s == 0 else full - (s * 104729) % (full - full // 8 + 1) for s in range(n)]


def _group_bytes(case):
    d = case["dim"]
    return 2 * GROUP * (d + d // 16) if case["cache"] == "q8_0" else 4 * GROUP * d


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d, hq, hk = case["dim"], case["q_heads"], case["kv_heads"]
    dt, dev = _dtype(case), "cuda"

    def normal(*shape, at=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * at).to(dt)

    s = {"case": case, "error": torch.zeros(1, dtype=torch.int32, device=dev)}
    if case["kind"] in ("turn", "write"):
        s["q_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
        s["k_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
        half = case["rotary"] // 2
        s["inv_freq"] = (1e6 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)).float()
    if case["kind"] == "turn":
        rows = case["rows"]
        s["q"], s["k"] = normal(rows, hq, d), normal(rows, hk, d, at=2.0)
        s["positions"] = torch.randint(0, case["far"], (rows,), generator=g, device=dev, dtype=torch.int32)
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s
    counts, lengths, page = _counts(case), _lengths(case), case["page"]
    n, rows = case["sequences"], sum(counts)
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=dev)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    per = max((l + c + page - 1) // page for l, c in zip(lengths, counts))
    pages = sum((l + c + page - 1) // page for l, c in zip(lengths, counts)) + 3
    # every sequence's pages lie in any order in the pool; entries behind a sequence's last page name no page
    ids = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    used = torch.tensor([(l + c + page - 1) // page for l, c in zip(lengths, counts)], device=dev)
    at = torch.cumsum(used, 0) - used
    col = torch.arange(per, device=dev)
    s["table"] = torch.where(col < used[:, None], ids[torch.clamp(at[:, None] + col, max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=dev)).contiguous()
    gb = _group_bytes(case)
    s["pages"] = torch.empty(pages, hk * (page // GROUP) * gb, dtype=torch.uint8, device=dev)
    groups = s["pages"].view(-1, gb)
    if case["cache"] == "f16":
        groups.view(torch.float16).copy_(torch.randn(groups.shape[0], gb // 2, generator=g, device=dev))
    else:
        # values of unit variance: codes of a normal block against its largest value, scales around that over 127
        half = gb // 2
        for part in (groups[:, :half], groups[:, half:]):
            codes = torch.randn(groups.shape[0], GROUP * d, generator=g, device=dev) * 50
            part[:, :GROUP * d] = (torch.clamp(torch.round(codes), -127, 127) + 128).to(torch.uint8)
            scales = ((0.7 + 0.6 * torch.rand(groups.shape[0], GROUP * d // 32, generator=g, device=dev)) / 50).half()
            part[:, GROUP * d:] = scales.view(torch.uint8)
    row = torch.arange(rows, device=dev)
    seq = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(counts, device=dev))
    node = row - s["offsets"][seq].long()
    if case["kind"] == "write":
        s["q"], s["k"], s["v"] = normal(rows, hq, d), normal(rows, hk, d, at=2.0), normal(rows, hk, d)
        s["positions"] = (s["lengths"][seq].long() + node).to(torch.int32)
        s["q_out"] = torch.empty_like(s["q"])
    if case["kind"] == "keep":
        s["k"], s["v"] = normal(rows, hk, d), normal(rows, hk, d)
        # an accepted path: about half of the nodes, ascending
        chosen = torch.rand(rows, generator=g, device=dev) < 0.5
        rank = torch.cumsum(chosen, 0) - chosen.long()
        before = rank[s["offsets"][:-1].long()]
        s["accepted"] = torch.zeros(rows, dtype=torch.int32, device=dev)
        s["accepted"][(s["offsets"][seq].long() + rank - before[seq])[chosen]] = node[chosen].to(torch.int32)
        s["counts"] = torch.zeros(n, dtype=torch.int32, device=dev).index_add_(0, seq, chosen.to(torch.int32))
    if case["kind"] in ("write", "keep", "read"):
        s["k_out"], s["v_out"] = torch.empty(rows, hk, d, dtype=dt, device=dev), torch.empty(rows, hk, d, dtype=dt, device=dev)
    if case["kind"] == "attend":
        s["q"], s["out"] = normal(rows, hq, d), torch.empty(rows, hq, d, dtype=dt, device=dev)
        if case["tree"]:
            # a tree drafted breadth first: a node's parent is an earlier node, its word holds its ancestors and itself
            parent = (torch.rand(rows, generator=g, device=dev) * node).long()
            word = torch.ones((), dtype=torch.int64, device=dev) << node
            up = torch.where(node > 0, s["offsets"][seq].long() + parent, row)
            for _ in range(6):
                word, up = word | word[up], up[up]
            s["mask"] = word
        else:
            s["mask"] = None
    return s


# ---- the plain form ----------------------------------------------------------------------------------------------------------
def _turned(x, weight, case, positions, inv_freq, dtype):
    """Norm and rotation of [rows, heads, dim] in `dtype`; the angles in 64 bits."""
    x = x.to(dtype)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.to(dtype)
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = torch.cos(angle).to(dtype)[:, None], torch.sin(angle).to(dtype)[:, None]
    r = case["rotary"]
    turned = y[..., :r]
    if case["style"] == "halves":
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, y[..., r:]], -1)


def _cached(x, case):
    """The values that the cache holds of rows [rows, heads, dim]: borders between two codes are looked at in 64 bits."""
    if case["cache"] == "f16":
        return x.half().float()
    blocks = x.double().unflatten(-1, (-1, 32))
    d16 = (blocks.abs().amax(-1, keepdim=True) / 127).float().half().double()
    code = torch.where(d16 > 0, torch.clamp(torch.round(blocks / torch.where(d16 > 0, d16, 1.0)), -127, 127), 0.0)
    return (code * d16).flatten(-2).float()


def _unpacked(groups, case):
    """[..., group bytes] of a cache -> K and V as FP32 [..., 16 slots, dim]."""
    d = case["dim"]
    lead = groups.shape[:-1]
    k, v = groups.split(groups.shape[-1] // 2, -1)
    if case["cache"] == "f16":
        k = k.contiguous().view(torch.float16).view(*lead, d // 32, GROUP, 32).float()
        v = v.contiguous().view(torch.float16).view(*lead, d // 32, 2, 8, 4, 2, 2, 2).float()   # b m g t i e1 e0
        n = len(lead)
        k = k.transpose(n, n + 1).flatten(n + 1)
        v = v.permute(*range(n), n + 5, n + 3, n + 6, n, n + 1, n + 4, n + 2)   # slot = (e1, t, e0), dim = (b, m, i, g)
        return k, v.flatten(n, n + 2).flatten(n + 1)
    n = len(lead)

    def parts(x):
        codes, scales = x.split([GROUP * d, GROUP * d // 16], -1)
        return codes.float() - 128, scales.contiguous().view(torch.float16).view(*lead, d // 32, GROUP).transpose(n, n + 1).float()
    kc, ks = parts(k)
    vc, vs = parts(v)
    kc = kc.view(*lead, d // 64, GROUP, 4, 2, 8).permute(*range(n), n + 1, n, n + 3, n + 2, n + 4)   # slot, dims (64, half, chunk, 8)
    vc = vc.view(*lead, d // 32, 8, 4, 4, 2, 2).permute(*range(n), n + 4, n + 2, n + 5, n, n + 3, n + 1)   # slot = (e1, t, e0), dim = (b, i, g)
    kc, vc = kc.flatten(n + 1), vc.flatten(n, n + 2).flatten(n + 1)
    return kc * ks.repeat_interleave(32, -1), vc * vs.repeat_interleave(32, -1)


def _dense(state):
    """K and V of every sequence's slots, FP32 [sequences, heads, slots, dim], and how many of them each sequence has; the others are zero."""
    case, table = state["case"], state["table"].long()
    counts = (state["offsets"][1:] - state["offsets"][:-1]).long()
    filled = state["lengths"].long() + counts
    taken = state["pages"][torch.clamp(table, min=0)].view(*table.shape, case["kv_heads"], case["page"] // GROUP, -1)
    k, v = _unpacked(taken.permute(0, 2, 1, 3, 4), case)                    # [s, h, page, group, 16, d]
    k, v = k.flatten(2, 4), v.flatten(2, 4)
    there = (torch.arange(k.shape[2], device=k.device) < filled[:, None])[:, None, :, None]
    return torch.where(there, k, 0.0), torch.where(there, v, 0.0), filled


def _rows_of(state):
    """Sequence and index in it of every row."""
    offsets = state["offsets"].long()
    row = torch.arange(_row_count(state["case"]), device=offsets.device)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    return seq, row - offsets[seq]


def _row_count(case):
    return sum(_counts(case))


def _attended(state):
    case = state["case"]
    hq, hk, d, most = case["q_heads"], case["kv_heads"], case["dim"], case["most"]
    k, v, filled = _dense(state)
    seq, node = _rows_of(state)
    n, slots = k.shape[0], k.shape[2]
    word = state["mask"] if state["mask"] is not None else torch.where(node >= 63, -1, (torch.ones_like(node) << (node + 1)) - 1)
    q = torch.zeros(n, most, hq, d, device=k.device)
    q[seq, node] = state["q"].float()
    seen = torch.zeros(n, most, dtype=torch.int64, device=k.device)
    seen[seq, node] = word
    slot = torch.arange(slots, device=k.device)
    draft = slot - state["lengths"].long()[:, None]                         # [s, slots]
    bit = (seen[:, :, None] >> torch.clamp(draft, 0, 63)[:, None]) & 1
    visible = (draft < 0)[:, None] | ((bit == 1) & (slot < filled[:, None])[:, None])       # [s, most, slots]
    q = q.view(n, most, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    scores = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    scores = scores.view(n, hk, most, -1, slots).masked_fill_(~visible[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp_(scores.sub_(torch.where(torch.isfinite(top), top, 0.0)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hk, -1, slots), v).view(n, hk, most, -1, d) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 2, 1, 3, 4).reshape(n, most, hq, d)[seq, node].to(_dtype(case))


def run(state):
    if own:
        return _run_own(state)
    case, dt = state["case"], _dtype(state["case"])
    if case["kind"] == "turn":
        return {"q": _turned(state["q"], state["q_norm"], case, state["positions"], state["inv_freq"], torch.float32).to(dt),
                "k": _turned(state["k"], state["k_norm"], case, state["positions"], state["inv_freq"], torch.float32).to(dt)}
    if case["kind"] == "write":
        k = _turned(state["k"], state["k_norm"], case, state["positions"], state["inv_freq"], torch.float64)
        return {"q": _turned(state["q"], state["q_norm"], case, state["positions"], state["inv_freq"], torch.float32).to(dt),
                "k": _cached(k, case).to(dt), "v": _cached(state["v"], case).to(dt)}
    if case["kind"] == "keep":
        seq, node = _rows_of(state)
        base = state["offsets"].long()[seq]
        source = base + torch.where(node < state["counts"].long()[seq], state["accepted"].long(), node)
        return {"k": _cached(state["k"], case)[source].to(dt), "v": _cached(state["v"], case)[source].to(dt)}
    if case["kind"] == "read":
        k, v, _ = _dense(state)
        seq, node = _rows_of(state)
        return {"k": k[seq, :, node].to(dt), "v": v[seq, :, node].to(dt)}
    return _attended(state)


# ---- the library's operators ---------------------------------------------------------------------------------------------------
def _run_own(state):
    from tokspur_public_b200 import attention as A
    case = state["case"]
    if "handles" not in state:   # what a program builds once: descriptors and the workspace
        h = state["handles"] = {}
        if case["kind"] in ("turn", "write"):
            h["turn"] = A.QkNormRope(case["dim"], case["rotary"], case["style"], state["inv_freq"], state["q_norm"], state["k_norm"], eps=1e-6)
        if case["kind"] != "turn":
            h["cache"] = A.KvCache(state["pages"], state["table"], case["page"], case["kv_heads"], case["dim"], case["cache"])
            h["batch"] = A.KvBatch(state["offsets"], state["lengths"], _row_count(case))
        if case["kind"] == "attend":
            h["scratch"] = A.tree_attention_scratch("cuda")
    h = state["handles"]
    if case["kind"] == "turn":
        A.qk_norm_rope(h["turn"], state["q"], state["k"], state["positions"], state["q_out"], state["k_out"], state["error"])
        return {"q": state["q_out"], "k": state["k_out"]}
    if case["kind"] == "write":
        A.qk_norm_rope_append(h["turn"], h["cache"], h["batch"], state["q"], state["k"], state["v"], state["positions"], state["q_out"], state["error"])
        A.kv_cache_read(h["cache"], h["batch"], state["k_out"], state["v_out"], state["error"])
        return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}
    if case["kind"] == "keep":
        A.kv_cache_append(h["cache"], h["batch"], state["k"], state["v"], state["error"])
        A.kv_cache_keep(h["cache"], h["batch"], state["accepted"], state["counts"], state["error"])
        A.kv_cache_read(h["cache"], h["batch"], state["k_out"], state["v_out"], state["error"])
        return {"k": state["k_out"], "v": state["v_out"]}
    if case["kind"] == "read":
        A.kv_cache_read(h["cache"], h["batch"], state["k_out"], state["v_out"], state["error"])
        return {"k": state["k_out"], "v": state["v_out"]}
    A.tree_attention(h["cache"], h["batch"], state["q"], state["out"], state["mask"], case["most"], 1.0 / math.sqrt(case["dim"]), h["scratch"], state["error"])
    return state["out"]


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def work(case):
    d, hq, hk, io = case["dim"], case["q_heads"], case["kv_heads"], 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "turn":
        return {"bytes": case["rows"] * ((hq + hk) * d * 2 * io + 4), "flops": case["rows"] * (hq + hk) * d * 8}
    rows, slot = _row_count(case), hk * _group_bytes(case) // GROUP
    held = sum(_lengths(case)) + rows
    if case["kind"] == "write":
        return {"bytes": rows * (hq * d * 2 * io + hk * d * 4 * io + 2 * slot + 4), "flops": rows * d * (8 * hq + 20 * hk)}
    if case["kind"] == "keep":
        return {"bytes": rows * (hk * d * 4 * io + 2 * slot) + rows // 2 * 2 * slot, "flops": rows * hk * d * 8}
    if case["kind"] == "read":
        return {"bytes": held * (slot + 2 * hk * d * io), "flops": held * hk * d * 2}
    return {"bytes": held * slot + rows * hq * d * 2 * io, "flops": 4 * d * hq * sum(c * (l + c) for c, l in zip(_counts(case), _lengths(case)))}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------
def _exact_head(state, s, h, first, count):
    """K and V of slots [first, first + count) of sequence s, head h, in 64 bits, each value by its own address in the pages."""
    case, d, page = state["case"], state["case"]["dim"], state["case"]["page"]
    dev = state["pages"].device
    gb = _group_bytes(case)
    slot = first + torch.arange(count, device=dev)
    at = state["table"][s].long()[slot // page] * state["pages"].shape[1] + (h * (page // GROUP) + slot % page // GROUP) * gb
    t, x = (slot % GROUP)[:, None], torch.arange(d, device=dev)[None]
    lane, e = t % 8 // 2, t % 2 + 2 * (t // 8)                       # a V slot's place: (t, e)
    flat = state["pages"].view(-1)
    if case["cache"] == "f16":
        k = (x // 32 * GROUP + t) * 32 + x % 32
        i = x % 32 // 8
        v = GROUP * d + ((((x // 32 * 2 + i // 2) * 8 + x % 8) * 4 + lane) * 2 + i % 2) * 4 + e
        halves = flat.view(torch.float16)
        return halves[at[:, None] // 2 + k].double(), halves[at[:, None] // 2 + v].double()
    k = x // 64 * (GROUP * 64) + t * 64 + x % 32 // 8 * 16 + x % 64 // 32 * 8 + x % 8
    v = ((x // 32 * 8 + x % 8) * 4 + lane) * 16 + x % 32 // 8 * 4 + e
    scale = GROUP * d + 2 * (x // 32 * GROUP + t)

    def values(where, base):
        low, high = flat[base + scale].long(), flat[base + scale + 1].long()
        bits = (low + 256 * high).to(torch.int32)
        d16 = torch.where(bits >= 32768, bits - 65536, bits).to(torch.int16).view(torch.float16).double()
        return (flat[base + where].double() - 128) * d16
    base = at[:, None]
    return values(k, base), values(v, base + gb // 2)


def _exact_turn(x, weight, state):
    case = state["case"]
    x = x.double()
    y = x / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    r = case["rotary"]
    out = y.clone()
    for p in range(r // 2):
        angle = state["positions"].double() * state["inv_freq"][p].double()
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        a, b = (p, p + r // 2) if case["style"] == "halves" else (2 * p, 2 * p + 1)
        out[:, :, a], out[:, :, b] = y[:, :, a] * c - y[:, :, b] * s, y[:, :, b] * c + y[:, :, a] * s
    return out


def _exact_cached(x, case):
    x = x.double()
    if case["cache"] == "f16":
        return x.float().half().double()
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], 32):
        block = x[..., b:b + 32]
        d16 = (block.abs().max(-1, keepdim=True).values / 127).float().half().double()
        out[..., b:b + 32] = torch.nan_to_num(torch.round(block / d16), nan=0.0).clamp(-127, 127) * d16
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "turn":
        return {"q": _exact_turn(s["q"], s["q_norm"], s), "k": _exact_turn(s["k"], s["k_norm"], s)}
    if case["kind"] == "write":
        return {"q": _exact_turn(s["q"], s["q_norm"], s), "k": _exact_cached(_exact_turn(s["k"], s["k_norm"], s), case), "v": _exact_cached(s["v"], case)}
    counts, lengths = _counts(case), _lengths(case)
    starts = [sum(counts[:i]) for i in range(len(counts))]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    rows = sum(counts)
    if case["kind"] == "keep":
        k, v = _exact_cached(s["k"], case), _exact_cached(s["v"], case)
        source = list(range(rows))
        accepted, kept = s["accepted"].tolist(), s["counts"].tolist()
        for at, n in zip(starts, kept):
            for j in range(n):
                source[at + j] = at + accepted[at + j]
        return {"k": k[source], "v": v[source]}
    if case["kind"] == "read":
        k, v = (torch.empty(rows, hk, d, dtype=torch.float64, device="cuda") for _ in range(2))
        for i in range(case["sequences"]):
            for h in range(hk):
                k[starts[i]:starts[i] + counts[i], h], v[starts[i]:starts[i] + counts[i], h] = _exact_head(s, i, h, 0, counts[i])
        return {"k": k, "v": v}
    out = torch.zeros(rows, hq, d, dtype=torch.float64, device="cuda")
    for i in range(case["sequences"]):
        at, n, length = starts[i], counts[i], lengths[i]
        visible = torch.ones(n, length + n, dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            visible[:, length:] = torch.tril(visible[:, length:])
        else:
            words = s["mask"][at:at + n].tolist()
            visible[:, length:] = torch.tensor([[bool(w >> j & 1) for j in range(n)] for w in words], device="cuda")
        for h in range(hk):
            k, v = _exact_head(s, i, h, 0, length + n)
            for r in range(hq // hk):
                x = s["q"][at:at + n, h * (hq // hk) + r].double() @ k.T / math.sqrt(d)
                out[at:at + n, h * (hq // hk) + r] = torch.softmax(x.masked_fill(~visible, -math.inf), -1) @ v
    return out
