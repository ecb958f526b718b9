"""Plain 64-bit restatements of the attention operators for the tests: head norm and rotation, the cache's quantiser and byte layout,
attention of drafted tokens. numpy only; nothing here is shared with the library."""
import numpy as np


def turned(x, weight, positions, inv_freq, rotary, style, eps, magnitude=1.0):
    """[rows, heads, dim] -> the same in float64."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * weight.astype(np.float64)
    out = y.copy()
    for p in range(rotary // 2):
        angle = positions.astype(np.float64) * np.float64(inv_freq[p])
        c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
        a, b = (p, p + rotary // 2) if style == "halves" else (2 * p, 2 * p + 1)
        out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    return out


def quantised(x):
    """[..., dim] -> (codes int, scales float16 [..., dim/32]) of the Q8_0 rule, in float64."""
    blocks = x.astype(np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    d = (np.abs(blocks).max(-1) / 127).astype(np.float32).astype(np.float16)
    df = d.astype(np.float64)[..., None]
    q = np.where(df > 0, np.clip(np.rint(blocks / np.where(df > 0, df, 1)), -127, 127), 0)
    return q.reshape(x.shape).astype(np.int64), d


def cached(x, type_):
    """What the cache holds of rows [..., dim], float64."""
    if type_ == "f16":
        return x.astype(np.float32).astype(np.float16).astype(np.float64)
    q, d = quantised(x)
    return q * np.repeat(d.astype(np.float64), 32, -1)


def half_bytes(dim, type_):
    return 17 * dim if type_ == "q8_0" else 32 * dim


def places(dim, type_):
    """Byte offsets within a group's K and V part of value (slot, dim): two [16, dim] tables, and of scale (slot, block)."""
    k, v = np.zeros((16, dim), np.int64), np.zeros((16, dim), np.int64)
    n = 0
    if type_ == "q8_0":
        for panel in range(dim // 64):
            for t in range(16):
                for chunk in range(4):
                    for half in range(2):
                        for i in range(8):
                            k[t, 64 * panel + 32 * half + 8 * chunk + i] = n
                            n += 1
        n = 0
        for b in range(dim // 32):
            for g in range(8):
                for t in range(4):
                    for i in range(4):
                        for e in range(4):
                            v[2 * t + (e & 1) + 8 * (e >> 1), 32 * b + 8 * i + g] = n
                            n += 1
        scale = 16 * dim + 2 * (np.arange(dim // 32)[None] * 16 + np.arange(16)[:, None])
        return k, v, scale
    for panel in range(dim // 32):
        for t in range(16):
            for x in range(32):
                k[t, 32 * panel + x] = n
                n += 2
    n = 0
    for b in range(dim // 32):
        for m in range(2):
            for g in range(8):
                for t in range(4):
                    for i in range(2):
                        for e in range(4):
                            v[2 * t + (e & 1) + 8 * (e >> 1), 32 * b + 8 * (2 * m + i) + g] = n
                            n += 2
    return k, v, None


class Pages:
    """A cache's bytes on the host: uint8 [pages, stride], page table [sequences, columns]."""

    def __init__(self, rng, type_, page, kv_heads, dim, slots, spare=2, pad=0, fill=None):
        """slots: slots of every sequence that have a page."""
        self.type, self.page, self.heads, self.dim = type_, page, kv_heads, dim
        need = [max(1, -(-n // page)) for n in slots]
        self.columns = max(need)
        pages = sum(need) + spare
        self.stride = kv_heads * (page // 16) * 2 * half_bytes(dim, type_) + pad
        self.data = (rng.integers(0, 256, (pages, self.stride)).astype(np.uint8) if fill is None else np.full((pages, self.stride), fill, np.uint8))
        order = rng.permutation(pages)
        self.table = np.full((len(slots), self.columns), 0xffffffff, np.uint32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.k_at, self.v_at, self.scale_at = places(dim, type_)

    def part(self, s, slot, h):
        row = self.data[self.table[s, slot // self.page]]
        hb = half_bytes(self.dim, self.type)
        at = (h * (self.page // 16) + slot % self.page // 16) * 2 * hb
        return row[at:at + hb], row[at + hb:at + 2 * hb]

    def put(self, s, slot, k, v):
        """k, v: [heads, dim], finite."""
        t = slot % 16
        for h in range(self.heads):
            for part, at, x in zip(self.part(s, slot, h), (self.k_at, self.v_at), (k[h], v[h])):
                if self.type == "q8_0":
                    q, d = quantised(x)
                    part[at[t]] = (q + 128).astype(np.uint8)
                    raw = d.view(np.uint8).reshape(-1, 2)
                    part[self.scale_at[t]], part[self.scale_at[t] + 1] = raw[:, 0], raw[:, 1]
                else:
                    raw = x.astype(np.float32).astype(np.float16).view(np.uint8).reshape(-1, 2)
                    part[at[t]], part[at[t] + 1] = raw[:, 0], raw[:, 1]

    def get(self, s, slot):
        """K and V of a slot, float64 [heads, dim]."""
        out = np.zeros((2, self.heads, self.dim))
        t = slot % 16
        for h in range(self.heads):
            for w, (part, at) in enumerate(zip(self.part(s, slot, h), (self.k_at, self.v_at))):
                if self.type == "q8_0":
                    d = np.stack([part[self.scale_at[t]], part[self.scale_at[t] + 1]], -1).reshape(-1).copy().view(np.float16).astype(np.float64)
                    out[w, h] = (part[at[t]].astype(np.float64) - 128) * np.repeat(d, 32)
                else:
                    out[w, h] = np.stack([part[at[t]], part[at[t] + 1]], -1).reshape(-1).copy().view(np.float16).astype(np.float64)
        return out[0], out[1]

    def poke_scale(self, s, slot, value, which=(0, 1)):
        """Q8_0: every scale of the slot; F16: every value of it, becomes `value` (a binary16 number, NaN and infinities too)."""
        raw = np.array([value], np.float16).view(np.uint8)
        t = slot % 16
        for h in range(self.heads):
            for w, (part, at) in enumerate(zip(self.part(s, slot, h), (self.k_at, self.v_at))):
                if w in which:
                    where = self.scale_at[t] if self.type == "q8_0" else at[t]
                    part[where], part[where + 1] = raw[0], raw[1]


def attended(q, k, v, visible, scale):
    """q [heads, dim], k / v [slots, kv heads, dim], visible [slots] -> [heads, dim] in float64; also the largest score's error scale
    sum_i |q_i k_i| over the visible slots, and the largest |v|."""
    heads, dim = q.shape
    group = heads // k.shape[1]
    out, spread, vmax = np.zeros((heads, dim)), 0.0, 0.0
    if not visible.any():
        return out, 0.0, 0.0
    k, v = k[visible], v[visible]
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = kh @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        out[h] = p @ vh / p.sum()
        spread = max(spread, float((np.abs(kh) @ np.abs(q[h].astype(np.float64))).max()) * abs(scale))
    return out, spread, float(np.abs(v).max())
