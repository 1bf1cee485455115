"""Plain restatements of the 4-bit key/value cache operators for the tests: the cache's bytes in numpy,
attention in float64, and the error bound that the operators' arithmetic allows."""
from __future__ import annotations

import numpy as np

LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)


def quantise(x: np.ndarray):
    """f32 [..., D] -> (codes u8 [..., D], scale bytes u8 [..., D/32]).  Scale: the smallest 2^n >= amax / 6 with
    n >= -126, found with exact integer arithmetic on frexp; code: nearest level, a tie to the smaller."""
    blocks = x.astype(np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(blocks).all(-1)
    safe = np.where(finite[..., None], blocks, 0.0)
    mant, exp = np.frexp(np.abs(safe).max(-1))
    n = np.where(mant == 0, -126, np.maximum(np.where(mant <= 0.75, exp - 3, exp - 2), -126))
    q = np.abs(safe) / 2.0 ** n[..., None]
    code = np.searchsorted((LEVELS[1:] + LEVELS[:-1]) / 2, q, side="left").astype(np.uint8)
    code |= np.where(np.signbit(safe), 8, 0).astype(np.uint8)
    code = np.where(finite[..., None], code, 0)
    return code.reshape(x.shape).astype(np.uint8), np.where(finite, n + 127, 255).astype(np.uint8)


def dequantise(code: np.ndarray, scale: np.ndarray) -> np.ndarray:
    with np.errstate(invalid="ignore"):
        s = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
    v = np.where(code & 8, -LEVELS[code & 7], LEVELS[code & 7])
    return (v.reshape(*code.shape[:-1], -1, 32) * s[..., None]).reshape(code.shape)


class HostCache:
    """The four byte arrays of a cache and element access by (page, head, token), written from the layout's formulas."""

    def __init__(self, pages, page_tokens, heads, d, fill=0):
        self.pages, self.p, self.h, self.d = pages, page_tokens, heads, d
        n = pages * heads * page_tokens
        self.arrays = [np.full(n * d // 2, fill, np.uint8), np.full(n * d // 32, fill, np.uint8),
                       np.full(n * d // 2, fill, np.uint8), np.full(n * d // 32, fill, np.uint8)]

    def _at(self, page, head, token, which):
        unit, piece = (32, min(self.d, 128) // 2) if which == 0 else (8, 1)
        base = ((page * self.h + head) * self.p + token // unit * unit)
        pair = np.arange(self.d // 2)
        payload = base * (self.d // 2) + pair // piece * (unit * piece) + token % unit * piece + pair % piece
        scales = base * (self.d // 32) + np.arange(self.d // 32) * unit + token % unit
        return payload, scales

    def put(self, page, head, token, which, code, scale):
        payload, scales = self._at(page, head, token, which)
        self.arrays[2 * which][payload] = code[0::2] | code[1::2] << 4
        self.arrays[2 * which + 1][scales] = scale

    def get(self, page, head, token, which):
        payload, scales = self._at(page, head, token, which)
        byte = self.arrays[2 * which][payload]
        code = np.empty(self.d, np.uint8)
        code[0::2], code[1::2] = byte & 15, byte >> 4
        return code, self.arrays[2 * which + 1][scales]

    def value(self, page, head, token, which):
        return dequantise(*self.get(page, head, token, which))

    def device(self):
        import torch
        from ferrule_amd.provider import HipKvCache, kv_cache_shapes
        shapes = kv_cache_shapes(self.pages, self.p, self.h, self.d)
        return HipKvCache(self.p, self.h, self.d, *[torch.from_numpy(a.reshape(s).copy()).cuda()
                                                    for a, s in zip(self.arrays, shapes)])

    def random(self, rng, lo=118, hi=130):
        """Random nibbles; scale bytes of ordinary values."""
        for i, a in enumerate(self.arrays):
            a[:] = rng.integers(0, 256, a.size) if i % 2 == 0 else rng.integers(lo, hi, a.size)
        return self


class HostBatch:
    """Rows and lengths of the sequences and a shuffled page table for them."""

    def __init__(self, rng, new, lengths, page_tokens, spare=2, extra_columns=1):
        self.new, self.lengths = list(new), list(lengths)
        needed = [-(-length // page_tokens) for length in self.lengths]
        self.pages = sum(needed) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(self.new), max(needed + [1]) + extra_columns), -1, np.int32)
        at = 0
        for b, n in enumerate(needed):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.unused = order[at:]
        self.indptr = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.p = page_tokens

    @property
    def total(self):
        return int(self.indptr[-1])

    def positions(self, b):
        return range(self.lengths[b] - self.new[b], self.lengths[b])

    def place(self, b, position):
        if position < 0 or position // self.p >= self.table.shape[1]:
            return None
        page = int(self.table[b, position // self.p])
        return (page, position % self.p) if 0 <= page < self.pages else None

    def device(self, rows=None, **kw):
        import torch
        from ferrule_amd.provider import HipKvBatch
        f = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
        kw.setdefault("max_query_length", max(self.new + [1]))
        kw.setdefault("max_sequence_length", max(self.lengths + [0]))
        return HipKvBatch(f(self.indptr), f(self.lengths), f(self.table), self.total if rows is None else rows, **kw)


def attention_reference(cache: HostCache, batch: HostBatch, q: np.ndarray, scale: float, window=0, sinks=0,
                        f32_output=False):
    """(output, bound) in float64 for q [rows, q_heads, d] holding BF16 values.

    The bound, with P = softmax weights, S = sum_j P_j |v_j| and A = scale * max_j sum_d |q_d k_jd| over the visible
    j (L of them):
      weights rounded to BF16                                   2^-8 S
      scores: a two-term split of q that keeps 2^-20 of a block's largest magnitude (at most 32 times an element's
      share of the sum, so 32 * 2^-20 A), and an f32 sum of d products (d 2^-23 A, twice the nearest-rounding
      bound because a matrix instruction may cut instead of round); then the product with scale * log2 e and the
      exponential, a few ulp of the score's size (2^-20 A + 2^-20).  An error e of the scores changes the
      weights by at most a factor exp(2 e), the output by 2 e S at most (times 1.1 while e < 0.05)
      sums over the tokens in f32                               2 L 2^-23 S
      the output's own rounding                                 2^-8 |o| in BF16, 2^-22 |o| in f32
    """
    rows, q_heads, d = q.shape
    group = q_heads // cache.h
    out = np.zeros((rows, q_heads, d))
    bound = np.zeros((rows, q_heads, d))
    q = q.astype(np.float64)
    for b in range(len(batch.new)):
        places = [batch.place(b, j) for j in range(batch.lengths[b])]
        for h in range(cache.h):
            if not places:
                continue
            there = np.array([p is not None for p in places])
            k = np.stack([cache.value(*_ph(p, h), 0) if p else np.zeros(d) for p in places])
            v = np.stack([cache.value(*_ph(p, h), 1) if p else np.zeros(d) for p in places])
            for i, p in enumerate(batch.positions(b)):
                r = batch.indptr[b] + i
                j = np.arange(len(places))
                seen = (j <= p) & there
                if window:
                    seen &= (p - j < window) | (j < sinks)
                if not seen.any():
                    continue
                ks, vs = k[seen], v[seen]
                for g in range(group):
                    head = h * group + g
                    s = (ks @ q[r, head]) * scale
                    w = np.exp(s - s.max()) if np.isfinite(s).all() else np.full(len(s), np.nan)
                    w = w / w.sum()
                    o = w @ vs
                    size = np.abs(w) @ np.abs(vs)
                    most = scale * (np.abs(ks) @ np.abs(q[r, head])).max()
                    e = most * (32 * 2.0 ** -20 + d * 2.0 ** -23 + 2.0 ** -20) + 2.0 ** -20
                    out[r, head] = o
                    bound[r, head] = size * (2.0 ** -8 + 2.2 * e + 2 * len(s) * 2.0 ** -23) + \
                        np.abs(o) * (2.0 ** -22 if f32_output else 2.0 ** -8) + 1e-37
    return out, bound


def _ph(place, head):
    return place[0], head, place[1]


def check_attention(got: np.ndarray, want: np.ndarray, bound: np.ndarray):
    assert got.shape == want.shape
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"NaN at {np.argwhere(np.isnan(got) != nan)[:4].tolist()}"
    err = np.abs(got.astype(np.float64) - want)[~nan]
    over = err > bound[~nan]
    assert not over.any(), f"{int(over.sum())} of {over.size} outside the bound, worst ratio " \
                           f"{float((err / bound[~nan]).max()):.3g}"


def bf16(x: np.ndarray) -> np.ndarray:
    """f32 values rounded to BF16, as f32."""
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((bits + 0x7fff + ((bits >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
