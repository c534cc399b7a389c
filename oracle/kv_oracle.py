"""The 8-bit paged key/value cache, its page table and its attention in numpy: the oracle of include/kv_cache.h.

Quantisation is restated with exact quotients (codes and scales are compared
bit for bit); attention in 64 bits; the page table in plain loops. A cache's
scales are the largest magnitudes of its pages and heads: a value is code *
scale / 127.
Codes are kept as [pages, heads, page_size, D] in token order; pack / unpack
translate the library's order (its bytes hold code + 128).
"""
from __future__ import annotations

import math

import numpy as np

F = np.float32


def unpack_k(raw: np.ndarray, D: int, page: int) -> np.ndarray:
    """Library bytes [pages, heads, page D] of K -> codes [pages, heads, page, D]."""
    P, H = raw.shape[:2]
    v = (raw.view(np.uint8) ^ 0x80).view(np.int8).reshape(P, H, page // 16, D // 64, 4, 16, 16)  # sub, chunk, kg, token, e
    return v.transpose(0, 1, 2, 5, 3, 4, 6).reshape(P, H, page, D).copy()


def pack_k(codes: np.ndarray) -> np.ndarray:
    P, H, page, D = codes.shape
    v = (codes.view(np.uint8) ^ 0x80).reshape(P, H, page // 16, 16, D // 64, 4, 16)
    return v.transpose(0, 1, 2, 4, 5, 3, 6).reshape(P, H, page * D).copy()


def unpack_v(raw: np.ndarray, D: int, page: int) -> np.ndarray:
    P, H = raw.shape[:2]
    v = (raw.view(np.uint8) ^ 0x80).view(np.int8).reshape(P, H, page // 16, D // 64, 4, 4, 4, 4, 4)  # sub, chunk, kg, q, r, i, tt
    # token = 4 q + tt, d = 64 c + 16 kg + 4 i + r
    return v.transpose(0, 1, 2, 5, 8, 3, 4, 7, 6).reshape(P, H, page, D).copy()


def pack_v(codes: np.ndarray) -> np.ndarray:
    P, H, page, D = codes.shape
    v = (codes.view(np.uint8) ^ 0x80).reshape(P, H, page // 16, 4, 4, D // 64, 4, 4, 4)  # sub, q, tt, chunk, kg, i, r
    return v.transpose(0, 1, 2, 5, 6, 3, 8, 7, 4).reshape(P, H, page * D).copy()


class Cache:
    """K or V of one layer."""

    def __init__(self, codes: np.ndarray, scales: np.ndarray):
        self.codes, self.scales = codes, scales

    def append(self, x: np.ndarray, cu, ctx, table) -> int:
        """x: float32 values of the 16-bit rows [total, heads, D]. Returns the tokens dropped."""
        P, H, page, D = self.codes.shape
        dropped = 0
        for b in range(len(ctx)):
            n = cu[b + 1] - cu[b]
            i = 0
            while i < n:
                pos = ctx[b] + i
                col, slot = divmod(pos, page)
                m = min(n - i, page - slot)
                pg = table[b, col] if col < table.shape[1] else -1
                if pg < 0 or pg >= P:
                    dropped += m
                else:
                    self._block(pg, slot, x[cu[b] + i:cu[b] + i + m])
                i += m
        return dropped

    def _block(self, pg, slot, x):
        H, page, D = self.codes.shape[1:]
        mag = np.where(np.isfinite(x), np.abs(x), F(0)).max(axis=(0, 2)).astype(F)   # [H]
        old = self.scales[pg].copy() if slot > 0 else np.zeros(H, F)
        s = np.maximum(old, mag)
        # 127 x and code old are exact in 64 bits; their quotients by s are half-integers exactly, or further from one
        # than a rounding of theirs (x and s have at most 11 significant bits).
        for h in range(H):
            m = np.float64(s[h])
            if slot > 0 and s[h] > old[h]:
                q = self.codes[pg, h, :slot].astype(np.float64) * np.float64(old[h]) / m
                self.codes[pg, h, :slot] = np.rint(q).astype(np.int8)
            if s[h] > 0:
                q = np.rint(127 * x[:, h].astype(np.float64) / m)
                q = np.where(np.isnan(q), 127, np.clip(q, -127, 127))
            else:
                q = np.zeros((len(x), D))
            self.codes[pg, h, slot:slot + len(x)] = q.astype(np.int8)
            self.codes[pg, h, slot + len(x):] = 0
        self.scales[pg] = s

    def read(self, cu, starts, table):
        """Values in float32 (code * RN(scale / 127)) of the tokens asked for, {row: [heads, D]}."""
        P, H, page, D = self.codes.shape
        out = {}
        for b in range(len(starts)):
            for i in range(cu[b + 1] - cu[b]):
                col, slot = divmod(starts[b] + i, page)
                pg = table[b, col] if col < table.shape[1] else -1
                ok = 0 <= pg < P
                out[cu[b] + i] = (self.codes[pg, :, slot].astype(F) * (self.scales[pg] / F(127))[:, None] if ok
                                  else np.zeros((H, D), F))
        return out


def attention(q, kc: Cache, vc: Cache, cu, lens, table, scale, window=0, sinks=0):
    """Attention of q [total, hq, D] in 64 bits: {row: (out, mag, dot, xmax, vmax, seen)}, out and mag [hq, D], the
    others by head: mag = sum_j w_j |v_j| / sum_j w_j, dot the largest scale sum_d |q_d| |k_jd|, xmax the largest
    |score|, vmax the largest |v| (by what an error bound is made of), seen the tokens that count."""
    P, H, page, D = kc.codes.shape
    hq = q.shape[1]
    G = hq // H
    got = {}
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        if n <= 0:
            continue
        L = min(max(lens[b], 0), table.shape[1] * page)
        j = np.arange(L)
        pg = table[b, j // page] if L else np.zeros(0, int)
        there = (pg >= 0) & (pg < P)
        safe = np.where(there, pg, 0)
        k = kc.codes[safe, :, j % page].astype(np.float64) * kc.scales[safe].astype(np.float64)[:, :, None] / 127
        v = vc.codes[safe, :, j % page].astype(np.float64) * vc.scales[safe].astype(np.float64)[:, :, None] / 127
        for i in range(n):
            p = lens[b] - n + i
            seen = there & (j <= p)
            if window:
                seen &= (j > p - window) | (j < sinks)
            o, a, top = np.zeros((hq, D)), np.zeros((hq, D)), np.zeros((3, hq))
            for h in range(hq if seen.any() else 0):
                qh, kh, vh = q[cu[b] + i, h].astype(np.float64), k[seen, h // G], v[seen, h // G]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = scale * (kh @ qh)
                    w = np.exp(x - x.max())
                    w /= w.sum()
                    o[h], a[h] = w @ vh, w @ np.abs(vh)
                    top[:, h] = scale * (np.abs(kh) @ np.abs(qh)).max(), np.abs(x).max(), np.abs(vh).max()
            got[cu[b] + i] = (o, a, *top, int(seen.sum()))
    return got


# ---------------------------------------------------------------- page table

def _pages(n, page):
    return -(-max(int(n), 0) // page)


def grow(table, refs, old, new, page):
    """Returns (table, refs, copy_src, copy_dst, missing); inputs are not changed."""
    R, W = table.shape
    src, dst = np.full(R, -1, np.int32), np.full(R, -1, np.int32)
    asks, over = [], 0
    for r in range(R):
        o, n = max(int(old[r]), 0), int(new[r])
        if n <= o:
            continue
        have, want = _pages(o, page), _pages(n, page)
        over += max(want - W, 0)
        want = min(want, W)
        have = min(have, want)
        if o % page and have and refs[table[r, have - 1]] > 1:
            asks.append((r, -1))
            src[r] = table[r, have - 1]
        asks += [(r, i) for i in range(have, want)]
    free = np.flatnonzero(refs <= 0)
    missing = over + max(len(asks) - len(free), 0)
    if missing:
        return table.copy(), refs.copy(), np.full(R, -1, np.int32), dst, missing
    t, c = table.copy(), refs.copy()
    for (r, i), pg in zip(asks, free):
        c[pg] = 1
        if i < 0:
            dst[r] = pg
            c[src[r]] -= 1
            t[r, _pages(old[r], page) - 1] = pg
        else:
            t[r, i] = pg
    return t, c, src, dst, 0


def fork(table, refs, parents, lens, page):
    R, W = table.shape
    t, c, n = np.full_like(table, -1), refs.copy(), np.zeros(R, np.int32)
    for r in range(R):
        if 0 <= parents[r] < R:
            k = min(_pages(lens[parents[r]], page), W)
            t[r, :k] = table[parents[r], :k]
            n[r] = max(lens[parents[r]], 0)
            for e in t[r, :k]:
                c[e] += e >= 0
        for e in table[r, :min(_pages(lens[r], page), W)]:
            c[e] -= e >= 0
    return t, c, n


def free(table, refs, old, keep, page):
    t, c = table.copy(), refs.copy()
    for r in range(len(old)):
        for i in range(_pages(keep[r], page), min(_pages(old[r], page), table.shape[1])):
            if t[r, i] >= 0:
                c[t[r, i]] -= 1
            t[r, i] = -1
    return t, c


def compact(table, refs, capacity):
    used = np.flatnonzero(refs > 0)
    n = len(used)
    back, front = used[used >= n], np.flatnonzero(refs[:n] <= 0)
    assert len(back) == len(front)
    src, dst = np.full(capacity, -1, np.int32), np.full(capacity, -1, np.int32)
    src[:len(back)], dst[:len(back)] = back, front
    t, c = table.copy(), refs.copy()
    to = dict(zip(back.tolist(), front.tolist()))
    for a, b in to.items():
        c[b], c[a] = refs[a], 0
    for i, e in enumerate(t.flat):
        t.flat[i] = to.get(int(e), int(e))
    return t, c, src, dst, len(back)
