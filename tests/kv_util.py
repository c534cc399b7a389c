"""What the key/value cache tests share: caches in device memory, packed batches, the attention's error bound."""
from __future__ import annotations

import ctypes as C

import numpy as np

from gpu_util import dev, empty, f32, get, ok
from neurogrid_amd._lib import KVInt8Cache, KVPages
from oracle import kv_oracle as K

PREFIX = {"f16": "ng_", "bf16": "ng_bf16_"}


def bits(x, dtype) -> np.ndarray:
    x = np.asarray(x, np.float32)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def starts(lens) -> np.ndarray:
    return np.concatenate(([0], np.cumsum(lens))).astype(np.int32)


class DeviceCache:
    """One layer's cache on the device, made from oracle caches of K and V."""

    def __init__(self, k: K.Cache, v: K.Cache):
        self.pages, self.heads, self.page, self.D = k.codes.shape
        self.bufs = [dev(K.pack_k(k.codes)), dev(K.pack_v(v.codes)), dev(k.scales), dev(v.scales)]
        self.c = KVInt8Cache(*[b.ptr for b in self.bufs], self.pages, self.heads, self.D, self.page)

    def get(self):
        """(K codes, V codes, K scales, V scales), codes in token order."""
        shape = (self.pages, self.heads, self.page * self.D)
        k, v = (get(b, np.int8, shape) for b in self.bufs[:2])
        ks, vs = (get(b, np.float32, (self.pages, self.heads)) for b in self.bufs[2:])
        return K.unpack_k(k, self.D, self.page), K.unpack_v(v, self.D, self.page), ks, vs


def random_cache(rng, pages, heads, page, D) -> tuple[K.Cache, K.Cache]:
    """Full pages of codes and scales as a cache in use has them; scales over one and a half decades."""
    def one():
        codes = np.clip(np.rint(rng.standard_normal((pages, heads, page, D)) * 40), -127, 127).astype(np.int8)
        return K.Cache(codes, (10.0 ** rng.uniform(-0.4, 1.1, (pages, heads))).astype(np.float32))
    return one(), one()


def random_table(rng, lens, page, spare=2, width=None):
    """Shuffled pages for sequences of these lengths; (table, number of pages). Unused entries are -1."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lens), width or max(max(need), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages, order[at:]


def pool(table, refs, page):
    """(KVPages, table buffer, refs buffer)."""
    t, r = dev(table), dev(refs)
    return KVPages(t.ptr, r.ptr, table.shape[0], table.shape[1], len(refs), page), t, r


def attend(lib, dtype, dc, qbits, cu, lens, table, scale, window=0, sinks=0, max_q=None, max_kv=None, workspace="asked",
           out=None):
    """One call; returns the output's bits [total, hq, D]. workspace: "asked", None or a number of bytes."""
    total, hq, D = qbits.shape
    qb = dev(qbits)
    ob = dev(out if out is not None else np.full_like(qbits, 0x1234))
    cub, lb, tb = dev(np.asarray(cu, np.int32)), dev(np.asarray(lens, np.int32)), dev(table)
    batch = len(lens)
    max_q = max_q or max(1, int(np.diff(cu).max()))
    max_kv = max_kv or max(1, int(max(lens)))
    n = lib.ng_kv_int8_attention_workspace(C.byref(dc.c), hq, batch, max_q, max_kv)
    n = n if workspace == "asked" else workspace or 0
    ws = empty(max(n, 1)) if n else None
    if ws is not None:
        ws.upload(np.full(n, 0xFF, np.uint8))  # NaN wherever it is read before it is written
    ok(getattr(lib, PREFIX[dtype] + "kv_int8_attention")(
        ob.vp, qb.vp, C.byref(dc.c), cub.vp, lb.vp, tb.vp, batch, table.shape[1], total, max_q, max_kv, hq,
        C.c_float(scale), window, sinks, ws.vp if ws is not None else None, n), "attention")
    return get(ob, np.uint16, qbits.shape)


# Half a step of the output's type, relative, and the least step's half.
HALF = {"f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}


def bound(dtype, D, ref):
    """Largest error of an output row [hq, D] that the documented roundings allow.

    A score is a sum of D products in fp32 (any order: D + 1 roundings of at most
    2^-24 of sum |q| |k|), times a factor of three roundings, with an exponential
    of an argument rounded to 2^-24 of at most 2 |x| log2 e, and of 2^-22 itself:
    relative error e of a weight. Weights enter the sum over V rounded to 11 bits
    (2^-11 relative; half of fp16's least step where subnormal, 2^-25, which is
    2^-32 of the largest as weights stand at least 2^7 above their value, of a unit
    that is at most twice the largest |v|), times V's scale factor (3 roundings),
    the sums over the tokens have a rounding a token. The quotient doubles the
    weights' error. Then the output's own rounding.
    """
    o, mag, dot, xmax, vmax, seen = ref
    u = 2.0 ** -24
    e = (D + 4) * u * dot + 8 * u * xmax + 2.0 ** -21
    half, least = HALF[dtype]
    err = (2 * e)[:, None] * mag + (2.0 ** -11 + (2 * seen + 16) * u) * mag + (seen * 2.0 ** -31 * vmax)[:, None]
    return err * (1 + half) + half * np.abs(o) + least


def check_attention(got, dtype, D, refs, untouched=None):
    """Rows of got (bits) against the oracle's; rows that it does not name keep their 0x1234."""
    g = f32(got, dtype).astype(np.float64)
    for row, ref in refs.items():
        d = np.abs(g[row] - ref[0])
        tol = bound(dtype, D, ref)
        assert (d <= tol).all(), (f"row {row}: off by {np.nanmax(d / tol):.2f} of its bound at "
                                  f"{np.argwhere(~(d <= tol))[:3].tolist()}: {d.max():.3g}")
    rest = [r for r in range(len(got)) if r not in refs]
    if rest:
        assert (got[rest] == 0x1234).all(), "rows of no sequence were written"
