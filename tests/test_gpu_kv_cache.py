"""Writing, reading and copying the 8-bit key/value cache on the GPU.

Codes and scales are compared with the numpy oracle bit for bit (the same fp32
operations), the whole cache at a time, so that pages and slots that a call has
no business with are seen to be unchanged. Reading back is one rounding of
code * scale.
"""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import C, HipRuntime, assert_bits_equal, banner, dev, empty, f32, get, ok
from kv_util import PREFIX, DeviceCache, bits, random_cache, random_table, starts
from neurogrid_amd._lib import KVInt8Cache
from oracle import kv_oracle as K

pytestmark = pytest.mark.gpu


def rng_of(*key):
    return np.random.default_rng(key)


def fresh(rng, pages, heads, page, D):
    """Caches whose unused pages hold rubbish: any codes, NaN scales."""
    k, v = random_cache(rng, pages, heads, page, D)
    for c in (k, v):
        c.scales[:] = np.nan
    return k, v


def append(lib, dtype, dc, kb, vb, cu, ctx, table, most=None, dropped=None):
    bufs = [dev(kb), dev(vb), dev(np.asarray(cu, np.int32)), dev(np.asarray(ctx, np.int32)), dev(table)]
    ok(getattr(lib, PREFIX[dtype] + "kv_int8_append")(
        C.byref(dc.c), *[b.vp for b in bufs], len(ctx), table.shape[1], len(kb),
        most or max(1, int(np.diff(cu).max())), dropped.vp if dropped else None), "append")
    ok(lib.cuda_sync_device(), "sync")


def same(dc, k, v, what):
    kc, vc, ks, vs = dc.get()
    for got, want, name in ((kc, k.codes, "K codes"), (vc, v.codes, "V codes"), (ks, k.scales, "K scales"),
                            (vs, v.scales, "V scales")):
        if got.dtype == np.float32:
            got, want = got.view(np.uint32), want.view(np.uint32)
        assert_bits_equal(got, want, f"{what}: {name}")


# (heads, D, page, new tokens, contexts): one token, page borders, several pages, empty sequences.
CASES = [
    (1, 64, 16, [1], [0]),
    (2, 128, 16, [1, 1, 1], [15, 16, 17]),
    (3, 128, 16, [5, 0, 40, 16], [3, 9, 0, 16]),
    (2, 64, 32, [33, 1, 64], [31, 63, 0]),
    (1, 192, 64, [100, 7], [0, 60]),
    (2, 256, 128, [129, 1, 300], [127, 5, 1]),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"h{c[0]}-D{c[1]}-p{c[2]}-{len(c[3])}seq")
def test_append_is_the_oracles_and_reads_back(lib, case, dtype):
    heads, D, page, new, ctx = case
    banner(f"kv append {case} {dtype}")
    rng = rng_of(heads, D, page, len(new))
    lens = [n + c for n, c in zip(new, ctx)]
    table, pages, _ = random_table(rng, lens, page)
    k, v = fresh(rng, pages, heads, page, D)
    dc = DeviceCache(k, v)
    zero = [0] * len(ctx)
    # the context first, then the new tokens: louder, softer and equal ones, so that scales grow and stay
    for counts, at, gain in ((ctx, zero, 1.0), (new, ctx, 1.7)):
        if not sum(counts):
            continue
        cu = starts(counts)
        x = rng.standard_normal((2, sum(counts), heads, D)) * gain * rng.uniform(0.2, 1.5, (2, sum(counts), 1, 1))
        kb, vb = bits(x[0], dtype), bits(x[1], dtype)
        for c, xb in ((k, kb), (v, vb)):
            c.append(f32(xb, dtype).reshape(xb.shape), cu, at, table)
        append(lib, dtype, dc, kb, vb, cu, at, table)
        same(dc, k, v, f"{counts} at {at}")
    cu = starts(lens)
    out = [empty(2 * max(1, sum(lens)) * heads * D) for _ in "kv"]
    args = [dev(cu), dev(np.zeros(len(lens), np.int32)), dev(table)]
    for o in out:
        o.upload(np.full(sum(lens) * heads * D, 0x1234, np.uint16))
    ok(getattr(lib, PREFIX[dtype] + "kv_int8_read")(
        C.byref(dc.c), out[0].vp, out[1].vp, *[a.vp for a in args], len(lens), table.shape[1], sum(lens), max(lens)),
       "read")
    for o, c in zip(out, (k, v)):
        got = get(o, np.uint16, (sum(lens), heads, D))
        want = c.read(cu, zero, table)
        for row in range(sum(lens)):
            assert_bits_equal(got[row], bits(want[row], dtype), f"row {row}")


@pytest.mark.parametrize("page", [16, 64])
def test_tokens_one_by_one(lib, page):
    """A page filled by single tokens, whose scale grows again and again."""
    banner(f"kv append one by one page={page}")
    rng = rng_of(page)
    heads, D, n = 2, 128, page + 5
    table, pages, _ = random_table(rng, [n], page)
    k, v = fresh(rng, pages, heads, page, D)
    dc = DeviceCache(k, v)
    for t in range(n):
        x = rng.standard_normal((2, 1, heads, D)) * (1 + 0.3 * t)
        if t % 7 == 3:
            x[:] = 0
        kb, vb = bits(x[0], "f16"), bits(x[1], "f16")
        for c, xb in ((k, kb), (v, vb)):
            c.append(f32(xb, "f16").reshape(xb.shape), [0, 1], [t], table)
        append(lib, "f16", dc, kb, vb, [0, 1], [t], table)
    same(dc, k, v, "after the last token")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_extreme_values(lib, dtype):
    """Infinities, NaN, zero blocks, subnormals and the type's largest values; a zero block that then grows."""
    banner(f"kv append extremes {dtype}")
    rng = rng_of(3)
    heads, D, page = 2, 64, 16
    big, tiny = (65504.0, 6e-8) if dtype == "f16" else (3.38e38, 1e-40)
    blocks = [np.zeros((16, heads, D)), np.full((16, heads, D), tiny), rng.standard_normal((16, heads, D)) * big / 8,
              rng.standard_normal((16, heads, D)), rng.standard_normal((16, heads, D)),
              np.full((16, heads, D), np.nan), rng.standard_normal((16, heads, D)) * tiny * 40]
    blocks[3][2, :, 5], blocks[3][3, :, 6], blocks[3][4, :, 7] = np.inf, -np.inf, np.nan
    blocks[4][:] = np.inf
    blocks[4][7, 0, 1] = -0.25
    x = np.concatenate(blocks + [np.zeros((3, heads, D))]).astype(np.float32)
    n = len(x)
    table, pages, _ = random_table(rng, [n + 4], page)
    k, v = fresh(rng, pages, heads, page, D)
    dc = DeviceCache(k, v)
    kb, vb = bits(x, dtype), bits(-x[:, ::-1], dtype)
    more = bits(np.array([1e-3, 2.0, 0.0, 7.0])[:, None, None] * np.ones((1, heads, D)), dtype)
    for a, b, cu, ctx in ((kb, vb, [0, n], [0]), (more, more, [0, 4], [n])):
        for c, xb in ((k, a), (v, b)):
            with np.errstate(all="ignore"):
                c.append(f32(xb, dtype).reshape(xb.shape), cu, ctx, table)
        append(lib, dtype, dc, a, b, cu, ctx, table)
        same(dc, k, v, f"tokens {cu[1]}")
    assert all(np.isfinite(c.scales[table[0]]).all() for c in (k, v))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_ties_go_to_the_even_code(lib, dtype):
    """Half-integer quotients: m / 2 for every significand of m (63.5 steps), a page of each, and codes that halve when
    a louder token follows."""
    banner(f"kv append ties {dtype}")
    n = 11 if dtype == "f16" else 8
    m = np.arange(2 ** (n - 1), 2 ** n, dtype=np.float64)
    heads, D, page = 1, 64, 16
    pages = len(m)
    x = np.zeros((pages, page - 1, heads, D), np.float32)
    x[:, 0, 0, 0], x[:, 0, 0, 1:4] = m, np.stack([m / 2, -m / 2, m / 4]).T
    table = np.arange(pages, dtype=np.int32)[::-1].copy()[:, None]
    k, v = fresh(rng_of(9), pages, heads, page, D)
    dc = DeviceCache(k, v)
    for part, at in ((x, 0), (np.full((pages, 1, heads, D), 1.0, np.float32) * 2 * m[:, None, None, None], page - 1)):
        part = part.reshape(-1, heads, D)
        cu = (np.arange(pages + 1) * (len(part) // pages)).astype(np.int32)
        b = bits(part, dtype)
        ctx = [at] * pages
        for c in (k, v):
            c.append(f32(b, dtype).reshape(b.shape), cu, ctx, table)
        append(lib, dtype, dc, b, b, cu, ctx, table)
        same(dc, k, v, f"at {at}")
        if at == 0:
            assert (k.codes[:, 0, 0, 1] == 64).all() and (k.codes[:, 0, 0, 2] == -64).all()


def test_missing_pages_are_counted_and_nothing_else_is_touched(lib):
    banner("kv append missing pages")
    rng = rng_of(4)
    heads, D, page = 2, 128, 16
    new, ctx = [40, 20, 64, 3], [10, 40, 0, 30]
    table, pages, _ = random_table(rng, [64, 64, 64, 64], page, width=4)
    table[0, 1] = -1           # a hole
    table[1, 2] = pages        # not a page's number
    table[2, 3] = 2 ** 31 - 1
    ctx[3] = 62                # past the last entry: 2 tokens fit, 1 does not
    k, v = random_cache(rng, pages, heads, page, D)
    dc = DeviceCache(k, v)
    cu = starts(new)
    x = rng.standard_normal((2, sum(new), heads, D))
    kb, vb = bits(x[0], "f16"), bits(x[1], "f16")
    want = [c.append(f32(xb, "f16").reshape(xb.shape), cu, ctx, table) for c, xb in ((k, kb), (v, vb))]
    d = dev(np.array([5], np.int32))
    append(lib, "f16", dc, kb, vb, cu, ctx, table, dropped=d)
    assert get(d, np.int32, (1,))[0] == 5 + want[0]
    same(dc, k, v, "missing pages")
    # reading the same range gives zeros there, and rows of no sequence keep what they hold
    o = [dev(np.full((sum(new) + 2, heads, D), 0x1234, np.uint16)) for _ in "kv"]
    args = [dev(cu), dev(np.asarray(ctx, np.int32)), dev(table)]
    ok(lib.ng_kv_int8_read(C.byref(dc.c), o[0].vp, o[1].vp, *[a.vp for a in args], 4, 4, sum(new) + 2, 1), "read")
    for buf, c in zip(o, (k, v)):
        got = get(buf, np.uint16, (sum(new) + 2, heads, D))
        for row, w in c.read(cu, ctx, table).items():
            assert_bits_equal(got[row], bits(w, "f16"), f"row {row}")
        assert (got[-2:] == 0x1234).all()


def test_longest_hint_changes_nothing(lib):
    """max_tokens below and above the real lengths; cu_tokens past the end and falling."""
    banner("kv append hints")
    rng = rng_of(5)
    heads, D, page = 1, 64, 16
    new = [70, 3]
    table, pages, _ = random_table(rng, new, page)
    x = rng.standard_normal((2, 73, heads, D))
    kb, vb = bits(x[0], "f16"), bits(x[1], "f16")
    first = None
    for most in (1, 70, 5000):
        k, v = random_cache(np.random.default_rng(1), pages, heads, page, D)
        dc = DeviceCache(k, v)
        append(lib, "f16", dc, kb, vb, starts(new), [0, 0], table, most=most)
        got = dc.get()
        first = first or got
        for a, b in zip(got, first):
            assert_bits_equal(a, b, f"most={most}")
    # rows past the total are not read: sequence 1 has none left, sequence 0 ends at the total
    k, v = random_cache(np.random.default_rng(1), pages, heads, page, D)
    dc = DeviceCache(k, v)
    append(lib, "f16", dc, kb[:50], vb[:50], [0, 1000, 20], [0, 0], table)
    for c, xb in ((k, kb), (v, vb)):
        c.append(f32(xb[:50], "f16").reshape(50, heads, D), [0, 50, 50], [0, 0], table)
    same(dc, k, v, "clamped rows")


def test_offsets_past_32_bits(lib):
    """Pages behind the first 4 GiB of codes."""
    banner("kv append, read and copy past 4 GiB")
    heads, D, page, pages = 8, 128, 64, 70000  # 65536 bytes of K a page
    size = heads * D * page
    bufs = [empty(pages * size), empty(pages * size), empty(4 * pages * heads), empty(4 * pages * heads)]
    cache = KVInt8Cache(*[b.ptr for b in bufs], pages, heads, D, page)
    rng = rng_of(6)
    table = np.array([[65535, 65536, 69999, 3]], np.int32)
    n = 4 * page
    x = rng.standard_normal((2, n, heads, D))
    kb, vb = bits(x[0], "f16"), bits(x[1], "f16")
    a = [dev(kb), dev(vb), dev(np.array([0, n], np.int32)), dev(np.zeros(1, np.int32)), dev(table)]
    ok(lib.ng_kv_int8_append(C.byref(cache), *[b.vp for b in a], 1, 4, n, n, None), "append")
    src, dst = dev(np.array([65535, 69999, 65536, 3], np.int32)), dev(np.array([69998, 7, 65534, 11], np.int32))
    ok(lib.ng_kv_int8_copy_pages(C.byref(cache), 1, src.vp, dst.vp, 4), "copy")
    k, v = (K.Cache(np.zeros((4, heads, page, D), np.int8), np.zeros((4, heads), np.float32)) for _ in "kv")
    small = np.arange(4, dtype=np.int32)[None]
    for c, xb in ((k, kb), (v, vb)):
        c.append(f32(xb, "f16").reshape(xb.shape), [0, n], [0], small)
    for t in (table, np.array([[69998, 65534, 7, 11]], np.int32)):
        o = [empty(2 * n * heads * D) for _ in "kv"]
        tb = dev(t)
        ok(lib.ng_kv_int8_read(C.byref(cache), o[0].vp, o[1].vp, a[2].vp, a[3].vp, tb.vp, 1, 4, n, n), "read")
        for buf, c in zip(o, (k, v)):
            got, want = get(buf, np.uint16, (n, heads, D)), c.read([0, n], [0], small)
            for row in range(n):
                assert_bits_equal(got[row], bits(want[row], "f16"), f"row {row}")


@pytest.mark.parametrize("layers,heads,D,page", [(1, 1, 64, 16), (5, 3, 192, 32), (40, 2, 128, 16)])
def test_copy_pages(lib, layers, heads, D, page):
    banner(f"kv copy pages layers={layers}")
    rng = rng_of(layers)
    pages = 40
    made = [random_cache(rng, pages, heads, page, D) for _ in range(layers)]
    dcs = [DeviceCache(*m) for m in made]
    order = rng.permutation(pages)
    src, dst = order[:15].astype(np.int32), order[15:30].astype(np.int32)
    src[4] = src[5]            # one page into two
    src[1], dst[2] = -1, -1    # nothing to copy
    src[3], dst[6] = pages, 2 ** 30
    caches = (KVInt8Cache * layers)(*[d.c for d in dcs])
    s, t = dev(src), dev(dst)
    ok(lib.ng_kv_int8_copy_pages(caches, layers, s.vp, t.vp, 15), "copy")
    for i, (d, m) in enumerate(zip(dcs, made)):
        for c in m:
            for a, b in zip(src, dst):
                if 0 <= a < pages and 0 <= b < pages:
                    c.codes[b], c.scales[b] = c.codes[a], c.scales[a]
        same(d, *m, f"layer {i}")


def test_captured_step(lib):
    """Append, copy and read as a graph, replayed after other contents came in."""
    banner("kv cache captured")
    rng = rng_of(8)
    heads, D, page = 2, 128, 16
    lens = [20, 33]
    table, pages, rest = random_table(rng, [x + 4 for x in lens], page)
    k, v = random_cache(rng, pages, heads, page, D)
    dc = DeviceCache(k, v)
    hip = HipRuntime()
    s = hip.stream()
    kb, vb = (dev(np.zeros((2, heads, D), np.uint16)) for _ in "kv")
    ctx, cu, tb = dev(np.array(lens, np.int32)), dev(np.array([0, 1, 2], np.int32)), dev(table)
    src, dst = dev(np.array([table[0, 0]], np.int32)), dev(np.array([rest[0]], np.int32))
    o = [empty(2 * 2 * heads * D) for _ in "kv"]

    def step():
        ok(lib.ng_kv_int8_append(C.byref(dc.c), kb.vp, vb.vp, cu.vp, ctx.vp, tb.vp, 2, table.shape[1], 2, 1, None), "append")
        ok(lib.ng_kv_int8_copy_pages(C.byref(dc.c), 1, src.vp, dst.vp, 1), "copy")
        ok(lib.ng_kv_int8_read(C.byref(dc.c), o[0].vp, o[1].vp, cu.vp, ctx.vp, tb.vp, 2, table.shape[1], 2, 1), "read")

    lib.ng_set_stream(s)
    try:
        g, ex = hip.capture(s, step)
    finally:
        lib.ng_set_stream(None)
    assert hip.kernel_nodes(g) == 3
    for t in range(3):
        x = rng.standard_normal((2, 2, heads, D)) * (1 + t)
        xb = bits(x, "f16")
        kb.upload(xb[0]), vb.upload(xb[1])
        pos = [n + t for n in lens]
        ctx.upload(np.array(pos, np.int32))
        hip.launch(ex, s)
        for c, b in ((k, xb[0]), (v, xb[1])):
            c.append(f32(b, "f16").reshape(b.shape), [0, 1, 2], pos, table)
            c.codes[rest[0]], c.scales[rest[0]] = c.codes[table[0, 0]], c.scales[table[0, 0]]
        same(dc, k, v, f"replay {t}")
        for buf, c in zip(o, (k, v)):
            got, want = get(buf, np.uint16, (2, heads, D)), c.read([0, 1, 2], pos, table)
            for row in range(2):
                assert_bits_equal(got[row], bits(want[row], "f16"), f"replay {t} row {row}")
    hip.destroy(g, ex)
