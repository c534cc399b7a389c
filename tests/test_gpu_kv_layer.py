"""The key/value cache and its attention as a program uses them: after q/k/v of the INT8 layer and before o, and with
a page table that grows, forks, is freed and moved together between steps."""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import C, HipRuntime, assert_bits_equal, banner, dev, empty, f32, get, ok
from kv_util import PREFIX, DeviceCache, attend, bits, check_attention, pool, random_cache, random_table, starts
from neurogrid_amd._lib import KVInt8Cache
from oracle import kv_oracle as K

pytestmark = pytest.mark.gpu


def blank(pages, heads, page, D):
    return tuple(K.Cache(np.zeros((pages, heads, page, D), np.int8), np.full((pages, heads), np.nan, np.float32))
                 for _ in "kv")


def test_attention_block_of_the_int8_layer(lib):
    """Norm, q/k/v and RoPE, append, attention, o: a prompt, then tokens one by one. Everything but the attention is
    bit for bit what its own tests check, so attention is compared on the q, k, v that the GPU made."""
    hidden, hq, hkv, D, page, theta = 512, 8, 2, 64, 16, 1e4
    banner("INT8 layer's attention block")
    rng = np.random.default_rng(21)
    ns = [hq * D, hkv * D, hkv * D]
    wq = [dev(rng.integers(-127, 128, (n, hidden)).astype(np.int8)) for n in ns]
    ws = [dev(rng.uniform(1e-3, 2e-3, n).astype(np.float32)) for n in ns]
    wo_h, so_h = rng.integers(-127, 128, (hidden, hq * D)).astype(np.int8), rng.uniform(1e-3, 2e-3, hidden).astype(np.float32)
    wo, so, wn = dev(wo_h), dev(so_h), dev(bits(1 + 0.05 * rng.standard_normal(hidden), "f16"))
    table, pages, _ = random_table(rng, [60], page)
    k, v = blank(pages, hkv, page, D)
    dc = DeviceCache(k, v)
    tb = dev(table)
    at = 0
    for n in (41, 1, 1, 3, 1):
        x = dev(bits(rng.standard_normal((n, hidden)), "f16"))
        y, q, kk, vv, o, out = (empty(2 * n * w) for w in (hidden, *ns, hq * D, hidden))
        pos = dev(np.arange(at, at + n, dtype=np.int32))
        ok(lib.ng_rmsnorm_qkv_rope_int8(y.vp, q.vp, kk.vp, vv.vp, x.vp, wn.vp, C.c_float(1e-5),
                                        (C.c_void_p * 3)(*[b.ptr for b in wq]), (C.c_void_p * 3)(*[b.ptr for b in ws]),
                                        pos.ip, n, hidden, hq, hkv, D, C.c_float(theta)), "qkv")
        cu, ctx, lens = (dev(np.array(a, np.int32)) for a in ([0, n], [at], [at + n]))
        ok(lib.ng_kv_int8_append(C.byref(dc.c), kk.vp, vv.vp, cu.vp, ctx.vp, tb.vp, 1, table.shape[1], n, n, None), "append")
        ok(lib.ng_kv_int8_attention(o.vp, q.vp, C.byref(dc.c), cu.vp, lens.vp, tb.vp, 1, table.shape[1], n, n, at + n,
                                    hq, C.c_float(1 / math.sqrt(D)), 0, 0, None, 0), "attention")
        ok(lib.cuda_gemm_int8(out.vp, o.vp, wo.vp, so.vp, n, hq * D, hidden, True), "o")
        for c, b in ((k, kk), (v, vv)):
            c.append(f32(get(b, np.uint16, (n, hkv, D)), "f16").reshape(n, hkv, D), [0, n], [at], table)
        got = dc.get()
        assert_bits_equal(got[0], k.codes, f"K codes at {at}")
        assert_bits_equal(got[1], v.codes, f"V codes at {at}")
        ob = get(o, np.uint16, (n, hq, D))
        check_attention(ob, "f16", D, K.attention(f32(get(q, np.uint16, (n, hq, D)), "f16").reshape(n, hq, D), k, v,
                                                  [0, n], [at + n], table, np.float32(1 / math.sqrt(D))))
        a = f32(ob, "f16").reshape(n, -1).astype(np.float64)
        w = wo_h.astype(np.float64) * so_h[:, None]
        want, mag = a @ w.T, np.abs(a) @ np.abs(w).T
        # fp16 rounding, and a sum of hq D products in fp32
        assert (np.abs(f32(get(out, np.uint16, (n, hidden)), "f16") - want)
                <= 2.0 ** -11 * np.abs(want) + 2.0 ** -24 * (hq * D + 2) * mag + 2.0 ** -25).all()
        at += n


@pytest.mark.parametrize("dtype,page", [("f16", 16), ("bf16", 32)])
def test_search_over_several_continuations(lib, dtype, page):
    """Rows fork, grow, copy what they share and write, attend; in between some are freed and the pool is compacted."""
    banner(f"kv search {dtype} page={page}")
    rng = np.random.default_rng(22)
    R, W, pages, hq, hkv, D = 6, 8, 60, 4, 2, 64
    k, v = blank(pages, hkv, page, D)
    dc = DeviceCache(k, v)
    table, refs, lens = np.full((R, W), -1, np.int32), np.zeros(pages, np.int32), np.zeros(R, np.int32)
    p, tb, rb = pool(table, refs, page)
    other = dev(np.full((R, W), -1, np.int32))
    src, dst, one, nl = empty(4 * pages), empty(4 * pages), empty(4), empty(4 * R)

    def state(t, r, tab, what):
        assert_bits_equal(get(tab, np.int32, (R, W)), t, what + ": table")
        assert_bits_equal(get(rb, np.int32, (pages,)), r, what + ": refs")

    def copy(n, s, d):
        ok(lib.ng_kv_int8_copy_pages(C.byref(dc.c), 1, src.vp, dst.vp, n), "copy")
        for c in (k, v):
            for a, b in zip(s, d):
                if a >= 0:
                    c.codes[b], c.scales[b] = c.codes[a], c.scales[a]

    for step in range(7):
        # every row takes new tokens: a prompt first, then one or two
        add = rng.integers(20, 40, R) if step == 0 else rng.integers(0, 3, R)
        new = (lens + add).astype(np.int32)
        old_b, new_b = dev(lens), dev(new)
        ok(lib.ng_kv_pages_grow(C.byref(p), old_b.vp, new_b.vp, src.vp, dst.vp, one.vp), "grow")
        table, refs, s, d, miss = K.grow(table, refs, lens, new, page)
        assert miss == 0 and get(one, np.int32, (1,))[0] == 0
        state(table, refs, tb, f"step {step} grow")
        copy(R, s, d)
        n = int(add.sum())
        if n:
            cu = starts(add)
            x = rng.standard_normal((2, n, hkv, D)) * (1 + 0.2 * step)
            kb, vb, qb = bits(x[0], dtype), bits(x[1], dtype), bits(rng.standard_normal((n, hq, D)), dtype)
            args = [dev(kb), dev(vb), dev(cu), old_b, tb]
            ok(getattr(lib, PREFIX[dtype] + "kv_int8_append")(C.byref(dc.c), *[a.vp for a in args], R, W, n,
                                                              int(add.max()), None), "append")
            for c, b in ((k, kb), (v, vb)):
                c.append(f32(b, dtype).reshape(b.shape), cu, lens, table)
            got = attend(lib, dtype, dc, qb, cu, new, table, 0.125)
            check_attention(got, dtype, D, K.attention(f32(qb, dtype).reshape(qb.shape), k, v, cu, new, table,
                                                       np.float32(0.125)))
        lens = new
        used = np.unique(table[table >= 0])
        kc, vc, ks, vs = dc.get()
        assert_bits_equal(kc[used], k.codes[used], f"step {step}: K")
        assert_bits_equal(vc[used], v.codes[used], f"step {step}: V")
        # the best rows go on
        parents = rng.integers(-1, R, R).astype(np.int32)
        lens_b, par = dev(lens), dev(parents)
        ok(lib.ng_kv_pages_fork(C.byref(p), other.vp, par.vp, lens_b.vp, nl.vp), "fork")
        table, refs, lens = K.fork(table, refs, parents, lens, page)
        tb, other = other, tb
        p.table = tb.ptr
        state(table, refs, tb, f"step {step} fork")
        assert_bits_equal(get(nl, np.int32, (R,)), lens, "lens")
        if step % 2:
            keep = np.where(np.arange(R) == step % R, 0, lens).astype(np.int32)
            a, b = dev(lens), dev(keep)
            ok(lib.ng_kv_pages_free(C.byref(p), a.vp, b.vp), "free")
            table, refs = K.free(table, refs, lens, keep, page)
            lens = keep
        if step % 3 == 2:
            ok(lib.ng_kv_pages_compact(C.byref(p), src.vp, dst.vp, pages // 2, one.vp), "compact")
            table, refs, s, d, moves = K.compact(table, refs, pages // 2)
            assert get(one, np.int32, (1,))[0] == moves
            copy(pages // 2, s, d)
        state(table, refs, tb, f"step {step} end")


@pytest.mark.parametrize("new", [1, 70])
def test_attention_past_4_gib(lib, new):
    """Pages behind the first 4 GiB of codes, one sequence's on both sides of it."""
    banner(f"kv attention past 4 GiB new={new}")
    heads, hq, D, page, pages = 8, 16, 128, 64, 70000
    size = heads * D * page
    rng = np.random.default_rng(23)
    bufs = [empty(pages * size), empty(pages * size), empty(4 * pages * heads), empty(4 * pages * heads)]
    cache = KVInt8Cache(*[b.ptr for b in bufs], pages, heads, D, page)
    table, small = np.array([[65535, 65536, 69999, 3]], np.int32), np.arange(4, dtype=np.int32)[None]
    n = 4 * page - 9
    x = rng.standard_normal((2, n, heads, D))
    a = [dev(bits(x[0], "f16")), dev(bits(x[1], "f16")), dev(np.array([0, n], np.int32)), dev(np.zeros(1, np.int32)), dev(table)]
    ok(lib.ng_kv_int8_append(C.byref(cache), *[b.vp for b in a], 1, 4, n, n, None), "append")
    k, v = blank(4, heads, page, D)
    for c, y in ((k, x[0]), (v, x[1])):
        b = bits(y, "f16")
        c.append(f32(b, "f16").reshape(b.shape), [0, n], [0], small)

    class Big:
        c = cache

    qb = bits(rng.standard_normal((new, hq, D)), "f16")
    got = attend(lib, "f16", Big, qb, [0, new], [n], table, 0.1)
    check_attention(got, "f16", D, K.attention(f32(qb, "f16").reshape(qb.shape), k, v, [0, new], [n], small, np.float32(0.1)))


def test_two_streams_at_once(lib):
    """Calls of two streams that overlap, each with a workspace of its own, give what they give alone."""
    banner("kv attention on two streams")
    hip = HipRuntime()
    jobs = []
    for i, (new, kv) in enumerate(((1, 20000), (64, 3000))):
        rng = np.random.default_rng(30 + i)
        table, pages, _ = random_table(rng, [kv], 16)
        dc = DeviceCache(*random_cache(rng, pages, 2, 16, 128))
        qb = bits(rng.standard_normal((new, 8, 128)), "f16")
        alone = attend(lib, "f16", dc, qb, [0, new], [kv], table, 0.1)
        n = lib.ng_kv_int8_attention_workspace(C.byref(dc.c), 8, 1, new, kv)
        assert n > 0
        jobs.append((hip.stream(), dc, new, kv, table.shape[1], alone, n, empty(n), dev(qb), empty(qb.nbytes),
                     dev(np.array([0, new], np.int32)), dev(np.array([kv], np.int32)), dev(table)))
    try:
        for _ in range(20):
            for s, dc, new, kv, width, alone, n, ws, q, o, cu, lens, tb in jobs:
                lib.ng_set_stream(s)
                ok(lib.ng_kv_int8_attention(o.vp, q.vp, C.byref(dc.c), cu.vp, lens.vp, tb.vp, 1, width, new, new, kv, 8,
                                            C.c_float(0.1), 0, 0, ws.vp, n), "attention")
    finally:
        lib.ng_set_stream(None)
    for s, dc, new, kv, width, alone, n, ws, q, o, *_ in jobs:
        assert_bits_equal(get(o, np.uint16, alone.shape), alone, f"new={new}")
