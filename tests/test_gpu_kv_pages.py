"""The page table on the GPU: grow, fork, free and compact against the oracle, integer for integer."""
from __future__ import annotations

import numpy as np
import pytest

from gpu_util import C, HipRuntime, assert_bits_equal, banner, dev, empty, get, ok
from kv_util import pool, random_table
from oracle import kv_oracle as K

pytestmark = pytest.mark.gpu


def start(seed, rows, width, page, extra, most=None):
    """A table of private pages and its counts, lengths drawn up to `most` tokens."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, (most or width * page) + 1, rows).astype(np.int32)
    table, pages, _ = random_table(rng, lens, page, spare=extra, width=width)
    refs = np.zeros(pages, np.int32)
    refs[table[table >= 0]] = 1
    return rng, table, refs, lens


def run_grow(lib, table, refs, old, new, page):
    p, t, r = pool(table, refs, page)
    R = len(old)
    o, n = dev(np.asarray(old, np.int32)), dev(np.asarray(new, np.int32))
    src, dst, miss = dev(np.full(R, 77, np.int32)), dev(np.full(R, 77, np.int32)), dev(np.full(1, 77, np.int32))
    ok(lib.ng_kv_pages_grow(C.byref(p), o.vp, n.vp, src.vp, dst.vp, miss.vp), "grow")
    return (get(t, np.int32, table.shape), get(r, np.int32, refs.shape), get(src, np.int32, (R,)),
            get(dst, np.int32, (R,)), int(get(miss, np.int32, (1,))[0]))


def run_fork(lib, table, refs, parents, lens, page):
    p, t, r = pool(table, refs, page)
    a, b = dev(np.asarray(parents, np.int32)), dev(np.asarray(lens, np.int32))
    nt, nl = dev(np.full(table.shape, 77, np.int32)), dev(np.full(len(lens), 77, np.int32))
    ok(lib.ng_kv_pages_fork(C.byref(p), nt.vp, a.vp, b.vp, nl.vp), "fork")
    assert_bits_equal(get(t, np.int32, table.shape), table, "the old table")
    return get(nt, np.int32, table.shape), get(r, np.int32, refs.shape), get(nl, np.int32, (len(lens),))


def same(got, want, what):
    for i, (a, b) in enumerate(zip(got, want)):
        assert_bits_equal(np.asarray(a), np.asarray(b), f"{what}: result {i}")


# rows, table width, page, free pages
POOLS = [(1, 1, 16, 1), (3, 5, 32, 10), (64, 40, 16, 400), (1500, 7, 64, 4000), (20, 600, 128, 9000)]


@pytest.mark.parametrize("rows,width,page,extra", POOLS)
def test_grow(lib, rows, width, page, extra):
    banner(f"kv pages grow rows={rows} width={width}")
    rng, table, refs, lens = start(rows, rows, width, page, extra)
    new = np.minimum(lens + rng.integers(-page, 3 * page, rows), width * page).astype(np.int32)
    want = K.grow(table, refs, lens, new, page)
    same(run_grow(lib, table, refs, lens, new, page), want, "grow")
    # a row's growth is refused as a whole when pages are too few
    full = refs.copy()
    free = np.flatnonzero(full == 0)
    need = int((want[1] != refs).sum())
    if need:
        full[free[:len(free) - need + 1]] = 5
        got = run_grow(lib, table, full, lens, new, page)
        assert got[4] == 1
        same(got, K.grow(table, full, lens, new, page), "too few")
        full[free] = 0
        full[free[:len(free) - need]] = 5
        same(run_grow(lib, table, full, lens, new, page), K.grow(table, full, lens, new, page), "just enough")


def test_grow_past_the_table_is_refused(lib):
    banner("kv pages grow past the table")
    _, table, refs, lens = start(5, 4, 3, 16, 100)
    for new in ([0, 49, 0, 0], [2 ** 31 - 1] * 4, [48, 48, 48, 48]):
        same(run_grow(lib, table, refs, lens, new, 16), K.grow(table, refs, lens, new, 16), str(new))


@pytest.mark.parametrize("rows,width,page,extra", POOLS[1:])
def test_fork_then_grow_copies_what_is_shared(lib, rows, width, page, extra):
    banner(f"kv pages fork rows={rows} width={width}")
    rng, table, refs, lens = start(rows + 1, rows, width, page, extra + 2 * rows, most=(width - 1) * page)
    parents = rng.integers(-1, rows, rows).astype(np.int32)
    parents[0] = rows + 3
    got = run_fork(lib, table, refs, parents, lens, page)
    want = K.fork(table, refs, parents, lens, page)
    same(got, want, "fork")
    t, c, n = want
    assert (c == np.bincount(t[t >= 0], minlength=len(c))).all()
    new = (n + rng.integers(0, 2, rows)).astype(np.int32)
    want = K.grow(t, c, n, new, page)
    same(run_grow(lib, t, c, n, new, page), want, "grow")
    assert want[4] == 0 and (rows < 10 or (want[2] >= 0).any())


@pytest.mark.parametrize("rows,width,page,extra", POOLS)
def test_free(lib, rows, width, page, extra):
    banner(f"kv pages free rows={rows} width={width}")
    rng, table, refs, lens = start(rows + 2, rows, width, page, extra)
    table, refs, lens = K.fork(table, refs, rng.integers(0, rows, rows), lens, page)
    keep = np.where(rng.random(rows) < 0.5, 0, rng.integers(-1, width * page + 2, rows)).astype(np.int32)
    p, t, r = pool(table, refs, page)
    o, k = dev(lens), dev(keep)
    ok(lib.ng_kv_pages_free(C.byref(p), o.vp, k.vp), "free")
    same((get(t, np.int32, table.shape), get(r, np.int32, refs.shape)), K.free(table, refs, lens, keep, page), "free")


@pytest.mark.parametrize("rows,width,page,extra", POOLS + [(300, 64, 16, 0), (8, 64, 16, 70000)])
def test_compact(lib, rows, width, page, extra):
    banner(f"kv pages compact rows={rows} width={width}")
    rng, table, refs, lens = start(rows + 3, rows, width, page, extra)
    table, refs, lens = K.fork(table, refs, rng.integers(-1, rows, rows), lens, page)
    for cap in (max(1, len(refs) // 2), len(refs) + 5):
        p, t, r = pool(table, refs, page)
        src, dst, mv = dev(np.full(cap, 77, np.int32)), dev(np.full(cap, 77, np.int32)), dev(np.full(1, 77, np.int32))
        ok(lib.ng_kv_pages_compact(C.byref(p), src.vp, dst.vp, cap, mv.vp), "compact")
        want = K.compact(table, refs, cap)
        same((get(t, np.int32, table.shape), get(r, np.int32, refs.shape), get(src, np.int32, (cap,)),
              get(dst, np.int32, (cap,)), get(mv, np.int32, (1,))[0]), want, f"compact {cap}")


def test_bad_entries_are_not_followed(lib):
    """Entries and parents that are no numbers of pages or rows."""
    banner("kv pages bad entries")
    table = np.array([[0, 99, -3], [2 ** 31 - 1, 1, 2], [3, -1, -1]], np.int32)
    refs = np.array([1, 1, 1, 1, 0, 0, 0], np.int32)
    lens = np.array([40, 48, 7], np.int32)
    nt, c, n = run_fork(lib, table, refs, [1, 5, 0], lens, 16)
    assert (nt[1] == -1).all() and list(n) == [48, 0, 40]
    assert list(c) == [1, 1, 1, 0, 0, 0, 0]
    p, t, r = pool(table, refs, 16)
    o, k = dev(lens), dev(np.zeros(3, np.int32))
    ok(lib.ng_kv_pages_free(C.byref(p), o.vp, k.vp), "free")
    assert list(get(r, np.int32, (7,))) == [0] * 7 and (get(t, np.int32, (3, 3)) == -1).all()
    got = run_grow(lib, table, refs, [40, 48, 7], [41, 48, 33], 16)  # row 0's last entry is no page: nothing to share
    assert got[4] == 0 and list(got[0][2]) == [3, 4, 5] and list(got[1]) == [1, 1, 1, 1, 1, 1, 0]


def test_a_captured_step_of_table_work(lib):
    """fork, grow and free captured, replayed on tables that changed in between."""
    banner("kv pages captured")
    page = 16
    rng, table, refs, lens = start(11, 12, 9, page, 60, most=100)
    p, t, r = pool(table, refs, page)
    R = 12
    nt, nl = empty(table.nbytes), empty(4 * R)
    par, old = dev(np.zeros(R, np.int32)), dev(lens)
    new, keep = dev(np.zeros(R, np.int32)), dev(np.zeros(R, np.int32))
    src, dst, miss = empty(4 * R), empty(4 * R), empty(4)
    p2 = type(p)(nt.ptr, r.ptr, R, 9, len(refs), page)
    hip = HipRuntime()
    s = hip.stream()

    def step():
        ok(lib.ng_kv_pages_fork(C.byref(p), nt.vp, par.vp, old.vp, nl.vp), "fork")
        ok(lib.ng_kv_pages_grow(C.byref(p2), nl.vp, new.vp, src.vp, dst.vp, miss.vp), "grow")
        ok(lib.ng_kv_pages_free(C.byref(p2), new.vp, keep.vp), "free")

    lib.ng_set_stream(s)
    try:
        g, ex = hip.capture(s, step)
    finally:
        lib.ng_set_stream(None)
    hip.kernel_nodes(g)
    for i in range(3):
        t.upload(table), r.upload(refs)
        parents = rng.integers(-1, R, R).astype(np.int32)
        ft, fc, fn = K.fork(table, refs, parents, lens, page)
        grown = (fn + rng.integers(1, 30, R)).astype(np.int32)
        kept = (grown - rng.integers(0, 40, R)).astype(np.int32)
        gt, gc, gs, gd, gm = K.grow(ft, fc, fn, grown, page)
        assert gm == 0
        et, ec = K.free(gt, gc, grown, kept, page)
        par.upload(parents), new.upload(grown), keep.upload(kept)
        hip.launch(ex, s)
        same((get(nt, np.int32, table.shape), get(r, np.int32, refs.shape), get(src, np.int32, (R,)),
              get(dst, np.int32, (R,)), get(miss, np.int32, (1,))[0]), (et, ec, gs, gd, gm), f"replay {i}")
    hip.destroy(g, ex)
