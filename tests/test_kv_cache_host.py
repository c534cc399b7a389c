"""The key/value cache on the CPU: what the entry points refuse, and the oracle against closed forms."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from neurogrid_amd import _lib
from neurogrid_amd._lib import KVInt8Cache, KVPages
from oracle import kv_oracle as K

P = 4096  # stands for a device pointer: no refused call reads it


def cache(**kw):
    c = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, num_pages=8, num_kv_heads=2, head_dim=128, page_size=16)
    c.update(kw)
    return KVInt8Cache(*c.values())


BAD_CACHES = [dict(k_codes=None), dict(v_scales=None), dict(num_pages=0), dict(num_kv_heads=0), dict(head_dim=96),
              dict(head_dim=512), dict(page_size=8), dict(page_size=24), dict(page_size=256), dict(k_codes=P + 8),
              dict(num_kv_heads=40000)]


def test_caches_that_are_refused(capfd):
    L = _lib.load()
    for kw in BAD_CACHES:
        c = C.byref(cache(**kw))
        assert L.ng_kv_int8_append(c, P, P, P, P, P, 1, 1, 1, 1, None) == -1, kw
        assert L.ng_kv_int8_read(c, P, P, P, P, P, 1, 1, 1, 1) == -1, kw
        assert L.ng_kv_int8_attention(P, P, c, P, P, P, 1, 1, 1, 1, 1, 2, 1.0, 0, 0, None, 0) == -1, kw
        assert L.ng_kv_int8_copy_pages(c, 1, P, P, 1) == -1, kw
    for f in (lambda: L.ng_kv_int8_append(None, P, P, P, P, P, 1, 1, 1, 1, None),
              lambda: L.ng_bf16_kv_int8_read(None, P, P, P, P, P, 1, 1, 1, 1),
              lambda: L.ng_bf16_kv_int8_attention(P, P, None, P, P, P, 1, 1, 1, 1, 1, 2, 1.0, 0, 0, None, 0),
              lambda: L.ng_kv_int8_copy_pages(None, 1, P, P, 1)):
        assert f() == -1
    assert "ng_kv_int8_append: head_dim 96 is not" in capfd.readouterr().err


@pytest.mark.parametrize("pre", ["ng_", "ng_bf16_"])
def test_batches_that_are_refused(pre, capfd):
    L = _lib.load()
    c = C.byref(cache())
    good = [P, P, P, P, P, 3, 4, 5, 6]  # k, v, cu, lens, table, batch, max_pages, total, longest
    bad = [(i, None) for i in range(5)] + [(5, 0), (5, 70000), (6, 0), (6, 1 << 29), (7, 0), (7, 2 ** 31 - 1), (8, 0),
                                           (8, -1), (0, P + 2), (1, P + 8)]
    for i, x in bad:
        a = list(good)
        a[i] = x
        assert getattr(L, pre + "kv_int8_append")(c, *a, None) == -1, (i, x)
        assert getattr(L, pre + "kv_int8_read")(c, *a) == -1, (i, x)
    # out, q, cache, cu, lens, table, batch, max_pages, total, max_q, max_kv, heads, scale, window, sinks, ws, bytes
    good = [P, P, c, P, P, P, 3, 4, 5, 6, 7, 4, 0.5, 0, 0, P, 64]
    bad = [(0, None), (1, None), (3, None), (4, None), (5, None), (6, 0), (6, 65536), (7, 0), (8, 0), (9, 0), (10, 0),
           (11, 0), (11, 3), (11, 40000), (12, math.nan), (12, math.inf), (12, -0.5), (12, 3e38), (13, -1), (14, -1), (15, P + 4),
           (0, P + 4), (1, P + 2)]
    for i, x in bad:
        a = list(good)
        a[i] = x
        assert getattr(L, pre + "kv_int8_attention")(*a) == -1, (i, x)
    for shift in (16, -16, 4 * 5 * 128 * 2 - 16):  # out inside q and q inside out
        a = list(good)
        a[0] = P + 65536 + shift
        a[1] = P + 65536
        assert getattr(L, pre + "kv_int8_attention")(*a) == -1, shift
    assert "neurogrid-amd: " + pre + "kv_int8_attention" in capfd.readouterr().err


def test_copies_that_are_refused():
    L = _lib.load()
    two = (KVInt8Cache * 2)(cache(), cache(num_pages=9))
    assert L.ng_kv_int8_copy_pages(two, 2, P, P, 1) == -1
    for n in (0, -1, 65):
        assert L.ng_kv_int8_copy_pages(two, n, P, P, 1) == -1
    one = C.byref(cache())
    assert L.ng_kv_int8_copy_pages(one, 1, None, P, 1) == -1
    assert L.ng_kv_int8_copy_pages(one, 1, P, None, 1) == -1
    assert L.ng_kv_int8_copy_pages(one, 1, P, P, 0) == -1


def test_pools_that_are_refused():
    L = _lib.load()
    good = dict(table=P, refs=P, max_seqs=4, max_pages=4, num_pages=16, page_size=16)
    Q = 1 << 20
    calls = [lambda p: L.ng_kv_pages_grow(p, P, P, P, P, P), lambda p: L.ng_kv_pages_fork(p, Q, P, P, Q),
             lambda p: L.ng_kv_pages_free(p, P, P), lambda p: L.ng_kv_pages_compact(p, P, P, 8, P)]
    for kw in (dict(table=None), dict(refs=None), dict(max_seqs=0), dict(max_pages=-1), dict(num_pages=0),
               dict(page_size=48), dict(max_pages=1 << 28), dict(max_seqs=1 << 23),
               dict(max_seqs=1 << 20, max_pages=1 << 12)):
        p = C.byref(KVPages(*{**good, **kw}.values()))
        assert all(f(p) == -1 for f in calls), kw
    assert all(f(None) == -1 for f in calls)
    p = C.byref(KVPages(*good.values()))
    for i in range(5):
        a = [P] * 5
        a[i] = None
        assert L.ng_kv_pages_grow(p, *a) == -1
    for i in range(4):
        a = [Q, P, P, Q]
        a[i] = None
        assert L.ng_kv_pages_fork(p, *a) == -1
    assert L.ng_kv_pages_fork(p, P + 32, P, P, Q) == -1     # new_table inside the table
    assert L.ng_kv_pages_fork(p, Q, P, P, P + 4) == -1      # new_lens inside lens
    assert L.ng_kv_pages_free(p, None, P) == -1 and L.ng_kv_pages_free(p, P, None) == -1
    assert L.ng_kv_pages_compact(p, P, P, 7, P) == -1       # fewer than num_pages / 2
    assert L.ng_kv_pages_compact(p, P, None, 8, P) == -1
    many = C.byref(KVPages(*{**good, "max_seqs": 9000}.values()))
    assert L.ng_kv_pages_grow(many, P, P, P, P, P) == -1


def test_workspace_size_of_refused_arguments_is_zero():
    L = _lib.load()
    assert L.ng_kv_int8_attention_workspace(None, 8, 1, 1, 1000) == 0
    c = C.byref(cache())
    for a in ((0, 1, 1, 1000), (3, 1, 1, 1000), (8, 0, 1, 1000), (8, 1, 0, 1000), (8, 1, 1, 0)):
        assert L.ng_kv_int8_attention_workspace(c, *a) == 0
    assert L.ng_kv_int8_attention_workspace(C.byref(cache(head_dim=100)), 8, 1, 1, 100000) == 0


def test_workspace_size():
    """As many slices as blocks are wanted, and never more bytes than that many outputs; any hints are taken."""
    L = _lib.load()
    c = C.byref(cache(num_kv_heads=8))
    row = 32 * (128 + 2) * 4  # a query's heads, fp32 outputs and (m, l)
    assert L.ng_kv_int8_attention_workspace(c, 32, 1, 1, 500) == 0         # too short to share out
    assert L.ng_kv_int8_attention_workspace(c, 32, 64, 1, 4096) == 0       # enough sequences
    n = L.ng_kv_int8_attention_workspace(c, 32, 1, 1, 131071)
    assert n % row == 0 and 32 <= n // row <= 64
    for a in ((32, 65535, 1, 2 ** 31 - 1), (32, 1, 2 ** 31 - 1, 2 ** 31 - 1), (32, 2 ** 31 - 1, 2 ** 31 - 1, 1)):
        assert L.ng_kv_int8_attention_workspace(c, *a) % row == 0


# ---------------------------------------------------------------- the oracle

def test_packing_is_a_permutation_and_its_formula():
    rng = np.random.default_rng(0)
    for D, page in ((64, 16), (192, 32), (256, 128)):
        codes = rng.integers(-127, 128, (2, 3, page, D)).astype(np.int8)
        k, v = K.pack_k(codes), K.pack_v(codes)
        assert (K.unpack_k(k, D, page) == codes).all() and (K.unpack_v(v, D, page) == codes).all()
        for _ in range(50):
            t, d = int(rng.integers(page)), int(rng.integers(D))
            base = (t // 16) * 16 * D + (d // 64) * 1024
            kg, e, tt = (d % 64) // 16, d % 16, t % 16
            assert k[1, 2, base + (16 * kg + tt) * 16 + e] == int(codes[1, 2, t, d]) + 128
            assert v[1, 2, base + (16 * kg + 4 * (tt // 4) + e % 4) * 16 + 4 * (e // 4) + tt % 4] == int(codes[1, 2, t, d]) + 128


def test_append_by_hand():
    c = K.Cache(np.zeros((2, 1, 16, 64), np.int8), np.full((2, 1), np.nan, np.float32))
    x = np.zeros((2, 1, 64), np.float32)
    x[0, 0, :3] = 127.0, -63.5, 0.5      # a step of 1: 127, -64 (ties to even), 0
    x[1, 0, 0] = 254.0                   # a step of 2: the first token's codes halve
    table = np.array([[1]], np.int32)
    assert c.append(x[:1], [0, 1], [0], table) == 0
    assert list(c.codes[1, 0, 0, :3]) == [127, -64, 0] and c.scales[1, 0] == 127
    assert c.append(x[1:], [0, 1], [1], table) == 0
    assert list(c.codes[1, 0, 0, :3]) == [64, -32, 0] and c.codes[1, 0, 1, 0] == 127 and c.scales[1, 0] == 254
    assert c.append(x, [0, 2], [15], table) == 1  # one past the table
    assert np.isnan(c.scales[0, 0])


def test_append_is_within_half_a_step():
    rng = np.random.default_rng(1)
    c = K.Cache(np.zeros((4, 2, 16, 64), np.int8), np.zeros((4, 2), np.float32))
    x = rng.standard_normal((40, 2, 64)).astype(np.float32)
    table = np.array([[2, 0, 3]], np.int32)
    c.append(x, [0, 40], [0], table)
    back = np.stack([c.read([0, 40], [0], table)[r] for r in range(40)])
    step = np.abs(x.reshape(40, -1, 64)).max()
    assert np.abs(back - x).max() <= step / 127 * (0.5 + 1e-4)


def test_attention_of_the_oracle_by_hand():
    """Equal scores give the mean of what is seen; a score far above the others gives its value."""
    codes = np.zeros((1, 1, 16, 64), np.int8)
    k, v = (K.Cache(codes.copy(), np.full((1, 1), 127, np.float32)) for _ in "kv")
    v.codes[0, 0, :, 0] = np.arange(16)
    table = np.zeros((1, 1), np.int32)
    q = np.zeros((2, 1, 64))
    q[:, 0, 1] = 1.0
    got = K.attention(q, k, v, [0, 2], [9], table, 1.0)
    assert math.isclose(got[0][0][0, 0], np.mean(range(8))) and math.isclose(got[1][0][0, 0], np.mean(range(9)))
    got = K.attention(q, k, v, [0, 2], [9], table, 1.0, window=3, sinks=2)
    assert math.isclose(got[1][0][0, 0], np.mean([0, 1, 6, 7, 8])) and got[1][5] == 5
    k.codes[0, 0, 4, 1] = 100
    assert math.isclose(K.attention(q, k, v, [0, 2], [9], table, 1.0)[1][0][0, 0], 4.0)
    assert (K.attention(q, k, v, [0, 2], [1], table, 1.0)[0][0] == 0).all()  # a query before the first token


def test_page_table_of_the_oracle_keeps_its_counts():
    rng = np.random.default_rng(2)
    page, R, W, pages = 16, 6, 8, 60
    table, refs, lens = np.full((R, W), -1, np.int32), np.zeros(pages, np.int32), np.zeros(R, np.int32)
    for _ in range(40):
        new = np.minimum(lens + rng.integers(0, 20, R), W * page).astype(np.int32)
        table, refs, src, dst, miss = K.grow(table, refs, lens, new, page)
        lens = lens if miss else new
        table, refs, lens = K.fork(table, refs, rng.integers(-1, R, R), lens, page)
        keep = np.maximum(lens - rng.integers(0, 25, R), 0).astype(np.int32)
        table, refs = K.free(table, refs, lens, keep, page)
        lens = np.minimum(lens, keep)
        if rng.random() < 0.3:
            table, refs, *_ = K.compact(table, refs, pages // 2)
            assert (np.diff((refs > 0).astype(int)) <= 0).all()
        assert (refs == np.bincount(table[table >= 0], minlength=pages)).all()
        assert ((table >= 0).sum(1) == -(-lens // page)).all()


# Without a device a launch is an error too: what is refused is told by its message.

def test_a_compactions_lists_are_at_most_2_30(capfd):
    """The kernel's index goes a stride past the capacity: it would wrap and never end."""
    L = _lib.load()
    p = C.byref(KVPages(P, P, 4, 4, 16, 16))
    for n in (2 ** 30 + 1, 2 ** 31 - 1):
        assert L.ng_kv_pages_compact(p, P, P, n, P) == -1
        assert f"ng_kv_pages_compact: capacity {n} is above 2^30" in capfd.readouterr().err


def test_page_copies_are_at_most_2_30(capfd):
    """The kernel's index goes a stride past the count: it would wrap, below the lists."""
    L = _lib.load()
    for n in (2 ** 30 + 1, 2 ** 31 - 1):
        assert L.ng_kv_int8_copy_pages(C.byref(cache()), 1, P, P, n) == -1
        assert f"ng_kv_int8_copy_pages: count {n} is above 2^30" in capfd.readouterr().err


@pytest.mark.parametrize("pre", ["ng_", "ng_bf16_"])
def test_a_batch_is_below_2_30_tokens(pre, capfd):
    """A start of 2^30 and as many rows would end at 2^31."""
    L = _lib.load()
    for total in (2 ** 30, 2 ** 30 + 1):
        assert getattr(L, pre + "kv_int8_read")(C.byref(cache()), P, P, P, P, P, 3, 4, total, 6) == -1
        assert "kv_int8_read: 2^30 tokens or more" in capfd.readouterr().err
