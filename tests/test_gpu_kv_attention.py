"""Attention over the 8-bit key/value cache on the GPU, against the oracle in 64 bits.

The bound of a row is worked out from its own scores and values (kv_util.bound).
Pages that no sequence holds have NaN scales, entries of the table behind a
sequence's pages are rubbish, the workspace is filled with NaN before a call.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from gpu_util import C, HipRuntime, assert_bits_equal, banner, dev, empty, f32, get, ok
from kv_util import PREFIX, DeviceCache, attend, bits, bound, check_attention, random_cache, random_table, starts
from oracle import kv_oracle as K

pytestmark = pytest.mark.gpu


def problem(seed, dtype, hq, hkv, D, page, new, kv, gain=1.5):
    rng = np.random.default_rng(seed)
    table, pages, rest = random_table(rng, kv, page, width=max(1, -(-max(kv) // page)) + 3)
    k, v = random_cache(rng, pages, hkv, page, D)
    for c in (k, v):
        c.scales[rest] = np.nan
    for b, n in enumerate(kv):  # rubbish behind the sequence's pages
        table[b, -(-n // page):] = rng.choice([-1, -7, pages, 2 ** 31 - 1, rest[0]], table.shape[1] - -(-n // page))
    q = rng.standard_normal((sum(new) + 1, hq, D)) * gain
    return table, k, v, bits(q, dtype)


def check(lib, seed, dtype, hq, hkv, D, page, new, kv, window=0, sinks=0, scale=None, gain=1.5, **kw):
    table, k, v, qb = problem(seed, dtype, hq, hkv, D, page, new, kv, gain)
    scale = scale if scale is not None else 1 / math.sqrt(D)
    cu = starts(new)
    got = attend(lib, dtype, DeviceCache(k, v), qb, cu, kv, table, scale, window, sinks, **kw)
    q = f32(qb, dtype).reshape(qb.shape)
    check_attention(got, dtype, D, K.attention(q, k, v, cu, kv, table, np.float32(scale), window, sinks))
    return got


# query heads, key/value heads, D, page: multi-head, grouped by 4, 8, 7 and 16, multi-query; every D and page size
LAYOUTS = [(4, 4, 128, 16), (8, 2, 64, 16), (32, 4, 64, 32), (7, 1, 128, 64), (16, 1, 256, 16), (6, 3, 192, 128),
           (40, 2, 128, 16)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda c: "x".join(map(str, c)))
def test_single_tokens(lib, layout, dtype):
    banner(f"kv attention decode {layout} {dtype}")
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 300, 1023]
    check(lib, 1, dtype, *layout, [1] * len(kv), kv)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda c: "x".join(map(str, c)))
def test_prompts_and_chunks(lib, layout, dtype):
    banner(f"kv attention prompts {layout} {dtype}")
    hq = layout[0]
    new = [1, 70, 5, 0, 33, 64]
    kv = [1, 70, 130, 40, 33, 200]
    check(lib, 2, dtype, *layout, new, kv)


@pytest.mark.parametrize("new,kv", [(2, 500), (3, 77), (4, 1000), (8, 64), (16, 333), (17, 400), (40, 41)])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_a_few_queries(lib, new, kv, group):
    banner(f"kv attention new={new} kv={kv} group={group}")
    check(lib, 3, "f16", 2 * group, 2, 128, 16, [new, new], [kv, kv + 5])


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (64, 4), (100, 17), (128, 64), (130, 200), (5000, 3),
                                          (0, 9), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("new", [1, 90])
def test_sliding_window_and_first_tokens(lib, new, window, sinks):
    banner(f"kv attention window={window} sinks={sinks} new={new}")
    check(lib, 4, "f16", 4, 1, 128, 16, [new] * 3, [700, 91, 129], window, sinks)
    check(lib, 5, "bf16", 4, 2, 64, 64, [new] * 2, [700, 300], window, sinks)


def test_long_sequences_are_shared_out(lib):
    """One sequence among short ones, long enough to be split, in every way of giving room for it."""
    banner("kv attention split")
    kv = [9000, 1, 0, 700, 4097]
    a = check(lib, 6, "f16", 8, 2, 128, 16, [1] * 5, kv)
    b = check(lib, 6, "f16", 8, 2, 128, 16, [1] * 5, kv, workspace=None)
    assert np.abs(f32(a, "f16") - f32(b, "f16")).max() < 1e-2
    check(lib, 6, "f16", 8, 2, 128, 16, [1] * 5, kv, workspace=40000)
    check(lib, 6, "f16", 8, 2, 128, 16, [1] * 5, kv, workspace=4096)
    check(lib, 6, "f16", 8, 2, 128, 16, [1] * 5, kv, max_kv=100)       # longer than was said
    check(lib, 6, "f16", 8, 2, 128, 16, [1] * 5, kv, max_kv=2 ** 30)   # much shorter
    check(lib, 6, "bf16", 8, 2, 64, 16, [20] * 5, kv, window=5000, sinks=100)
    check(lib, 6, "bf16", 8, 8, 128, 16, [3] * 5, [5000, 2, 3, 4, 5], max_q=1)


@pytest.mark.parametrize("new", [1, 40])
def test_windows_in_long_sequences_are_shared_out(lib, new):
    """A window that is a small part of the context, with first tokens, split and not."""
    banner(f"kv attention window split new={new}")
    for window, sinks in ((2000, 4), (1500, 700), (64, 5000)):
        check(lib, 20, "f16", 8, 2, 128, 16, [new, new], [9000, 300], window, sinks)
        check(lib, 20, "f16", 8, 2, 128, 16, [new, new], [9000, 300], window, sinks, workspace=None)


def test_rows_that_see_nothing(lib):
    """No tokens, fewer tokens than queries, no page where the tokens should be: zeros, and never NaN."""
    banner("kv attention empty rows")
    for seed, new, kv in ((7, [1, 3, 70, 2], [0, 1, 5, -4]), (8, [5, 1], [2, 17])):
        table, k, v, qb = problem(seed, "f16", 8, 2, 128, 16, new, [max(n, 0) for n in kv])
        if seed == 8:
            table[1, :] = -1
        cu = starts(new)
        for ws in ("asked", None):
            got = attend(lib, "f16", DeviceCache(k, v), qb, cu, kv, table, 0.1, workspace=ws)
            refs = K.attention(f32(qb, "f16").reshape(qb.shape), k, v, cu, kv, table, np.float32(0.1))
            check_attention(got, "f16", 128, refs)
            assert (got[0] == 0).all() if seed == 7 else (got[0:3] == 0).all() and (got[5] == 0).all()


def test_holes_and_lengths_past_the_table(lib):
    banner("kv attention holes")
    new, kv = [1, 40, 1], [400, 400, 400]
    table, k, v, qb = problem(9, "f16", 4, 2, 64, 16, new, kv)
    table = np.ascontiguousarray(table[:, :20])   # 320 tokens of 400
    table[0, 3], table[1, 0], table[2, 5:9] = -1, 10 ** 9, -5
    cu = starts(new)
    got = attend(lib, "f16", DeviceCache(k, v), qb, cu, kv, table, 0.125)
    check_attention(got, "f16", 64, K.attention(f32(qb, "f16").reshape(qb.shape), k, v, cu, kv, table, np.float32(0.125)))


@pytest.mark.parametrize("new", [1, 50])
def test_not_finite_queries_stay_in_their_row(lib, new):
    banner(f"kv attention NaN rows new={new}")
    table, k, v, qb = problem(10, "f16", 4, 1, 128, 16, [new, new], [300, 60])
    cu = starts([new, new])
    clean = attend(lib, "f16", DeviceCache(k, v), qb, cu, [300, 60], table, 0.1)
    qb[0, 1, 5], qb[new, 2, 0] = 0x7E00, 0x7C00
    got = attend(lib, "f16", DeviceCache(k, v), qb, cu, [300, 60], table, 0.1)
    hit = np.zeros((len(qb), 4), bool)
    hit[0, 1] = hit[new, 2] = True
    assert np.isnan(f32(got, "f16").reshape(got.shape)[hit]).all()
    assert_bits_equal(got[~hit], clean[~hit], "other rows")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_large_scores_and_uneven_scales(lib, dtype, new):
    """Scores of hundreds (one token takes all), V scales over 12 orders of magnitude, pages of zeros."""
    banner(f"kv attention extremes {dtype} new={new}")
    kv = [200, 33]
    table, k, v, qb = problem(11, dtype, 4, 2, 128, 16, [new] * 2, kv, gain=60.0)
    used = np.unique(table[(table >= 0) & (table < len(k.scales))])
    rng = np.random.default_rng(12)
    v.scales[used] *= (10.0 ** rng.uniform(-9, 3 if dtype == "bf16" else 1, v.scales[used].shape)).astype(np.float32)
    k.scales[table[0, 2]], k.codes[table[0, 2]] = 0, 0
    v.scales[table[0, 4]], v.codes[table[0, 4]] = 0, 0
    cu = starts([new] * 2)
    got = attend(lib, dtype, DeviceCache(k, v), qb, cu, kv, table, 1.0)
    check_attention(got, dtype, 128, K.attention(f32(qb, dtype).reshape(qb.shape), k, v, cu, kv, table, 1.0))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_many_small_weights_beside_a_large_one(lib, dtype, new):
    """One token, whose value is 0, outweighs each of the others by 2^25.5: together they are the output."""
    banner(f"kv attention small weights {dtype} {new}")
    hq, hkv, D, page, n = 4, 1, 128, 16, 60000
    table = np.arange(-(-n // page), dtype=np.int32)[None]
    shape = (table.size, hkv, page, D)
    rng = np.random.default_rng(8)
    kc, vc = np.zeros(shape, np.int8), rng.integers(100, 128, shape).astype(np.int8)
    kc[0, 0, 0], vc[0, 0, 0] = 127, 0
    k, v = (K.Cache(c, np.full((table.size, hkv), m, np.float32)) for c, m in ((kc, 1.0), (vc, 3.0)))
    qb = bits(np.ones((new, hq, D)), dtype)
    scale = float(np.float32(25.5 * math.log(2) / D))
    got = attend(lib, dtype, DeviceCache(k, v), qb, starts([new]), [n], table, scale, workspace=None)  # one slice
    check_attention(got, dtype, D, K.attention(f32(qb, dtype).reshape(qb.shape), k, v, starts([new]), [n], table,
                                               np.float32(scale)))


@pytest.mark.parametrize("gain", [1e-6, 1e4, 1e30])
def test_bf16_queries_of_any_size(lib, gain):
    """bf16 holds queries that fp16 cannot; the scale makes up for it."""
    banner(f"kv attention bf16 gain={gain}")
    check(lib, 13, "bf16", 4, 2, 128, 16, [1, 40], [100, 90], scale=0.1 / gain if gain < 1e20 else 1e-31, gain=gain)


@pytest.mark.parametrize("new", [1, 40])
def test_bf16_values_at_the_ends_of_the_type(lib, new):
    """Sums of values near 3e38 pass fp32's range, their mean does not; values near 1e-37 keep their precision."""
    banner(f"kv attention bf16 V extremes new={new}")
    for m in (3.38e38, 2e-37):
        table, k, v, qb = problem(17, "bf16", 4, 2, 128, 16, [new] * 2, [500, 90])
        used = np.unique(table[(table >= 0) & (table < len(k.scales))])
        v.scales[used] = np.float32(m) * np.float32(0.9) ** (used[:, None] % 7)
        cu = starts([new] * 2)
        got = attend(lib, "bf16", DeviceCache(k, v), qb, cu, [500, 90], table, 0.05)
        check_attention(got, "bf16", 128, K.attention(f32(qb, "bf16").reshape(qb.shape), k, v, cu, [500, 90], table,
                                                      np.float32(0.05)))


def test_scale_zero_is_the_mean(lib):
    banner("kv attention scale 0")
    check(lib, 14, "f16", 4, 2, 64, 16, [1, 30], [100, 30], scale=0.0)


def test_output_in_the_queries_place_and_two_calls_agree(lib):
    banner("kv attention in place, repeated")
    table, k, v, qb = problem(15, "f16", 8, 2, 128, 16, [1, 40, 1], [2000, 300, 50])
    dc = DeviceCache(k, v)
    cu, kv = starts([1, 40, 1]), [2000, 300, 50]
    first = attend(lib, "f16", dc, qb, cu, kv, table, 0.1)
    assert_bits_equal(attend(lib, "f16", dc, qb, cu, kv, table, 0.1)[:-1], first[:-1], "again")
    qd = dev(qb)
    b = [dev(cu), dev(np.array(kv, np.int32)), dev(table)]
    n = lib.ng_kv_int8_attention_workspace(C.byref(dc.c), 8, 3, 40, 2000)
    ws = empty(max(n, 1))
    ok(lib.ng_kv_int8_attention(qd.vp, qd.vp, C.byref(dc.c), *[x.vp for x in b], 3, table.shape[1], 42, 40, 2000, 8,
                                C.c_float(0.1), 0, 0, ws.vp, n), "attention")
    assert_bits_equal(get(qd, np.uint16, qb.shape)[:-1], first[:-1], "in place")


def test_captured_and_replayed_with_growing_lengths(lib):
    banner("kv attention captured")
    table, k, v, qb = problem(16, "f16", 8, 2, 128, 16, [1, 1], [3000, 900])
    qb = qb[:2]
    dc = DeviceCache(k, v)
    hip = HipRuntime()
    s = hip.stream()
    qd, od, cu, lens, tb = dev(qb), empty(qb.nbytes), dev(starts([1, 1])), dev(np.array([1, 1], np.int32)), dev(table)
    n = lib.ng_kv_int8_attention_workspace(C.byref(dc.c), 8, 2, 1, 3000)
    ws = empty(max(n, 1))

    def call():
        ok(lib.ng_kv_int8_attention(od.vp, qd.vp, C.byref(dc.c), cu.vp, lens.vp, tb.vp, 2, table.shape[1], 2, 1, 3000,
                                    8, C.c_float(0.1), 0, 0, ws.vp, n), "attention")

    lib.ng_set_stream(s)
    try:
        g, ex = hip.capture(s, call)
    finally:
        lib.ng_set_stream(None)
    hip.kernel_nodes(g)
    for kv in ([3000, 900], [5, 0], [1500, 64], [3000, 900]):
        lens.upload(np.array(kv, np.int32))
        od.upload(np.full(qb.shape, 0x7E00, np.uint16))
        hip.launch(ex, s)
        got = get(od, np.uint16, qb.shape)
        check_attention(got, "f16", 128, K.attention(f32(qb, "f16").reshape(qb.shape), k, v, [0, 1, 2], kv, table,
                                                     np.float32(0.1)))
    hip.destroy(g, ex)
