"""The 8-bit paged key/value cache and the attention that reads it, as timed cases.

Four kinds of pass, each over its range of sizes, types and options:

  append     the new tokens of a batch written into the cache (a scale for each
             page and head), and read back as the cache holds them
  attention  queries of a batch against their sequences' cached keys and values:
             one token each (decode), whole prompts, chunks of a prompt behind
             a context, with and without a sliding window and first tokens that
             stay visible
  fork       one step of a search over several continuations: rows of the page
             table become forks of others, every row grows by a token, shared
             pages that it writes are copied
  compact    the used pages of a pool moved to its front, the page table renamed

With `own` false a pass is made of elementary torch operations in 32 bits; with
`own` true it is the calls that a host program makes of libgpu_engine.so. Head
layouts are those of neurogrid_amd.workloads and of the benchmark.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

own = False

# query heads, key/value heads, head dim
HEADS = {
    "tinyllama": (32, 4, 64),
    "llama2_7b": (32, 32, 128),
    "mistral7b": (32, 8, 128),
    "llama2_13b": (40, 40, 128),
    "mistral_nemo": (32, 8, 128),
    "wide_head": (8, 1, 256),
}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


def listed():
    return [
        # One user's token of a step: the smallest write there is.
        {"name": "append_t1", "kind": "append", "heads": "mistral7b", "dtype": "f16", "page": 16, "batch": 1,
         "new": 1, "context": 1003},
        # The tokens of a decoding batch, contexts of all lengths.
        {"name": "append_b64", "kind": "append", "heads": "mistral_nemo", "dtype": "bf16", "page": 16, "batch": 64,
         "new": 1, "context": 4093},
        # Three prompts of uneven length behind short contexts.
        {"name": "append_prompt", "kind": "append", "heads": "mistral7b", "dtype": "f16", "page": 16, "batch": 3,
         "new": 4096, "context": 100},
        # The smallest attention: a single user's token early in a conversation.
        {"name": "decode_b1_kv500", "kind": "attention", "heads": "tinyllama", "dtype": "f16", "page": 16, "batch": 1,
         "new": 1, "context": 499, "window": 0, "sinks": 0},
        # A full decoding batch, uneven contexts: what serving spends its time on.
        {"name": "decode_b64_kv4096", "kind": "attention", "heads": "mistral7b", "dtype": "f16", "page": 16,
         "batch": 64, "new": 1, "context": 4095, "window": 0, "sinks": 0},
        # One user with a whole book in the context: the sequence has to be shared out.
        {"name": "decode_b1_kv131071", "kind": "attention", "heads": "mistral_nemo", "dtype": "bf16", "page": 16,
         "batch": 1, "new": 1, "context": 131070, "window": 0, "sinks": 0},
        # As many key/value heads as query heads, a middling batch, larger pages.
        {"name": "decode_mha_b16", "kind": "attention", "heads": "llama2_13b", "dtype": "f16", "page": 64,
         "batch": 16, "new": 1, "context": 1777, "window": 0, "sinks": 0},
        # Three uneven prompts in one call.
        {"name": "prompt_b3_t1000", "kind": "attention", "heads": "llama2_7b", "dtype": "f16", "page": 16, "batch": 3,
         "new": 1000, "context": 0, "window": 0, "sinks": 0},
        # A long prompt at once: the largest product of scores.
        {"name": "prompt_t8192", "kind": "attention", "heads": "mistral7b", "dtype": "f16", "page": 16, "batch": 1,
         "new": 8192, "context": 0, "window": 0, "sinks": 0},
        # A chunk of a long prompt under a sliding window, four first tokens visible.
        {"name": "chunk_window4096", "kind": "attention", "heads": "mistral_nemo", "dtype": "bf16", "page": 16,
         "batch": 1, "new": 2047, "context": 16001, "window": 4096, "sinks": 4},
        # A step of beam search: 64 rows, most of them forked, one layer's pages copied.
        {"name": "fork_r64", "kind": "fork", "heads": "mistral7b", "page": 16, "rows": 64, "context": 2011,
         "layers": 4},
        # A pool in which every second page went free, moved together.
        {"name": "compact_p16384", "kind": "compact", "heads": "mistral7b", "page": 16, "rows": 64, "pages": 16384,
         "layers": 1},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


MOST_FLOPS = 4 * 32 * 128 * 8192 * 8193 // 2   # of the largest listed attention
MOST_TOKENS = 64 * 4096                        # of context that a case keeps, times heads and head dim
MOST_KV = MOST_TOKENS * 8 * 128


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "fork", "compact"])
    heads = rng.choice(sorted(HEADS))
    _, hkv, D = HEADS[heads]
    page = rng.choice([16, 16, 32, 64])
    if kind == "append":
        while True:
            batch, context = _log(rng, 1, 128), _log(rng, 1, 8192)
            new = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
            if batch * (context + new) * hkv * D <= MOST_KV and batch * new * hkv * D <= 3 * 4096 * 8 * 128:
                return {"kind": kind, "heads": heads, "dtype": rng.choice(sorted(DTYPES)), "page": page,
                        "batch": batch, "new": new, "context": context}
    if kind == "attention":
        while True:
            new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 8192)])
            batch = _log(rng, 1, 128) if new <= 16 else _log(rng, 1, 8)
            context = rng.choice([0, _log(rng, 1, 131070), _log(rng, 1, 8192)])
            window = rng.choice([0, 0, _log(rng, 64, 8192)])
            case = {"kind": kind, "heads": heads, "dtype": rng.choice(sorted(DTYPES)), "page": page, "batch": batch,
                    "new": new, "context": context, "window": window,
                    "sinks": rng.choice([0, 4, 70]) if window else 0}
            if batch * (context + new) * hkv * D <= MOST_KV and work(case)["flops"] <= MOST_FLOPS:
                return case
    if kind == "fork":
        while True:
            case = {"kind": kind, "heads": heads, "page": page, "rows": _log(rng, 2, 256),
                    "context": _log(rng, 1, 4096), "layers": rng.choice([1, 4, 8])}
            if 2 * case["rows"] * case["context"] * hkv * D * case["layers"] <= 8 * MOST_KV:
                return case
    pages = _log(rng, 64, 16384)
    while pages * page * hkv * D > 16384 * 16 * 8 * 128:
        pages //= 2
    return {"kind": kind, "heads": heads, "page": page, "rows": _log(rng, 1, 64), "pages": pages, "layers": 1}


def _spread(most, batch):
    """The uneven lengths of a batch: the first the longest, the others down to a quarter of it."""
    return [most if b == 0 else max(min(most, 1), int(most * (0.25 + 0.75 * ((0.618034 * b) % 1.0))))
            for b in range(batch)]


def _lens(case):
    new = _spread(case["new"], case["batch"])
    return new, _spread(case["context"], case["batch"])


# ---------------------------------------------------------------- inputs, from the seed alone

def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _starts(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def _table(g, lens, page):
    """A page table of shuffled pages, rows of different sequences disjoint, and the number of pages (the last is
    nobody's)."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total - 1, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def _rows(g, n, heads, D, dtype, spread):
    """Keys or values of n tokens: heavy channels among ordinary ones, as caches have them."""
    x = torch.randn((n, heads, D), generator=g, device=DEVICE, dtype=torch.float32)
    gain = 1 + spread * (torch.rand((heads, D), generator=g, device=DEVICE) < 0.03)
    return (x * gain).to(dtype)


def _inputs(case, seed):
    g = _gen(seed)
    kind, page = case["kind"], case["page"]
    hq, hkv, D = HEADS[case["heads"]]
    d = {}
    if kind in ("append", "attention"):
        dt = DTYPES[case["dtype"]]
        new, ctx = _lens(case)
        d["new"], d["ctx"] = new, ctx
        d["table"], d["pages"] = _table(g, [n + c for n, c in zip(new, ctx)], page)
        # An append's cache holds the context, an attention's the new tokens too.
        held = ctx if kind == "append" else [n + c for n, c in zip(new, ctx)]
        d["held"] = held
        d["hk"] = _rows(g, sum(held), hkv, D, dt, 3.0)
        d["hv"] = _rows(g, sum(held), hkv, D, dt, 0.0)
        if kind == "append":
            d["k"], d["v"] = _rows(g, sum(new), hkv, D, dt, 3.0), _rows(g, sum(new), hkv, D, dt, 0.0)
        else:
            d["q"] = torch.randn((sum(new), hq, D), generator=g, device=DEVICE).mul_(1.5).to(dt)
        return d
    bytes_ = hkv * page * D
    if kind == "fork":
        lens = _spread(case["context"], case["rows"])
        need = [-(-n // page) for n in lens]
        d["table"], used = _table(g, lens, page)
        spare = max(need) - d["table"].shape[1] + 1  # a forked row may be longer by a page
        d["table"] = torch.nn.functional.pad(d["table"], (0, spare), value=-1).contiguous()
        d["pages"] = used + 2 * case["rows"]
        group = torch.arange(case["rows"], device=DEVICE) // 4 * 4
        pick = torch.randint(0, 4, (case["rows"],), generator=g, device=DEVICE)
        parents = torch.minimum(group + pick, torch.tensor(case["rows"] - 1, device=DEVICE))
        d["parents"] = parents.to(torch.int32)
        d["lens"] = _i32(lens)
    else:
        P = case["pages"]
        d["pages"] = P
        n = P // 2
        held = torch.randperm(P, generator=g, device=DEVICE)[:n].to(torch.int32)
        width = -(-n // case["rows"]) + 1
        d["table"] = torch.full((case["rows"], width), -1, dtype=torch.int32, device=DEVICE)
        flat = torch.full((case["rows"] * (width - 1),), -1, dtype=torch.int32, device=DEVICE)
        flat[:n] = held
        d["table"][:, :width - 1] = flat.view(case["rows"], width - 1)
    refs = torch.zeros(d["pages"], dtype=torch.int32, device=DEVICE)
    t = d["table"][d["table"] >= 0].long()
    d["refs"] = refs.index_put((t,), torch.ones_like(t, dtype=torch.int32), accumulate=True)
    for i in range(case["layers"]):
        for n in "kv":
            d[f"{n}{i}"] = torch.randint(-127, 128, (d["pages"], bytes_), generator=g, device=DEVICE, dtype=torch.int8)
            d[f"{n}s{i}"] = torch.empty((d["pages"], hkv), device=DEVICE).uniform_(0.01, 0.05, generator=g)
    return d


# ---------------------------------------------------------------- the plain forms

def _tokens(starts, counts, table, total, page):
    """Page and slot of every token of a packed batch: counts[b] tokens from position starts[b]."""
    n = torch.tensor(counts, device=DEVICE)
    b = torch.repeat_interleave(torch.arange(len(counts), device=DEVICE), n, output_size=total)
    first = torch.cumsum(n, 0) - n
    pos = torch.tensor(starts, device=DEVICE)[b] + torch.arange(total, device=DEVICE) - first[b]
    return table[b, pos // page].long(), pos % page


def _plain_write(codes, scales, x, starts, counts, table, page):
    """New tokens x [N, heads, D] into codes [pages, heads, page, D], scales [pages, heads]."""
    total = sum(counts)
    if not total:
        return
    pg, slot = _tokens(starts, counts, table, total, page)
    xf = x.float()
    mag = torch.where(torch.isfinite(xf), xf.abs(), torch.zeros_like(xf)).amax(-1)
    fresh = torch.zeros_like(scales)
    fresh.scatter_reduce_(0, pg[:, None].expand_as(mag), mag, "amax", include_self=True)
    fresh = fresh / 127.0
    # Only a sequence's first page can hold tokens already.
    st, n = torch.tensor(starts, device=DEVICE), torch.tensor(counts, device=DEVICE)
    col = torch.minimum(st // page, torch.tensor(table.shape[1] - 1, device=DEVICE))
    p0 = table[torch.arange(len(counts), device=DEVICE), col].long()
    holds = (st % page > 0) & (n > 0)
    p0 = torch.where(holds, p0, torch.full_like(p0, scales.shape[0] - 1))  # the last page belongs to nobody
    old = torch.where(holds[:, None], scales[p0], torch.zeros_like(scales[p0]))
    s0 = torch.maximum(old, torch.where(holds[:, None], fresh[p0], torch.zeros_like(old)))
    r = torch.where(s0 > old, old / torch.where(s0 > 0, s0, torch.ones_like(s0)), torch.ones_like(s0))
    q = torch.round(codes[p0].float() * r[:, :, None, None])
    codes[p0] = q.to(torch.int8)
    scales[pg] = fresh[pg]
    scales[p0] = torch.where(holds[:, None], s0, scales[p0])
    s = scales[pg][:, :, None]
    c = torch.round(xf / s).clamp_(-127, 127).nan_to_num_(nan=127.0)
    codes[pg, :, slot] = torch.where(s > 0, c, torch.zeros_like(c)).to(torch.int8)


def _plain_read(codes, scales, starts, counts, table, page, dtype):
    pg, slot = _tokens(starts, counts, table, sum(counts), page)
    return (codes[pg, :, slot].float() * scales[pg][:, :, None]).to(dtype)


def _plain_attention(s):
    """Softmax over each sequence's visible tokens, a block of queries at a time."""
    case, page = s["case"], s["case"]["page"]
    hq, hkv, D = HEADS[case["heads"]]
    G, dt = hq // hkv, DTYPES[case["dtype"]]
    out = torch.empty_like(s["q"])
    at = 0
    for b, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        L = n + c
        pages = s["table"][b, :-(-L // page)].long()
        k, v = ((s[x][pages].float() * s[x + "s"][pages][:, :, None, None]).transpose(0, 1).reshape(hkv, -1, D)[:, :L]
                for x in ("kc", "vc"))
        kt = k.transpose(1, 2).contiguous()
        step = max(1, (1 << 28) // (L * hq))
        for i0 in range(0, n, step):
            m = min(step, n - i0)
            q = s["q"][at + i0:at + i0 + m].float().view(m, hkv, G, D).permute(1, 2, 0, 3).reshape(hkv, G * m, D)
            z = torch.matmul(q, kt).mul_(1.0 / math.sqrt(D)).view(hkv, G, m, L)
            p = torch.arange(c + i0, c + i0 + m, device=DEVICE)[:, None]
            j = torch.arange(L, device=DEVICE)[None, :]
            seen = j <= p
            if case["window"]:
                seen &= (j > p - case["window"]) | (j < case["sinks"])
            z.masked_fill_(~seen, float("-inf"))
            z.sub_(z.amax(-1, keepdim=True)).exp_()
            z.div_(z.sum(-1, keepdim=True))
            o = torch.matmul(z.view(hkv, G * m, L), v.contiguous()).view(hkv, G, m, D)
            out[at + i0:at + i0 + m] = o.permute(2, 0, 1, 3).reshape(m, hq, D).to(dt)
        at += n
    return {"out": out}


def _plain_copy(s, src, dst, spare):
    """Pages src -> dst where dst >= 0; elsewhere page spare onto itself (it is no destination)."""
    go = dst >= 0
    a, b = torch.where(go, src.long(), spare), torch.where(go, dst.long(), spare)
    for i in range(s["case"]["layers"]):
        for n in ("k", "v", "ks", "vs"):
            t = s[f"{n}{i}"]
            t[b] = t[a]


def _plain_fork(s):
    page, R = s["case"]["page"], s["case"]["rows"]
    P, W = s["pages"], s["table"].shape[1]
    parents = s["parents"].long()
    lens = s["lens"].long()
    cols = torch.arange(W, device=DEVICE)[None, :]
    new_lens = lens[parents]
    held = -(-lens // page)
    table = torch.where(cols < held[parents][:, None], s["table"][parents], torch.full_like(s["table"], -1))
    refs = torch.zeros(P + 1, dtype=torch.int32, device=DEVICE)
    t = torch.where(table >= 0, table, torch.full_like(table, P)).long().flatten()
    refs.index_put_((t,), torch.ones_like(t, dtype=torch.int32), accumulate=True)
    refs = refs[:P]
    # Grow by a token: a shared last page is copied, a full one followed by a fresh one.
    rows = torch.arange(R, device=DEVICE)
    at = new_lens // page
    last = table[rows, at].long()
    partly = new_lens % page > 0
    shared = partly & (refs[torch.where(partly, last, torch.zeros_like(last))] > 1)
    need = (shared | ~partly).int()
    rank = torch.cumsum(need, 0) - need
    order = torch.cumsum((refs == 0).int(), 0) - 1
    free = torch.full((P + 1,), -1, dtype=torch.int64, device=DEVICE)
    free.scatter_(0, torch.where(refs == 0, order.long(), torch.full_like(order, P).long()), torch.arange(P, device=DEVICE))
    fresh = free[rank.long()]
    src = torch.where(shared, last, torch.full_like(last, -1)).int()
    dst = torch.where(shared, fresh, torch.full_like(fresh, -1)).int()
    table[rows, at] = torch.where(need > 0, fresh, last).int()
    refs = torch.cat((refs, refs.new_zeros(1)))
    refs.index_put_((torch.where(shared, last, torch.full_like(last, P)),), -torch.ones_like(src), accumulate=True)
    refs.index_put_((torch.where(need > 0, fresh, torch.full_like(fresh, P)),), torch.ones_like(src), accumulate=True)
    _plain_copy(s, src, dst, table[rows, at].long())
    return {"table": table, "refs": refs[:P], "lens": new_lens.int(), "src": src, "dst": dst,
            "missing": torch.zeros(1, dtype=torch.int32, device=DEVICE), **_layers(s)}


def _plain_compact(s):
    P = s["pages"]
    cap = P // 2 + 1
    refs = s["refs"]
    used = refs > 0
    n = used.sum()
    i = torch.arange(P, device=DEVICE)
    a, b = used & (i >= n), ~used & (i < n)
    src, dst = (torch.full((cap + 1,), -1, dtype=torch.int64, device=DEVICE).scatter_(
        0, torch.where(m, torch.cumsum(m, 0) - 1, torch.full_like(i, cap)), i)[:cap] for m in (a, b))
    to = i.scatter(0, torch.where(src >= 0, src, i[:cap]), torch.where(src >= 0, dst, i[:cap]))
    t = s["table"].long()
    table = torch.where(t >= 0, to[t.clamp(min=0)], t).int()
    ext = torch.cat((torch.where(i < n, refs, torch.zeros_like(refs)), refs.new_zeros(1)))
    ext.scatter_(0, torch.where(src >= 0, dst, torch.full_like(dst, P)),
                 torch.where(src >= 0, refs[src.clamp(min=0)], torch.zeros_like(refs[:cap])))
    out = ext[:P]
    _plain_copy(s, src, dst, torch.where(src[0] >= 0, src[0], torch.zeros_like(src[0])))
    return {"table": table, "refs": out, "src": src.int(), "dst": dst.int(), "moves": a.sum().int().reshape(1),
            **_layers(s)}


def _layers(s):
    return {f"{n}{i}": s[f"{n}{i}"] for i in range(s["case"]["layers"]) for n in ("k", "v", "ks", "vs")}


# ---------------------------------------------------------------- what a host program has and calls

def _p(t):
    return C.c_void_p(t.data_ptr())


def _ok(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed")


def _library():
    from neurogrid_amd import _lib
    return _lib, _lib.load()


def _cache(kc, vc, ks, vs, pages, hkv, D, page):
    m, _ = _library()
    return m.KVInt8Cache(_p(kc), _p(vc), _p(ks), _p(vs), pages, hkv, D, page)


def _name(case, what):
    return ("ng_bf16_" if case["dtype"] == "bf16" else "ng_") + "kv_int8_" + what


def _own_append(s, k, v, cu, starts, total, most):
    _, L = _library()
    _ok(getattr(L, _name(s["case"], "append"))(
        C.byref(s["cache"]), _p(k), _p(v), _p(cu), _p(starts), _p(s["table"]), s["case"]["batch"],
        s["table"].shape[1], total, most, None), "append")


def prepare(case, seed):
    d = _inputs(case, seed)
    kind, page = case["kind"], case["page"]
    hq, hkv, D = HEADS[case["heads"]]
    s = dict(d, case=case)
    if kind in ("append", "attention"):
        pages, batch = d["pages"], case["batch"]
        new, ctx, held = d["new"], d["ctx"], d["held"]
        shape = (pages, hkv, page * D) if own else (pages, hkv, page, D)
        for n in "kv":
            s[n + "c"] = torch.zeros(shape, dtype=torch.int8, device=DEVICE)
            s[n + "cs"] = torch.zeros((pages, hkv), device=DEVICE)
        # Where a read-back begins: at the first page that the new tokens touch.
        s["from"] = [c // page * page for c in ctx]
        s["count"] = [c + n - f for c, n, f in zip(ctx, new, s["from"])]
        hk, hv = s.pop("hk"), s.pop("hv")
        if own:
            _, L = _library()
            L.ng_set_stream(C.c_void_p(torch.cuda.current_stream().cuda_stream))
            s["cache"] = _cache(s["kc"], s["vc"], s["kcs"], s["vcs"], pages, hkv, D, page)
            if sum(held):
                _own_append(s, hk, hv, _i32(_starts(held)), _i32([0] * batch), sum(held), max(held))
            s["cu"], s["dctx"] = _i32(_starts(new)), _i32(ctx)
            if kind == "append":
                s["dfrom"], s["cufrom"] = _i32(s["from"]), _i32(_starts(s["count"]))
                s["rk"], s["rv"] = (torch.empty((sum(s["count"]), hkv, D), dtype=hk.dtype, device=DEVICE)
                                    for _ in "kv")
            else:
                s["lens"] = _i32([n + c for n, c in zip(new, ctx)])
                s["out"] = torch.empty_like(s["q"])
                s["most"] = (max(new), max(n + c for n, c in zip(new, ctx)))
                bytes_ = L.ng_kv_int8_attention_workspace(C.byref(s["cache"]), hq, batch, *s["most"])
                s["workspace"] = torch.empty(max(1, bytes_), dtype=torch.int8, device=DEVICE)
        else:
            zero = [0] * batch
            _plain_write(s["kc"], s["kcs"], hk, zero, held, s["table"], page)
            _plain_write(s["vc"], s["vcs"], hv, zero, held, s["table"], page)
        return s
    if own:
        m, L = _library()
        n = case["layers"]
        s["caches"] = (m.KVInt8Cache * n)(*[
            _cache(s[f"k{i}"], s[f"v{i}"], s[f"ks{i}"], s[f"vs{i}"], d["pages"], hkv, D, page) for i in range(n)])
        s["table2"], s["refs2"] = torch.empty_like(d["table"]), torch.empty_like(d["refs"])
        s["one"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        count = case["rows"] if kind == "fork" else d["pages"] // 2 + 1
        s["src"], s["dst"] = (torch.empty(count, dtype=torch.int32, device=DEVICE) for _ in "sd")
        if kind == "fork":
            s["lens2"] = torch.empty_like(d["lens"])
    return s


def _own_run(s):
    m, L = _library()
    case = s["case"]
    kind, page = case["kind"], case["page"]
    hq, hkv, D = HEADS[case["heads"]]
    L.ng_set_stream(C.c_void_p(torch.cuda.current_stream().cuda_stream))
    if kind == "append":
        _own_append(s, s["k"], s["v"], s["cu"], s["dctx"], sum(s["new"]), max(s["new"]))
        _ok(getattr(L, _name(case, "read"))(
            C.byref(s["cache"]), _p(s["rk"]), _p(s["rv"]), _p(s["cufrom"]), _p(s["dfrom"]), _p(s["table"]),
            case["batch"], s["table"].shape[1], sum(s["count"]), max(s["count"])), "read")
        return {"k": s["rk"], "v": s["rv"]}
    if kind == "attention":
        _ok(getattr(L, _name(case, "attention"))(
            _p(s["out"]), _p(s["q"]), C.byref(s["cache"]), _p(s["cu"]), _p(s["lens"]), _p(s["table"]), case["batch"],
            s["table"].shape[1], sum(s["new"]), *s["most"], hq, C.c_float(1.0 / math.sqrt(D)), case["window"],
            case["sinks"], _p(s["workspace"]), s["workspace"].numel()), "attention")
        return {"out": s["out"]}
    rows, width = s["table"].shape
    s["refs2"].copy_(s["refs"])  # the pool as it was, so that a pass can be made again
    pool = m.KVPages(_p(s["table"]), _p(s["refs2"]), rows, width, s["pages"], page)
    if kind == "fork":
        _ok(L.ng_kv_pages_fork(C.byref(pool), _p(s["table2"]), _p(s["parents"]), _p(s["lens"]), _p(s["lens2"])), "fork")
        grown = s["lens2"] + 1
        pool = m.KVPages(_p(s["table2"]), _p(s["refs2"]), rows, width, s["pages"], page)
        _ok(L.ng_kv_pages_grow(C.byref(pool), _p(s["lens2"]), _p(grown), _p(s["src"]), _p(s["dst"]), _p(s["one"])),
            "grow")
        _ok(L.ng_kv_int8_copy_pages(s["caches"], case["layers"], _p(s["src"]), _p(s["dst"]), s["src"].numel()), "copy")
        return {"table": s["table2"], "refs": s["refs2"], "lens": s["lens2"], "src": s["src"], "dst": s["dst"],
                "missing": s["one"], **_layers(s)}
    s["table2"].copy_(s["table"])
    pool = m.KVPages(_p(s["table2"]), _p(s["refs2"]), rows, width, s["pages"], page)
    _ok(L.ng_kv_pages_compact(C.byref(pool), _p(s["src"]), _p(s["dst"]), s["src"].numel(), _p(s["one"])), "compact")
    _ok(L.ng_kv_int8_copy_pages(s["caches"], case["layers"], _p(s["src"]), _p(s["dst"]), s["src"].numel()), "copy")
    return {"table": s["table2"], "refs": s["refs2"], "src": s["src"], "dst": s["dst"], "moves": s["one"],
            **_layers(s)}


def run(state):
    s = state
    if own:
        return _own_run(s)
    case = s["case"]
    kind, page = case["kind"], case["page"]
    if kind == "append":
        dt = DTYPES[case["dtype"]]
        for n in "kv":
            _plain_write(s[n + "c"], s[n + "cs"], s[n], s["ctx"], s["new"], s["table"], page)
        return {n: _plain_read(s[n + "c"], s[n + "cs"], s["from"], s["count"], s["table"], page, dt) for n in "kv"}
    if kind == "attention":
        return _plain_attention(s)
    if kind == "fork":
        return _plain_fork(s)
    return _plain_compact(s)


# ---------------------------------------------------------------- what a pass cannot do without

def _visible(case):
    """Pairs of a query and a token that it sees, and tokens that some query of their sequence sees."""
    pairs = tokens = 0
    w, sinks = case["window"], case["sinks"]
    for n, c in zip(*_lens(case)):
        if not w:
            pairs += n * c + n * (n + 1) // 2
            tokens += n + c
            continue
        first = max(0, c - w + 1)  # the oldest token in the first query's window
        tokens += n + c - first + min(sinks, first)
        for p in range(c, c + n):
            start = max(0, p - w + 1)
            pairs += p + 1 - start + min(sinks, start)
    return pairs, tokens


def work(case):
    kind, page = case["kind"], case["page"]
    hq, hkv, D = HEADS[case["heads"]]
    row = hkv * D
    if kind == "append":
        new, ctx = _lens(case)
        n, held = sum(new), sum(c % page for c in ctx)
        pages = sum(-(-(c % page + m) // page) for m, c in zip(new, ctx))
        # New rows in, their pages' codes out (read and written where they held tokens), all of them read back.
        return {"bytes": 2 * (2 * n * row + (n + 2 * held) * row + 4 * pages * hkv + 3 * (n + held) * row) + 8 * pages,
                "flops": 2 * 6 * n * row}
    if kind == "attention":
        pairs, tokens = _visible(case)
        n, scales = sum(_lens(case)[0]), -(-tokens // page) * hkv * 4
        return {"bytes": 2 * (tokens * row + scales) + 2 * 2 * n * hq * D, "flops": 4 * pairs * hq * D}
    body = 2 * (page * row + 4 * hkv) * case["layers"]
    if kind == "fork":
        lens = _spread(case["context"], case["rows"])
        table = sum(-(-n // page) for n in lens)
        pages = table + 2 * case["rows"] + 3
        # A parent in four is taken more than once and ends inside a page: about half the rows copy one.
        moved = case["rows"] // 2
        return {"bytes": 8 * table + 8 * pages + 2 * moved * body, "flops": 0}
    P = case["pages"]
    return {"bytes": 8 * P + 8 * (P // 2) + 4 * P + 2 * (P // 4) * body, "flops": 0}


# ---------------------------------------------------------------- the same in 64 bits

def _exact_values(parts, page):
    """What a sequence's block-quantised rows stand for, its tokens written part by part. [tokens, heads, D]"""
    codes, scale, pos = None, None, 0
    n = sum(len(p) for p in parts)
    heads, D = parts[0].shape[1:]
    width = -(-n // page)
    codes = torch.zeros((width, page, heads, D), dtype=torch.float64, device=DEVICE)
    scale = torch.zeros((width, heads), dtype=torch.float64, device=DEVICE)
    for x in parts:
        if not len(x):
            continue
        a, b = pos // page, -(-(pos + len(x)) // page)
        flat = torch.zeros(((b - a) * page, heads, D), dtype=torch.float64, device=DEVICE)
        flat[pos - a * page:pos - a * page + len(x)] = x.double()
        blocks = flat.view(b - a, page, heads, D)
        s = torch.maximum(scale[a:b], blocks.abs().amax((1, 3)) / 127)
        safe = torch.where(s > 0, s, torch.ones_like(s))
        codes[a:b] = (codes[a:b] * (scale[a:b] / safe)[:, None, :, None]).round()
        codes[a:b] += (blocks / safe[:, None, :, None]).round()
        scale[a:b] = s
        pos += len(x)
    return (codes * scale[:, None, :, None]).reshape(-1, heads, D)[:n]


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None
    d = _inputs(case, seed)
    page = case["page"]
    hq, hkv, D = HEADS[case["heads"]]
    if case["kind"] == "append":
        got = {}
        for n in "kv":
            rows, a, h = [], 0, 0
            for new, ctx in zip(d["new"], d["ctx"]):
                first = ctx // page * page
                # Pages before the first touched one are not read: they hold only context.
                v = _exact_values([d["h" + n][h + first:h + ctx], d[n][a:a + new]], page)
                rows.append(v)
                a, h = a + new, h + ctx
            got[n] = torch.cat(rows)
        return got
    out = torch.empty((sum(d["new"]), hq, D), dtype=torch.float64, device=DEVICE)
    at = h = 0
    for new, ctx in zip(d["new"], d["ctx"]):
        L = new + ctx
        k, v = (_exact_values([d[n][h:h + L]], page) for n in ("hk", "hv"))
        h += L
        for g in range(hkv):
            kg, vg = k[:, g].contiguous(), v[:, g].contiguous()
            heads = slice(g * (hq // hkv), (g + 1) * (hq // hkv))
            step = max(1, (1 << 26) // L)
            for i in range(0, new, step):
                q = d["q"][at + i:min(at + i + step, at + new), heads].double()
                m = q.shape[0]
                pos = ctx + i + torch.arange(m, device=DEVICE)
                tok = torch.arange(L, device=DEVICE)
                hide = tok[None] > pos[:, None]
                if case["window"]:
                    hide |= (tok[None] <= pos[:, None] - case["window"]) & (tok[None] >= case["sinks"])
                for e in range(q.shape[1]):
                    z = (q[:, e] @ kg.t()) / math.sqrt(D)
                    z[hide] = -math.inf
                    out[at + i:at + i + m, heads.start + e] = torch.softmax(z, -1) @ vg
        at += new
    return {"out": out}
