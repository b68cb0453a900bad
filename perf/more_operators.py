"""Operators of a server that keeps its KV caches in pages, as cases that can be timed and compared: rows rotated and
appended to the pages, attention over them, attention of a batch that shares a long prefix, and attention over the
pages that a bound of their scores selects.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what the program holds before
the call, run() is one pass (the plain form in elementary torch operations, or, with `own`, this library's
calls) and exact() the same outputs in 64 bits, written apart.

The kinds of case:
  store    new rows of N sequences: queries and keys rotated by their positions, keys and values into the pages, and,
           where asked, the smallest and largest key of each channel of the pages written to
  attend   attention of rows of N sequences, each over its own pages
  prefix   the same where the first `prefix` positions of all sequences are the same pages
  sparse   each row and KV head over its first and last pages and the `top` others of largest score: the largest,
           over the group's heads, of sum_d max(q_d lo_d, q_d hi_d) with the page's bounds lo and hi

A pool holds pages of `page` positions: per page and KV head, keys [unit of 16 positions][t][HD / 8][h][r][8] for position
8 h + 4 t + r of the unit, and values [position / 8][HD][position % 8], all in fp16. A table gives each sequence's pages.
"""
import ctypes
import math

import numpy as np
import torch

own = False

# heads, KV heads, head dim (the 8B and 70B Llama layers of the benchmark, and the shape of a 1B model)
DIMS = {"1b": (32, 8, 64), "8b": (32, 8, 128), "70b": (64, 8, 128)}


def listed():
    return [
        # a decode step's row of one chat: the smallest call
        {"name": "store_8b_one_row", "kind": "store", "dims": "8b", "page": 64, "N": 1, "top": 701, "rows": 1,
         "mixed": False, "bounds": False, "neox": False, "freqs": True},
        # a server's decode step with the pages' bounds kept for sparse attention
        {"name": "store_70b_batch_64", "kind": "store", "dims": "70b", "page": 64, "N": 64, "top": 90001, "rows": 1,
         "mixed": False, "bounds": True, "neox": False, "freqs": True},
        # prompts of several sequences beside decode steps, odd lengths, small pages
        {"name": "store_8b_prompts", "kind": "store", "dims": "8b", "page": 16, "N": 5, "top": 2600, "rows": 1801,
         "mixed": True, "bounds": True, "neox": True, "freqs": False},
        # a small server's step of a 1B model, smallest pages
        {"name": "attend_1b_batch_6", "kind": "attend", "dims": "1b", "page": 16, "N": 6, "top": 900, "rows": 1,
         "mixed": False},
        # a large server's step: conversations of all lengths
        {"name": "attend_70b_batch_48", "kind": "attend", "dims": "70b", "page": 64, "N": 48, "top": 9001, "rows": 1,
         "mixed": False},
        # prompts, a guess-ahead pass and decode steps in one call
        {"name": "attend_8b_prompts", "kind": "attend", "dims": "8b", "page": 32, "N": 5, "top": 4300, "rows": 2001,
         "mixed": True},
        # a few agents on one tool description
        {"name": "prefix_8b_7_on_2048", "kind": "prefix", "dims": "8b", "page": 64, "N": 7, "prefix": 2048, "top": 333,
         "rows": 1, "mixed": False},
        # a service whose users share a long system prompt
        {"name": "prefix_70b_64_on_8192", "kind": "prefix", "dims": "70b", "page": 64, "N": 64, "prefix": 8192, "top": 700,
         "rows": 1, "mixed": False},
        # questions about one book, a guess-ahead pass of four rows each
        {"name": "prefix_8b_20_on_60000", "kind": "prefix", "dims": "8b", "page": 32, "N": 20, "prefix": 60000, "top": 250,
         "rows": 4, "mixed": False},
        # a guess-ahead pass in a chat of middle length, small pages
        {"name": "sparse_1b_t5_at_6000", "kind": "sparse", "dims": "1b", "page": 16, "N": 1, "top": 6005, "rows": 5,
         "mixed": False, "first": 1, "recent": 4, "best": 59},
        # a decode step over a book
        {"name": "sparse_8b_t1_at_131000", "kind": "sparse", "dims": "8b", "page": 64, "N": 1, "top": 131001, "rows": 1,
         "mixed": False, "first": 1, "recent": 2, "best": 61},
        # a server's step over long documents
        {"name": "sparse_70b_batch_16", "kind": "sparse", "dims": "70b", "page": 64, "N": 16, "top": 32001, "rows": 1,
         "mixed": False, "first": 1, "recent": 2, "best": 29},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "prefix", "prefix", "sparse", "sparse"])
    dims = rng.choice(["1b", "8b", "70b"])
    c = {"kind": kind, "dims": dims, "page": rng.choice([16, 32, 64, 64, 128, 256]), "rows": 1, "mixed": False}
    if kind == "store":
        c.update(N=_log(rng, 1, 100), top=_log(rng, 16, 100000), bounds=rng.random() < 0.5, neox=rng.random() < 0.5,
                 freqs=rng.random() < 0.5)
        if c["N"] <= 8 and rng.random() < 0.6:
            c.update(rows=min(_log(rng, 2, 4000 // c["N"]), c["top"]), mixed=rng.random() < 0.5)
    elif kind == "attend":
        c.update(N=_log(rng, 1, 48))
        c.update(top=_log(rng, 20, 60000 if c["N"] == 1 else 9000 if c["N"] < 25 else 5000))
        if c["N"] <= 6 and rng.random() < 0.6:
            c.update(top=min(c["top"], 4500), mixed=rng.random() < 0.5)
            c.update(rows=min(_log(rng, 2, (1000 if dims == "70b" else 2000) // c["N"]), c["top"]))
    elif kind == "prefix":
        c.update(N=_log(rng, 2, 64), top=_log(rng, 1, 600), rows=rng.choice([1, 1, 1, rng.randint(2, 6)]))
        c.update(prefix=c["page"] * max(1, _log(rng, 200, 50000 if c["N"] < 20 else 9000) // c["page"]))
        c.update(top=max(c["top"], c["rows"]))
    else:
        c.update(N=_log(rng, 1, 16), first=rng.randint(0, 2), recent=rng.randint(1, 4), best=_log(rng, 1, 64))
        c.update(top=_log(rng, 100, 100000 if c["N"] <= 2 else 30000))
        if c["N"] == 1 and rng.random() < 0.5:
            c.update(rows=rng.randint(2, 40))
    return c


def _rows_of(case):
    """Sequence, first position and number of rows of each entry: lengths from short to full, sequences in another order."""
    N, top, rows = case["N"], case["top"], case["rows"]
    seq = [(5 * i + 3) % N if N % 5 else N - 1 - i for i in range(N)]
    pos, num = [], []
    for i in range(N):
        n = top - (i * top) // N * (i % 4) // 3
        t = (rows, 1, max(1, rows // 40), max(1, rows // 3))[i % 4] if case["mixed"] else rows
        t = min(t, n)
        pos.append(n - t + case.get("prefix", 0))
        num.append(t)
    return seq, pos, num


# ------------------------------------------------------------------------------------- inputs


class State:
    pass


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000 + salt)
    return g


def _normal(shape, seed, salt, scale=1.0):
    return torch.randn(shape, device="cuda", generator=_gen(seed, salt)) * scale


def _channels(KH, HD, seed, salt):
    """Keys as trained models have them: a few channels of every head far larger than the rest."""
    big = torch.rand((KH, HD), device="cuda", generator=_gen(seed, salt)) < 0.03
    return torch.where(big, 5.0, 1.0)


def _key_rows(K, HD):
    """Keys [..., KH, page, HD] of a pool [..., KH, page * HD], and _key_pool the other way."""
    lead = K.shape[:-1]
    x = K.reshape(*lead, -1, 2, HD // 8, 2, 4, 8).movedim((-3, -5, -2, -4, -1), (-5, -4, -3, -2, -1))
    return x.reshape(*lead, -1, HD)


def _key_pool(k):
    lead, HD = k.shape[:-2], k.shape[-1]
    x = k.reshape(*lead, -1, 2, 2, 4, HD // 8, 8).movedim((-4, -2, -5, -3, -1), (-5, -4, -3, -2, -1))
    return x.reshape(*lead, -1)


def _val_rows(V, HD):
    x = V.reshape(*V.shape[:-1], -1, HD, 8).transpose(-1, -2)
    return x.reshape(*V.shape[:-1], -1, HD)


def _val_pool(v):
    HD = v.shape[-1]
    x = v.reshape(*v.shape[:-2], -1, 8, HD).transpose(-1, -2)
    return x.reshape(*v.shape[:-2], -1)


def prepare(case, seed):
    s = State()
    s.case, kind, page = case, case["kind"], case["page"]
    H, KH, HD = DIMS[case["dims"]]
    s.seq, s.pos, s.num = _rows_of(case)
    prefix = case.get("prefix", 0) // page
    need = [(p + t + page - 1) // page for p, t in zip(s.pos, s.num)]
    # a free pool's pages in no order, the prefix' pages in every table
    # (a store's sequences: of theirs only those it writes to)
    lo = [p // page if kind == "store" else prefix for p in s.pos]
    total = prefix + sum(n - a for n, a in zip(need, lo))
    s.pages = total + 5
    order = torch.randperm(s.pages, generator=torch.Generator().manual_seed(int(seed) * 7 + 1)).tolist()
    s.width = max(need) + 3
    table = [[-1] * s.width for _ in range(case["N"])]
    at = prefix
    for i, n in enumerate(need):
        table[s.seq[i]][:prefix] = order[:prefix]
        table[s.seq[i]][lo[i]:n] = order[at:at + n - lo[i]]
        at += n - lo[i]
    s.table = torch.tensor(table, dtype=torch.int32, device="cuda")
    s.K = torch.empty((s.pages, KH, page * HD), dtype=torch.float16, device="cuda")
    s.V = torch.empty_like(s.K)
    scale, g, h = _channels(KH, HD, seed, 5), _gen(seed, 6), _gen(seed, 7)
    # a key's neighbours are like it, as in a text: each page has its own direction
    for i in range(0, s.pages, 512):
        m = min(512, s.pages - i)
        k = torch.randn((m, KH, page, HD), device="cuda", generator=g)
        k += torch.randn((m, KH, 1, HD), device="cuda", generator=g)
        s.K[i:i + m] = _key_pool((k * scale[:, None]).to(torch.float16))
        s.V[i:i + m] = torch.randn((m, KH, page * HD), device="cuda", generator=h).to(torch.float16)
    R = sum(s.num)
    s.q = _normal((R, H, HD), seed, 1, 1.5)
    if kind == "store":
        s.k = _normal((R, KH, HD), seed, 2) * scale
        s.v = _normal((R, KH, HD), seed, 3)
        s.half = HD // 2
        f = 1.0 + 7.0 * torch.rand(s.half, device="cuda", generator=_gen(seed, 4))
        s.freqs = torch.where(torch.arange(s.half, device="cuda") < s.half // 2, 1.0, f) if case["freqs"] else None
        s.bounds = torch.zeros((s.pages, KH, 2, HD), dtype=torch.float16, device="cuda") if case["bounds"] else None
        s.qr = torch.empty_like(s.q)
    if kind == "sparse":
        s.bounds = torch.zeros((s.pages, KH, 2, HD), dtype=torch.float16, device="cuda")
        for i, n in enumerate(need):
            ids = s.table[s.seq[i], :n].long()
            k = _key_rows(s.K[ids], HD)
            there = torch.arange(n * page, device="cuda").reshape(n, 1, page, 1) < s.pos[i] + s.num[i]
            s.bounds[ids, :, 0] = torch.where(there, k, math.inf).amin(2)
            s.bounds[ids, :, 1] = torch.where(there, k, -math.inf).amax(2)
    return s


# ------------------------------------------------------------------------------------- plain forms

BASE = 500000.0


def _positions(s):
    return torch.cat([p + torch.arange(t, device="cuda") for p, t in zip(s.pos, s.num)])


def _pairs(HD, neox):
    i = torch.arange(HD // 2, device="cuda")
    return (i, i + HD // 2) if neox else (2 * i, 2 * i + 1)


def _turn(x, cos, sin, a, b):
    y = torch.empty_like(x)
    x0, x1 = x[..., a], x[..., b]
    y[..., a] = x0 * cos - x1 * sin
    y[..., b] = x0 * sin + x1 * cos
    return y


def _plain_store(s):
    case, page = s.case, s.case["page"]
    HD = DIMS[case["dims"]][2]
    pos = _positions(s)
    ang = pos[:, None].double() * BASE ** (-2.0 * torch.arange(HD // 2, device="cuda").double() / HD)
    if s.freqs is not None:
        ang = ang / s.freqs.double()
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    a, b = _pairs(HD, case["neox"])
    s.qr.copy_(_turn(s.q, cos, sin, a, b))
    k, v = _turn(s.k, cos, sin, a, b).to(torch.float16), s.v.to(torch.float16)
    # the pages written to as rows, the new rows in their places, and back
    at = 0
    for q, p, t in zip(s.seq, s.pos, s.num):
        lo, hi = p // page, (p + t - 1) // page + 1
        ids = s.table[q, lo:hi].long()
        K, V = _key_rows(s.K[ids], HD).transpose(1, 2), _val_rows(s.V[ids], HD).transpose(1, 2)
        shape = K.shape
        K, V = K.reshape(-1, *shape[2:]), V.reshape(-1, *shape[2:])
        K[p - lo * page:p - lo * page + t] = k[at:at + t]
        V[p - lo * page:p - lo * page + t] = v[at:at + t]
        K, V = K.reshape(shape).transpose(1, 2), V.reshape(shape).transpose(1, 2)
        s.K[ids], s.V[ids] = _key_pool(K), _val_pool(V)
        if s.bounds is not None:
            there = torch.arange(lo * page, hi * page, device="cuda").reshape(-1, 1, page, 1) < p + t
            s.bounds[ids] = torch.stack([torch.where(there, K, math.inf).amin(2), torch.where(there, K, -math.inf).amax(2)], 2)
        at += t
    out = {"q": s.qr, "K": s.K, "V": s.V}
    return out if s.bounds is None else dict(out, bounds=s.bounds)


def _attend(q, K, V, see):
    """Rows q [T, H, HD] over K, V [KH, n, HD] in fp32; see [T or T, KH, n]: which positions a row sees."""
    T, H, HD = q.shape
    KH, n = K.shape[0], K.shape[1]
    q = q.reshape(T, KH, -1, HD).movedim(0, 2)                                        # KH, G, T, HD
    S = torch.matmul(q.reshape(KH, -1, HD), K.transpose(-1, -2).contiguous()).reshape(KH, -1, T, n) / math.sqrt(HD)
    see = see if see.dim() == 2 else see.movedim(1, 0)[:, None]
    S = S.masked_fill(~see, -math.inf)
    P = torch.exp(S - S.amax(-1, keepdim=True))
    P = P / P.sum(-1, keepdim=True)
    o = torch.matmul(P.reshape(KH, -1, n), V)
    return o.reshape(KH, -1, T, HD).movedim(2, 0).reshape(T, H, HD)


def _sequence(s, i):
    """Keys and values [KH, n, HD] in fp32 of entry i's sequence."""
    page, HD = s.case["page"], DIMS[s.case["dims"]][2]
    n = s.pos[i] + s.num[i]
    ids = s.table[s.seq[i], :(n + page - 1) // page].long()
    K = _key_rows(s.K[ids], HD).movedim(0, 1).flatten(1, 2)[:, :n]
    V = _val_rows(s.V[ids], HD).movedim(0, 1).flatten(1, 2)[:, :n]
    return K.float(), V.float()


def _plain_blocks(s, i, q):
    """The pages that each row of entry i takes: [T, KH, first + best + recent], in order, -1 after the last."""
    case, page = s.case, s.case["page"]
    KH = DIMS[case["dims"]][1]
    T, n = s.num[i], s.pos[i] + s.num[i]
    nb = (n + page - 1) // page
    b = s.bounds[s.table[s.seq[i], :nb].long()].double()                              # nb, KH, 2, HD
    g = q.reshape(T, KH, -1, q.shape[-1]).movedim(0, 2).double()                      # KH, G, T, HD
    lo, hi = (b[:, :, x].permute(1, 2, 0).contiguous() for x in (0, 1))
    sc = torch.matmul(g.clamp(min=0).flatten(1, 2), hi) + torch.matmul(g.clamp(max=0).flatten(1, 2), lo)
    sc = sc.reshape(KH, -1, T, nb).amax(1).movedim(0, 1)                              # T, KH, nb
    cur = ((s.pos[i] + torch.arange(T, device="cuda")) // page)[:, None, None]
    j = torch.arange(nb, device="cuda")
    kept = ((j < case["first"]) | (j > cur - case["recent"])) & (j <= cur)
    open_ = (j <= cur) & ~kept
    sc = torch.where(open_, sc, -math.inf)
    order = torch.sort(sc, dim=-1, descending=True, stable=True).indices[..., :case["best"]]
    taken = torch.zeros_like(sc, dtype=torch.bool).scatter_(-1, order, True) & open_ | kept
    width = case["first"] + case["best"] + case["recent"]
    out = torch.full((T, KH, width), -1, dtype=torch.int32, device="cuda")
    t, h, x = torch.nonzero(taken, as_tuple=True)
    out[t, h, (torch.cumsum(taken, -1) - 1)[t, h, x]] = x.to(torch.int32)
    return out


def _plain(s):
    case, page = s.case, s.case["page"]
    if case["kind"] == "store":
        return _plain_store(s)
    out, blocks, at = torch.empty_like(s.q), [], 0
    for i, (p, t) in enumerate(zip(s.pos, s.num)):
        K, V = _sequence(s, i)
        q = s.q[at:at + t]
        see = torch.arange(p + t, device="cuda") <= p + torch.arange(t, device="cuda")[:, None]
        if case["kind"] == "sparse":
            b = _plain_blocks(s, i, q)
            blocks.append(b)
            taken = torch.zeros((t, K.shape[0], s.width + 1), dtype=torch.bool, device="cuda")
            taken.scatter_(-1, torch.where(b < 0, s.width, b).long(), True)
            see = see[:, None] & taken[..., torch.arange(p + t, device="cuda") // page]
        out[at:at + t] = _attend(q, K, V, see)
        at += t
    return {"out": out, "blocks": torch.cat(blocks)} if blocks else out


# ------------------------------------------------------------------------------------- the library's calls

_ctx = []


def _p(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def _own(s):
    from windlass_amd._lib import check, load
    from windlass_amd.backend import Context, PageRows, Pages, SparseOpts
    if not _ctx:
        _ctx.append(Context(0))
    case, L, h = s.case, load(), _ctx[0].handle
    if not hasattr(s, "call"):  # the buffers and arguments that a program keeps from step to step
        H, KH, HD = DIMS[case["dims"]]
        kind, scale = case["kind"], ctypes.c_float(1.0 / math.sqrt(HD))
        bounds = getattr(s, "bounds", None)
        s.desc = Pages(d_K=_p(s.K), d_V=_p(s.V), d_bounds=_p(bounds), pages=s.pages, page=case["page"], kv_heads=KH,
                       head_dim=HD, d_table=_p(s.table), sequences=case["N"], table_pages=s.width)
        s.rows = PageRows(s.seq, s.pos, s.num)
        d, r = ctypes.byref(s.desc), ctypes.byref(s.rows)
        if kind == "store":
            s.out = {"q": s.qr, "K": s.K, "V": s.V}
            if bounds is not None:
                s.out["bounds"] = bounds
            s.call = (L.wl_paged_store_dev, (h, d, r, _p(s.q), H, _p(s.k), _p(s.v), HD, int(case["neox"]), BASE, 1.0,
                                             _p(s.freqs), _p(s.qr)))
        elif kind == "sparse":
            s.opts = SparseOpts(case["first"], case["recent"], case["best"])
            width = case["first"] + case["recent"] + case["best"]
            s.out = {"out": torch.empty_like(s.q),
                     "blocks": torch.empty((s.q.shape[0], KH, width), dtype=torch.int32, device="cuda")}
            s.call = (L.wl_paged_sparse_dev, (h, d, r, _p(s.q), H, ctypes.byref(s.opts), scale, _p(s.out["out"]),
                                              _p(s.out["blocks"])))
        else:
            s.out = torch.empty_like(s.q)
            s.call = (L.wl_paged_attention_dev, (h, d, r, _p(s.q), H, case.get("prefix", 0), scale, _p(s.out)))
        torch.cuda.synchronize()  # the context's stream does not wait for torch's
    f, a = s.call
    check(f(*a))
    return s.out


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------------------------- work, exact results


def work(case):
    H, KH, HD = DIMS[case["dims"]]
    page, prefix = case["page"], case.get("prefix", 0)
    _, pos, num = _rows_of(case)
    R = sum(num)
    if case["kind"] == "store":
        b = R * (8 * H * HD + 2 * KH * HD * (4 + 2))
        if case["bounds"]:
            b += sum((p + t - 1) // page + 1 - p // page for p, t in zip(pos, num)) * KH * HD * 4
        return {"bytes": b, "flops": 3 * R * (H + KH) * HD}
    row, qo = 4 * KH * HD, 8 * R * H * HD  # bytes of a position's key and value; queries and outputs
    if case["kind"] == "sparse":
        width, b, f = case["first"] + case["best"] + case["recent"], 0, 0
        for p, t in zip(pos, num):
            seen = [min(p + x + 1, width * page) for x in range(t)]
            b += (p + t + page - 1) // page * KH * HD * 4 + min(p + t, sum(seen)) * row
            f += sum(4 * HD * H * n + 4 * HD * H * ((p + t) // page) for n in seen)
        return {"bytes": b + qo + 4 * R * KH * width, "flops": f}
    read = prefix + sum(p + t - prefix for p, t in zip(pos, num))
    seen = sum(t * (p + 1) + t * (t - 1) // 2 for p, t in zip(pos, num))
    return {"bytes": read * row + qo, "flops": 4 * HD * H * seen}


def _exact_rows(pool, ids, n, page, HD, keys):
    """Values [KH, n, HD] in 64 bits of the pages ids, each by its own address."""
    off, x = torch.arange(page, device="cuda")[:, None], torch.arange(HD, device="cuda")
    if keys:
        where = off // 16 * 16 * HD + off // 4 % 2 * 8 * HD + x // 8 * 64 + (off // 8 % 2 * 4 + off % 4) * 8 + x % 8
    else:
        where = off // 8 * 8 * HD + x * 8 + off % 8
    v = pool[ids][:, :, where].double()
    return v.transpose(0, 1).reshape(v.shape[1], -1, HD)[:, :n]


def _exact_store(s, case):
    H, KH, HD = DIMS[case["dims"]]
    page, pos = case["page"], _positions(s).double()
    w = torch.exp(-torch.arange(HD // 2, device="cuda").double() * (2.0 * math.log(BASE) / HD))
    if s.freqs is not None:
        w = w / s.freqs.double()
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos[:, None] * w)[:, None]
    out = {}
    for name, x in (("q", s.q), ("k", s.k)):
        x = x.double()
        c = torch.complex(x[..., :HD // 2], x[..., HD // 2:]) if case["neox"] else torch.view_as_complex(
            x.reshape(*x.shape[:-1], HD // 2, 2).contiguous())
        c = c * z
        out[name] = torch.cat([c.real, c.imag], -1) if case["neox"] else torch.view_as_real(c).flatten(-2)
    K, V = s.K.double(), s.V.double()
    p = _positions(s)
    ids = torch.cat([s.table[q, (a + torch.arange(t, device="cuda")) // page] for q, a, t in
                     zip(s.seq, s.pos, s.num)]).long()
    off, x, h = (p % page)[:, None, None], torch.arange(HD, device="cuda"), torch.arange(KH, device="cuda")[:, None]
    kat = off // 16 * 16 * HD + off // 4 % 2 * 8 * HD + x // 8 * 64 + (off // 8 % 2 * 4 + off % 4) * 8 + x % 8
    vat = off // 8 * 8 * HD + x * 8 + off % 8
    K[ids[:, None, None], h, kat] = out["k"]
    V[ids[:, None, None], h, vat] = s.v.double()
    res = {"q": out["q"], "K": K, "V": V}
    if s.bounds is not None:
        b = s.bounds.double()
        for q, a, t in zip(s.seq, s.pos, s.num):
            for j in range(a // page, (a + t - 1) // page + 1):
                i = s.table[q, j:j + 1].long()
                k = _exact_rows(K, i, min(page, a + t - j * page), page, HD, True)
                b[i, :, 0], b[i, :, 1] = k.amin(1), k.amax(1)
        res["bounds"] = b
    return res


def _exact_blocks(q, lo, hi, case, cur):
    """The pages one row takes of one KV head: q [G, HD], lo, hi [pages, HD] in 64 bits."""
    first, recent, best = case["first"], case["recent"], case["best"]
    from_, to = min(first, cur + 1), max(min(first, cur + 1), cur + 1 - recent)
    sc = torch.maximum(q[:, None] * lo[from_:to], q[:, None] * hi[from_:to]).sum(-1).amax(0).cpu().numpy()
    pick = np.argsort(-sc, kind="stable")[:best] + from_
    return sorted(set(range(from_)) | set(int(x) for x in pick) | set(range(to, cur + 1)))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_store(s, case)
    H, KH, HD = DIMS[case["dims"]]
    page, G = case["page"], H // KH
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    width = case["first"] + case["best"] + case["recent"] if case["kind"] == "sparse" else 0
    blocks = torch.full((s.q.shape[0], KH, width), -1, dtype=torch.int32)
    at = 0
    for i, (p, t) in enumerate(zip(s.pos, s.num)):
        n = p + t
        ids = s.table[s.seq[i], :(n + page - 1) // page].long()
        q = s.q[at:at + t].double()
        place = torch.arange(n, device="cuda")
        K, V = _exact_rows(s.K, ids, n, page, HD, True), _exact_rows(s.V, ids, n, page, HD, False)
        for g in range(KH):
            see = (place <= p + torch.arange(t, device="cuda")[:, None])
            if case["kind"] == "sparse":
                b = s.bounds[ids, g].double()
                for r in range(t):
                    got = _exact_blocks(q[r, g * G:(g + 1) * G], b[:, 0], b[:, 1], case, (p + r) // page)
                    blocks[at + r, g, :len(got)] = torch.tensor(got, dtype=torch.int32)
                    see[r] &= torch.isin(place // page, torch.tensor(got, device="cuda"))
            for h in range(g * G, (g + 1) * G):
                S = torch.mm(q[:, h], K[g].t().contiguous()) * HD ** -0.5
                S[~see] = -math.inf
                out[at:at + t, h] = torch.mm(torch.softmax(S, 1), V[g])
        at += t
    return {"out": out, "blocks": blocks} if width else out
