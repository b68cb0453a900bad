"""Operators of a long served conversation, as cases that can be timed and compared: the KV cache in 4 bits,
the attention that reads it, attention with a sliding window and a few first tokens that stay visible, and
the draw of the next token.

listed() names the cases, draw() gives more of the same ranges, prepare() makes what the program holds before
the call, run() is one pass (the plain form in elementary torch operations, or, with `own`, this library's
calls) and exact() the same outputs in 64 bits, written apart.

The kinds of case:
  store   a sequence's keys and values into the 4-bit caches, and those rows read back as values
  kv4     attention of T rows of one sequence over 4-bit caches (window and first tokens optional)
  batch   attention of one row of each of N sequences, each over its slot of the 4-bit pools
  window  attention of T rows of one sequence over fp16 caches with a window and first tokens
  sample  the next token of each row of logits by temperature, top-k, top-p, min-p and a given number

A 4-bit cache holds, per KV head, tiles of 32 positions. Values come in blocks of 32 of a head's row: a scale
d of 8 significant bits (held as 16 d in fp16) and 16 codes n, the value (n - 8) d. A tile is its codes, then
its scales; TILES below says in which order.
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
        # a decode step's new row of one layer: the smallest call
        {"name": "store_8b_t1", "kind": "store", "dims": "8b", "T": 1, "pos0": 700},
        # a prompt's rows of one layer
        {"name": "store_8b_t2000", "kind": "store", "dims": "8b", "T": 2000, "pos0": 41},
        # a guess-ahead pass of a small model, odd lengths
        {"name": "kv4_1b_t7_at_333", "kind": "kv4", "dims": "1b", "T": 7, "pos0": 333, "window": 0, "sinks": 0},
        # a decode step of the benchmark's model late in a conversation
        {"name": "kv4_70b_t1_at_4000", "kind": "kv4", "dims": "70b", "T": 1, "pos0": 4000, "window": 0, "sinks": 0},
        # a decode step over a book: what the 4 bits are for
        {"name": "kv4_8b_t1_at_131000", "kind": "kv4", "dims": "8b", "T": 1, "pos0": 131000, "window": 0, "sinks": 0},
        # a server's step: conversations of all lengths
        {"name": "kv4_70b_batch_32", "kind": "batch", "dims": "70b", "N": 32, "positions": 9001, "window": 0, "sinks": 0},
        # the second part of a long document's prompt
        {"name": "kv4_8b_t2048_at_2048", "kind": "kv4", "dims": "8b", "T": 2048, "pos0": 2048, "window": 0, "sinks": 0},
        # a decode step of an endless chat: fp16 caches, a window and four first tokens
        {"name": "window_8b_t1_at_30000", "kind": "window", "dims": "8b", "T": 1, "pos0": 30000, "window": 4096,
         "sinks": 4},
        # a long prompt through a window
        {"name": "window_8b_t1500_at_6001", "kind": "window", "dims": "8b", "T": 1500, "pos0": 6001, "window": 1024,
         "sinks": 4},
        # one chat's next token with the usual filters
        {"name": "sample_1x128256", "kind": "sample", "rows": 1, "n": 128256, "temperature": 0.8, "top_k": 40,
         "top_p": 0.95, "min_p": 0.05, "mixed": False},
        # a server's step: every row with its own settings
        {"name": "sample_64x128256_mixed", "kind": "sample", "rows": 64, "n": 128256, "temperature": 1.0, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "mixed": True},
        # no filter at all: the whole vocabulary of a small model
        {"name": "sample_5x32003_plain", "kind": "sample", "rows": 5, "n": 32003, "temperature": 1.3, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0, "mixed": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "kv4", "kv4", "kv4", "batch", "window", "window", "sample", "sample"])
    dims = rng.choice(["1b", "8b", "70b"])
    if kind == "store":
        return {"kind": kind, "dims": dims, "T": _log(rng, 1, 2500), "pos0": rng.choice([0, _log(rng, 1, 5000)])}
    mask = rng.choice([(0, 0), (0, 0), (_log(rng, 1, 5000), 0), (_log(rng, 16, 5000), rng.randint(1, 70))])
    if kind == "batch":
        return {"kind": kind, "dims": dims, "N": rng.randint(2, 40), "positions": _log(rng, 30, 8000), "window": mask[0],
                "sinks": mask[1]}
    if kind in ("kv4", "window"):
        T = rng.choice([1, 1, rng.randint(2, 15), _log(rng, 16, 300), _log(rng, 16, 1500)])
        if kind == "window" and not mask[0]:
            mask = (_log(rng, 16, 5000), rng.randint(0, 16))
        top = 100000 if T == 1 else 10000 if T < 400 else 2500
        return {"kind": kind, "dims": dims if T < 400 else rng.choice(["1b", "8b"]), "T": T,
                "pos0": rng.choice([0, _log(rng, 1, top), _log(rng, 1, top)]), "window": mask[0], "sinks": mask[1]}
    return {"kind": kind, "rows": rng.choice([1, 1, rng.randint(2, 48)]), "n": _log(rng, 1000, 130000),
            "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.6]), "top_k": rng.choice([0, 0, 1, 20, _log(rng, 2, 2000)]),
            "top_p": rng.choice([1.0, 0.5, 0.9, 0.95, 0.999]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]),
            "mixed": rng.random() < 0.3}


# ------------------------------------------------------------------------------------- inputs


class State:
    pass


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000 + salt)
    return g


def _normal(shape, seed, salt, scale=1.0):
    return torch.randn(shape, device="cuda", generator=_gen(seed, salt)) * scale


def _keys(rows, KH, HD, seed, salt):
    """Keys as trained models have them: a few channels of every head far larger than the rest."""
    k = _normal((rows, KH, HD), seed, salt)
    big = torch.rand((KH, HD), device="cuda", generator=_gen(seed, salt + 1)) < 0.03
    return torch.where(big, 5.0 * k, k)


# The tile of 32 positions of a KV head. Keys: position 0..31, then 8 values to a 32-bit word (value 2 p + h of
# the 8 at bit 16 h + 4 p); scales: position % 16, block, position / 16. Values: word order e, kq, x, jp and in
# a word half h, nibble i, for value 4 E x + 4 e + i (E = head dim / 64) of position 16 t + 4 kq + r, where
# 4 t + r = 2 jp + h; scales: kq, block, 4 t + r.
TILE = 32


def _held(x):
    """x [rows][KH][HD] as 4-bit blocks: codes (int32, 0..15) and d (float32, [rows][KH][HD / 32])."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = b.abs()
    at = torch.where(a == a.amax(-1, keepdim=True), torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = b.gather(-1, at) / -8
    e = (torch.frexp(d).exponent - 8).clamp_(min=-24)
    d = torch.ldexp(torch.round(torch.ldexp(d, -e)), e).clamp_(-2720, 2720)
    one = torch.where(d == 0, torch.ones_like(d), d).double()
    n = torch.where(d == 0, 8.0, (torch.round(b.double() / one) + 8).clamp_(0, 15))
    return n.to(torch.int32).reshape(x.shape), d.squeeze(-1)


def _pack(x, positions, keys):
    """The bytes of one cache [KH][tiles][18 HD] with x [rows][KH][HD] in its first rows, zeros after them."""
    rows, KH, HD = x.shape
    tiles, E, NB = (positions + TILE - 1) // TILE, HD // 64, HD // 32
    n, d = _held(x)
    pad = tiles * TILE - rows
    n = torch.nn.functional.pad(n, (0, 0, 0, 0, 0, pad), value=8).reshape(tiles, TILE, KH, HD)
    d = torch.nn.functional.pad(d, (0, 0, 0, 0, 0, pad)).reshape(tiles, 2, 16, KH, NB)
    if keys:
        w = n.reshape(tiles, TILE, KH, HD // 8, 4, 2)
        at = 4 * torch.arange(4, device=x.device)[:, None] + 16 * torch.arange(2, device=x.device)
        w = (w.to(torch.int64) << at).sum((-1, -2)).permute(2, 0, 1, 3)
        s = d.permute(3, 0, 2, 4, 1)
    else:
        w = n.reshape(tiles, 2, 4, 2, 2, KH, 16, E, 4)  # t, kq, jp % 2, h; x, e, i
        at = 16 * torch.arange(2, device=x.device).reshape(2, 1, 1, 1, 1) + 4 * torch.arange(4, device=x.device)
        w = (w.to(torch.int64) << at).sum((4, 8)).permute(4, 0, 6, 2, 5, 1, 3)
        s = d.reshape(tiles, 2, 4, 4, KH, NB).permute(4, 0, 2, 5, 1, 3)
    w = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32).reshape(KH, tiles, -1).contiguous().view(torch.uint8)
    s = (16 * s).to(torch.float16).reshape(KH, tiles, -1).contiguous().view(torch.uint8)
    return torch.cat([w, s], -1)


def _batch_rows(case):
    """Position and slot of each row: lengths from short to full, slots in another order."""
    N, top = case["N"], case["positions"]
    pos = [top - 1 - (i * top) // N * (i % 4) // 3 for i in range(N)]
    return pos, [(5 * i + 3) % N if N % 5 else N - 1 - i for i in range(N)]


def _settings(case):
    """(temperature, top_k, top_p, min_p) of each row."""
    base = (case["temperature"], case["top_k"], case["top_p"], case["min_p"])
    if not case["mixed"]:
        return [base] * case["rows"]
    more = [base, (0.7, 40, 1.0, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.05), (0.9, 200, 0.9, 0.02),
            (1.0, 0, 1.0, 0.0)]
    return [more[i % len(more)] for i in range(case["rows"])]


def prepare(case, seed):
    s = State()
    s.case, kind = case, case["kind"]
    if kind == "sample":
        # a flat bulk and some dozens of tokens that stand out
        s.logits = _normal((case["rows"], case["n"]), seed, 0, 2.0)
        up = torch.rand(s.logits.shape, device="cuda", generator=_gen(seed, 1)) < 60.0 / case["n"]
        s.logits += up * torch.rand(s.logits.shape, device="cuda", generator=_gen(seed, 2)) * 12.0
        s.u = torch.rand(case["rows"], device="cuda", generator=_gen(seed, 3))
        s.settings = _settings(case)
        return s
    H, KH, HD = DIMS[case["dims"]]
    if kind == "batch":
        N, top = case["N"], case["positions"]
        s.pos, s.slot = _batch_rows(case)
        s.K = torch.stack([_pack(_keys(top, KH, HD, seed, 10 + 3 * i), top, True) for i in range(N)])
        s.V = torch.stack([_pack(_normal((top, KH, HD), seed, 12 + 3 * i), top, False) for i in range(N)])
        s.q = _normal((N, H, HD), seed, 1, 2.0)
        s.row_pos, s.row_slot = torch.tensor(s.pos, device="cuda"), torch.tensor(s.slot, device="cuda")
        return s
    T, n = case["T"], case["pos0"] + case["T"]
    k, v = _keys(n, KH, HD, seed, 10), _normal((n, KH, HD), seed, 12)
    if kind == "store":
        # the cache before the call, and the rows to come
        s.K, s.V = _pack(k[:case["pos0"]], n, True), _pack(v[:case["pos0"]], n, False)
        s.k, s.v = k[case["pos0"]:].contiguous(), v[case["pos0"]:].contiguous()
        return s
    s.q = _normal((T, H, HD), seed, 1, 2.0)
    if kind == "kv4":
        s.K, s.V = _pack(k, n, True), _pack(v, n, False)
    else:
        s.K, s.V = k.to(torch.float16), v.to(torch.float16)
    return s


# ------------------------------------------------------------------------------------- plain forms


def _unpack(c, HD, keys):
    """The values [..., KH, positions, HD] in fp32 of caches [..., KH, tiles, 18 HD]."""
    E, NB, lead = HD // 64, HD // 32, c.shape[:-1]
    w = c[..., :16 * HD].contiguous().view(torch.int32)
    d = c[..., 16 * HD:].contiguous().view(torch.float16).float() / 16
    if keys:
        at = (4 * torch.arange(4, device=c.device)[:, None] + 16 * torch.arange(2, device=c.device)).int()
        n = (w[..., None, None] >> at) & 15
        d = d.reshape(*lead, 16, NB, 2).movedim(-1, -3)
    else:
        at = (16 * torch.arange(2, device=c.device)[:, None] + 4 * torch.arange(4, device=c.device)).int()
        n = (w.reshape(*lead, E, 4, 16, 2, 2)[..., None, None] >> at) & 15  # e, kq, x, t, jp % 2, h, i
        n = n.movedim((-4, -6, -3, -2, -5, -7), (-7, -6, -5, -4, -3, -2))   # t, kq, jp % 2, h, x, e, i
        d = d.reshape(*lead, 4, NB, 2, 4).movedim((-2, -4, -1), (-4, -3, -2))
    x = (n.reshape(*lead, TILE, NB, 32) - 8) * d.reshape(*lead, TILE, NB, 1)
    return x.reshape(*lead[:-1], lead[-1] * TILE, HD)


def _attend(q, K, V, see, HD):
    """Rows q [..., T, H, HD] over K, V [..., KH, n, HD]; see [..., T, n] says which positions a row sees."""
    T, H, KH = q.shape[-3], q.shape[-2], K.shape[-3]
    q = q.reshape(*q.shape[:-2], KH, H // KH, HD).movedim(-4, -2)               # KH, G, T, HD
    S = torch.matmul(q.reshape(*q.shape[:-3], -1, HD), K.transpose(-1, -2).contiguous()) / math.sqrt(HD)
    S = S.reshape(*q.shape[:-1], K.shape[-2]).masked_fill_(~see[..., None, None, :, :], -math.inf)
    P = torch.exp(S - S.amax(-1, keepdim=True))
    P = P / P.sum(-1, keepdim=True)
    o = torch.matmul(P.reshape(*P.shape[:-4], KH, -1, P.shape[-1]), V)
    return o.reshape(*q.shape).movedim(-2, -4).reshape(*q.shape[:-4], T, H, HD)


def _sees(pos, at, window, sinks):
    """Whether a row at position pos sees position at."""
    see = at <= pos
    return see & ((at < sinks) | (at > pos - window)) if window else see


def _plain(s):
    case, kind = s.case, s.case["kind"]
    if kind == "sample":
        return _plain_sample(s.logits, s.u, s.settings)
    H, KH, HD = DIMS[case["dims"]]
    if kind == "store":
        out = []
        for x in (s.k, s.v):
            n, d = _held(x)
            out.append(((n - 8).reshape(*d.shape, 32) * d[..., None]).reshape(x.shape))
        return {"k": out[0], "v": out[1]}
    if kind == "batch":
        K, V = _unpack(s.K[s.row_slot], HD, True), _unpack(s.V[s.row_slot], HD, False)
        at = torch.arange(K.shape[-2], device="cuda")
        see = _sees(s.row_pos[:, None], at, case["window"], case["sinks"])
        return _attend(s.q[:, None], K, V, see[:, None], HD)[:, 0]
    pos0, T = case["pos0"], case["T"]
    lo = max(0, pos0 - case["window"] + 1) if case["window"] else 0
    lo = lo // TILE * TILE  # positions before the first row's window, but for the first tokens, are left out
    first = min(lo, case["sinks"])
    at = torch.cat([torch.arange(first, device="cuda"), torch.arange(lo, pos0 + T, device="cuda")])
    if kind == "kv4":
        K, V = _unpack(s.K, HD, True)[:, at], _unpack(s.V, HD, False)[:, at]
    else:
        K, V = s.K[at].float().movedim(0, 1), s.V[at].float().movedim(0, 1)
    see = _sees(pos0 + torch.arange(T, device="cuda")[:, None], at, case["window"], case["sinks"])
    return _attend(s.q, K, V, see, HD)


def _plain_sample(logits, u, settings):
    t, k, p, m = (torch.tensor(x, dtype=torch.float32, device="cuda").double()[:, None] for x in zip(*settings))
    n = logits.shape[1]
    l, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    w = torch.exp((l.double() - l[:, :1].double()) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(n, device="cuda")
    k = torch.where((k <= 0) | (k > n), n, k).long()
    k = torch.where(t > 0, k, 1)
    mass = torch.cumsum(w, 1)
    kept = (rank < k) & (w >= m) & ((p >= 1) | (rank == 0) | (mass - w < p * mass.gather(1, k - 1)))
    last = kept.sum(1, keepdim=True) - 1
    drawn = (mass <= u.double()[:, None] * mass.gather(1, last)).sum(1, keepdim=True)
    return ids.gather(1, torch.minimum(drawn, last))[:, 0].to(torch.int32)


# ------------------------------------------------------------------------------------- the library's calls

_ctx = []


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def _own(s):
    from windlass_amd._lib import check, load
    from windlass_amd.backend import Context, SampleParams
    if not _ctx:
        _ctx.append(Context(0))
    case, L, h = s.case, load(), _ctx[0].handle
    if not hasattr(s, "call"):  # the buffers and arguments that a program keeps from step to step
        kind = case["kind"]
        if kind == "sample":
            ps = (SampleParams * case["rows"])(*[SampleParams(*x) for x in s.settings])
            s.out = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
            a = (h, _p(s.logits), case["rows"], case["n"], ps, _p(s.u), _p(s.out))
            s.call = [(L.wl_sample_dev, a)]
        else:
            H, KH, HD = DIMS[case["dims"]]
            scale = ctypes.c_float(1.0 / math.sqrt(HD))
            if kind == "store":
                n, pos0, T = case["pos0"] + case["T"], case["pos0"], case["T"]
                s.out = {"k": torch.empty_like(s.k), "v": torch.empty_like(s.v)}
                s.call = [(L.wl_kv4_store_dev, (h, _p(s.k), _p(s.v), T, KH, HD, _p(s.K), _p(s.V), n, pos0)),
                          (L.wl_kv4_read_dev, (h, _p(s.K), _p(s.V), n, KH, HD, pos0, T, _p(s.out["k"]), _p(s.out["v"])))]
            elif kind == "batch":
                N = case["N"]
                s.out = torch.empty_like(s.q)
                a = (h, _p(s.q), N, H, KH, HD, _p(s.K), _p(s.V), (ctypes.c_int32 * N)(*s.pos),
                     (ctypes.c_int32 * N)(*s.slot), N, case["positions"], case["window"], case["sinks"], scale, _p(s.out))
                s.call = [(L.wl_kv4_attention_batch_dev, a)]
            else:
                n = case["pos0"] + case["T"]
                s.out = torch.empty_like(s.q)
                a = (h, _p(s.q), case["T"], H, KH, HD, _p(s.K), _p(s.V)) + ((n,) if kind == "kv4" else ())
                a += (case["pos0"], case["window"], case["sinks"], scale, _p(s.out))
                s.call = [(L.wl_kv4_attention_dev if kind == "kv4" else L.wl_attention_window_dev, a)]
        torch.cuda.synchronize()  # the context's stream does not wait for torch's
    for f, a in s.call:
        check(f(*a))
    return s.out


def run(s):
    return _own(s) if own else _plain(s)


# ------------------------------------------------------------------------------------- work, exact results


def _visible(p, window, sinks):
    return p + 1 if not window or window > p else window + min(sinks, p + 1 - window)


def work(case):
    kind = case["kind"]
    if kind == "sample":
        return {"bytes": case["rows"] * (4 * case["n"] + 8), "flops": 10 * case["rows"] * case["n"]}
    H, KH, HD = DIMS[case["dims"]]
    if kind == "store":  # fp32 rows in, 4.5 bits a value into the caches, fp32 rows out
        return {"bytes": case["T"] * 2 * KH * HD * (4 + 0.5625 + 4), "flops": 4 * case["T"] * 2 * KH * HD}
    w, f = case["window"], case["sinks"]
    per = 2 * KH * HD * (2 if kind == "window" else 0.5625)  # bytes of a position's key and value
    if kind == "batch":
        seen = [_visible(p, w, f) for p in _batch_rows(case)[0]]
        read, rows = sum(seen), case["N"]
    else:
        seen = [_visible(case["pos0"] + t, w, f) for t in range(case["T"])]
        rows, last = case["T"], case["pos0"] + case["T"] - 1
        lo = max(0, case["pos0"] - w + 1) if w else 0
        read = last + 1 - lo + min(f, lo)
    return {"bytes": read * per + 8 * rows * H * HD, "flops": 4 * HD * H * sum(seen)}


def _exact_values(c, HD, keys, at):
    """Values [KH][len(at)][HD] in 64 bits of one cache's positions, each by its own address in the tile."""
    E, NB = HD // 64, HD // 32
    p, x = at[:, None], torch.arange(HD, device=at.device)
    tile, r = p // TILE, p % TILE
    if keys:
        byte = r * (HD // 2) + (x // 8) * 4 + 2 * (x % 2) + (x % 8) // 4
        shift = 4 * ((x % 8 // 2) % 2) + 0 * r
        sc = ((r % 16) * NB + x // 32) * 2 + r // 16
    else:
        kq, j = r % 16 // 4, 4 * (r // 16) + r % 4
        lane, e, i = x // (4 * E), x % (4 * E) // 4, x % 4
        byte = (((e * 4 + kq) * 16 + lane) * 4 + j // 2) * 4 + 2 * (j % 2) + i // 2
        shift = 4 * (i % 2) + 0 * r
        sc = (kq * NB + x // 32) * 8 + j
    codes = (c[:, tile.expand_as(byte), byte].long() >> shift) & 15
    scales = c[..., 16 * HD:].contiguous().view(torch.float16)[:, tile.expand_as(sc), sc].double() * 2.0 ** -4
    return (codes - 8).double() * scales


def _exact_rows(q, K, V, see):
    """q [T][HD] over K, V [n][HD] of one head, in 64 bits."""
    S = torch.mm(q, K.t().contiguous()) * K.shape[1] ** -0.5
    S[~see] = -math.inf
    S = torch.softmax(S, 1)
    return torch.mm(S, V)


def _exact_held(x):
    b = x.double().reshape(-1, 32)
    out = torch.empty_like(b)
    a = b.abs()
    m = b[torch.arange(b.shape[0], device=b.device), (a == a.max(1, keepdim=True).values).double().argmax(1)]
    e = torch.floor(torch.log2((m / 8).abs().clamp(min=1e-300))).clamp(min=-17.0) - 7.0
    d = (torch.round(-m / 8 * torch.exp2(-e)) * torch.exp2(e)).clamp(-2720, 2720)
    # the nearest of the sixteen multiples of d; of two as near, the even one
    v = torch.arange(-8, 8, device=b.device, dtype=torch.float64)
    for i in range(0, b.shape[0], 1 << 16):
        c = v * d[i:i + (1 << 16), None]
        off = (b[i:i + (1 << 16), :, None] - c[:, None, :]).abs()
        near = torch.where(off == off.min(-1, keepdim=True).values, v.abs() % 2, 2.0)
        out[i:i + (1 << 16)] = c.gather(1, near.argmin(-1))
    return out.reshape(x.shape)


def _exact_sample(l, u, t, k, p, m):
    l = l.cpu().numpy()
    order = np.argsort(-l, kind="stable")
    if t == 0:
        return int(order[0])
    l = l[order].astype(np.float64)
    w = np.exp((l - l[0]) / np.float64(np.float32(t)))
    mass = np.cumsum(w)
    n = k if 0 < k < len(w) else len(w)
    if p < 1:
        cut = np.searchsorted(np.concatenate([[0.0], mass[:-1]]), np.float64(np.float32(p)) * mass[n - 1], side="left")
        n = min(n, max(1, int(cut)))
    n = min(n, int(np.count_nonzero(w >= np.float64(np.float32(m)))))
    return int(order[min(n - 1, int(np.searchsorted(mass[:n], np.float64(u) * mass[n - 1], side="right")))])


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "sample":
        u = s.u.cpu().numpy()
        got = [_exact_sample(s.logits[i], u[i], *s.settings[i]) for i in range(case["rows"])]
        return torch.tensor(got, dtype=torch.int32)
    if kind == "store":
        return {"k": _exact_held(s.k), "v": _exact_held(s.v)}
    H, KH, HD = DIMS[case["dims"]]
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    rows = range(case["N"]) if kind == "batch" else [None]
    for i in rows:
        pos = torch.tensor([s.pos[i]], device="cuda") if kind == "batch" else case["pos0"] + torch.arange(case["T"], device="cuda")
        at = torch.arange(int(pos[-1]) + 1, device="cuda")
        see = _sees(pos[:, None], at, case["window"], case["sinks"])
        at, see = at[see.any(0)], see[:, see.any(0)]
        q = s.q[i:i + 1] if kind == "batch" else s.q
        o = out[i:i + 1] if kind == "batch" else out
        for g in range(KH):
            if kind == "window":
                K, V = s.K[at, g].double(), s.V[at, g].double()
            else:
                Kc, Vc = (s.K[s.slot[i]], s.V[s.slot[i]]) if kind == "batch" else (s.K, s.V)
                K, V = (_exact_values(c[g:g + 1], HD, keys, at)[0] for c, keys in ((Kc, True), (Vc, False)))
            for h in range(g * (H // KH), (g + 1) * (H // KH)):
                o[:, h] = _exact_rows(q[:, h].double(), K, V, see)
    return out
