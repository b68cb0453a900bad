"""KV caches in pages: rows rotated and stored, read back, attended to, with a shared prefix, and pages chosen by their
bounds, each against a plain restatement in 64 bits (tests/paged_ref.py)."""
import ctypes

import numpy as np
import pytest

from paged_ref import F32, Pool, attend_ref, blocks_ref, key_at, rope_ref, val_at
from windlass_amd._lib import check, load
from windlass_amd.backend import Context, PageRows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with Context(0) as c:
        yield c


def normal(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(F32)


def same(a, b):
    return np.array_equal(np.ascontiguousarray(a).view(np.uint32), np.ascontiguousarray(b).view(np.uint32))


def near(got, want, tol, what):
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= tol)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of %.3g" % (
        what, int(bad.sum()), bad.size, float(np.nanmax(off)), float(np.broadcast_to(tol, off.shape).flat[np.nanargmax(off)]))


def entries_ref(pool, seq, pos, rows, q, scale, prefix=0):
    out, tol, at = [], [], 0
    for s, p, t in zip(seq, pos, rows):
        sees = [[np.arange(p + i + 1)] * pool.KH for i in range(t)]
        o, e = attend_ref(q[at:at + t], pool.K[s], pool.V[s], sees, scale)
        out.append(o)
        tol.append(e)
        at += t
    return np.concatenate(out), np.concatenate(tol)


# ------------------------------------------------------------------------------------- stores


@pytest.mark.parametrize("H,KH,HD,page,n,neox", [(8, 2, 64, 16, 64, 0), (8, 2, 64, 64, 64, 1), (16, 2, 128, 64, 128, 0),
                                                 (6, 2, 128, 32, 64, 1), (3, 3, 128, 256, 128, 1), (5, 1, 64, 128, 2, 0),
                                                 (8, 8, 128, 16, 0, 0)])
def test_store_rotates_and_places(ctx, H, KH, HD, page, n, neox):
    rng = np.random.default_rng(H * HD + page)
    lengths = [300, 17, 1, 64, 90]
    pool = Pool(ctx, lengths, KH, HD, page, seed=3, bounds=True, room=400)
    before = [pool.read(s, 0, lengths[s]) for s in range(5)]
    for s in range(5):  # what the constructor stored
        assert same(before[s][0], pool.K[s]) and same(before[s][1], pool.V[s])
    seq, pos, rows = [3, 0, 4, 2], [64, 300, 83, 1], [33, 1, 150, 0]  # a rewrite, and an entry without rows
    R = sum(rows)
    q, k, v = normal(rng, R, H, HD), normal(rng, R, KH, HD), normal(rng, R, KH, HD)
    freqs = (1 + 7 * rng.random(max(n // 2, 1))).astype(F32) if page != 32 else None
    got = pool.store(seq, pos, rows, q, k, v, n, neox, 500000.0, 0.25 if page == 16 else 1.0, freqs)
    fs = 0.25 if page == 16 else 1.0
    places = np.concatenate([p + np.arange(t) for p, t in zip(pos, rows)])
    want, tol = rope_ref(q, places, n, neox, 500000.0, fs, freqs)
    near(got, want, tol, "q")
    wk, ktol = rope_ref(k, places, n, neox, 500000.0, fs, freqs)
    at = 0
    for s, p, t in zip(seq, pos, rows):
        gk, gv = pool.read(s, 0, p + t)
        assert same(gk[:p], before[s][0][:p]) and same(gv[:p], before[s][1][:p])  # rows before are as they were
        w = wk[at:at + t]
        near(gk[p:], w, ktol[at:at + t] + np.abs(w) * 2.0 ** -11 + 2.0 ** -25, "k of %d" % s)
        assert same(gv[p:], v[at:at + t].astype(np.float16).astype(F32))
        pool.K[s] = np.concatenate([pool.K[s][:p], gk[p:]])
        at += t
    # bounds: over the pages' positions up to the last one stored
    for s, p, t in zip(seq, pos, rows):
        if not t:
            continue
        b = pool.bounds_of(s, (p + t + page - 1) // page)
        for j in range((p + t + page - 1) // page):
            part = pool.K[s][j * page:min((j + 1) * page, p + t)]
            assert np.array_equal(b[j, :, 0], part.min(0)) and np.array_equal(b[j, :, 1], part.max(0)), (s, j)
    # everything else in the pool is NaN still
    raw = pool.dK.reshape(pool.pages, KH, page * HD).cpu().numpy()
    rawv = pool.dV.reshape(pool.pages, KH, page * HD).cpu().numpy()
    off, d = np.arange(page)[:, None], np.arange(HD)
    for s in range(5):
        top = max([lengths[s]] + [p + t for z, p, t in zip(seq, pos, rows) if z == s])
        for j in range(pool.table.shape[1]):
            free = np.arange(page) + j * page >= top
            for r, f in ((raw, key_at), (rawv, val_at)):
                x = r[pool.table[s, j]][:, f(off, d, HD)]
                assert np.isnan(x[:, free]).all() and not np.isnan(x[:, ~free]).any(), (s, j)
    unused = sorted(set(range(pool.pages)) - set(pool.table.reshape(-1).tolist()))
    assert np.isnan(raw[unused]).all() and np.isnan(rawv[unused]).all()


@pytest.mark.parametrize("T", [1, 5, 70])
@pytest.mark.parametrize("HD,n,neox", [(64, 64, 1), (128, 128, 0), (128, 96, 1)])
def test_stored_rows_have_the_other_caches_bits(ctx, T, HD, n, neox):
    """The same queries and keys as wl_rope_dev and wl_kv_store_dev give, bit for bit, also in place."""
    import torch
    L, KH, H, pos0 = load(), 2, 6, 4090
    rng = np.random.default_rng(T)
    q, k, v = normal(rng, T, H, HD), normal(rng, T, KH, HD, scale=3), normal(rng, T, KH, HD)
    freqs = (1 + 7 * rng.random(n // 2)).astype(F32)
    pool = Pool(ctx, [1], KH, HD, 64, room=5000)
    a = pool.store([0], [pos0], [T], q, k, v, n, neox, 10000.0, 1.0, freqs)
    b = pool.store([0], [pos0], [T], q, k, v, n, neox, 10000.0, 1.0, freqs, inplace=True)
    dq, dk, dv, df = (pool.dev(x) for x in (q, k, v, freqs))
    Kc, Vc = (torch.zeros((pos0 + T, KH * HD), dtype=torch.float16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    for x, heads in ((dq, H), (dk, KH)):
        check(L.wl_rope_dev(ctx.handle, x.data_ptr(), T, heads, HD, n, neox, pos0, None, 10000.0, 1.0, df.data_ptr()))
    check(L.wl_kv_store_dev(ctx.handle, dk.data_ptr(), dv.data_ptr(), T, KH * HD, Kc.data_ptr(), Vc.data_ptr(), pos0))
    ctx.sync()
    assert same(a, dq.cpu().numpy()) and same(b, a)
    gk, gv = pool.read(0, pos0, T)
    assert same(gk, Kc[pos0:].float().reshape(T, KH, HD).cpu().numpy())
    assert same(gv, Vc[pos0:].float().reshape(T, KH, HD).cpu().numpy())


@pytest.mark.parametrize("H,KH,HD,page,n,neox", [(32, 8, 128, 64, 128, 0), (63, 3, 64, 16, 64, 1), (48, 1, 128, 256, 96, 1),
                                                 (64, 64, 64, 32, 0, 0)])
def test_prompts_of_many_rows(ctx, H, KH, HD, page, n, neox):
    """Past the rows that go by themselves: the formulas' values, and the bits of small calls."""
    rng = np.random.default_rng(H)
    every = (11 << 20) // ((H + KH) * HD)
    seq, pos, rows = [2, 0, 4, 1, 3], [5, 300, 16, 0, 37], [every // 2 + 3, every // 4, 1, 0, every // 4 + 8]
    lengths = [p + t + 1 for s, p, t in sorted(zip(seq, pos, rows))]
    R = sum(rows)
    assert R * (H + KH) * HD > 10 << 20
    q, k, v = normal(rng, R, H, HD), normal(rng, R, KH, HD), normal(rng, R, KH, HD)
    k[R // 3, 0, 3], k[R // 3 + 1, 0, 4] = np.nan, -np.inf
    freqs = (1 + 7 * rng.random(n // 2)).astype(F32) if n == 128 else None
    pools, got = [], []
    for many in (True, False):
        pool = Pool(ctx, [40] * 5, KH, HD, page, seed=3, bounds=True, room=max(lengths))
        if many:
            got.append(pool.store(seq, pos, rows, q, k, v, n, neox, 500000.0, 0.5, freqs))
        else:
            parts, at = [], 0
            for s, p, t in zip(seq, pos, rows):
                for i in range(0, t, 200):
                    m = min(200, t - i)
                    a = slice(at + i, at + i + m)
                    parts.append(pool.store([s], [p + i], [m], q[a], k[a], v[a], n, neox, 500000.0, 0.5, freqs))
                at += t
            got.append(np.concatenate(parts))
        pools.append(pool)
    assert same(*got)
    for x in ("dK", "dV", "dB"):
        a, b = (getattr(p, x).cpu().numpy().view(np.uint16) for p in pools)
        assert np.array_equal(a, b), x
    some = sorted({0, R // 3, R - 1, *rng.permutation(R)[:40].tolist()})
    places = np.concatenate([p + np.arange(t) for p, t in zip(pos, rows)])[some]
    want, tol = rope_ref(q[some], places, n, neox, 500000.0, 0.5, freqs)
    near(got[0][some], want, tol, "q")
    at = 0
    for s, p, t in zip(seq, pos, rows):
        if t:
            assert same(pools[0].read(s, p, t)[1], v[at:at + t].astype(np.float16).astype(F32))
        at += t


def test_more_entries_than_a_launch_takes(ctx):
    """300 sequences: stores, bounds and attention of entries past the first launch's."""
    rng = np.random.default_rng(5)
    N, KH, HD, H = 300, 1, 64, 4
    lengths = [1 + (7 * i) % 40 for i in range(N)]
    pool = Pool(ctx, lengths, KH, HD, 16, seed=9, bounds=True, room=1)
    seq = [(7 * i + 3) % N for i in range(N)]
    pos, rows = [lengths[s] for s in seq], [1] * N
    q, k, v = normal(rng, N, H, HD), normal(rng, N, KH, HD), normal(rng, N, KH, HD)
    pool.store(seq, pos, rows, q, k, v)
    for i, s in enumerate(seq):
        pool.K[s] = np.concatenate([pool.K[s], k[i:i + 1].astype(np.float16).astype(F32)])
        pool.V[s] = np.concatenate([pool.V[s], v[i:i + 1].astype(np.float16).astype(F32)])
        b = pool.bounds_of(s, pos[i] // 16 + 1)
        part = pool.K[s][pos[i] // 16 * 16:]
        assert np.array_equal(b[-1, :, 0], part.min(0)) and np.array_equal(b[-1, :, 1], part.max(0)), i
    want, tol = entries_ref(pool, seq, pos, rows, q, HD ** -0.5)
    near(pool.attend(seq, pos, rows, q), want, tol, "attention")


def test_bounds_keep_nan_and_infinity_and_forget_what_is_rewritten(ctx):
    KH, HD, page = 2, 64, 32

    def values(s, k, v):
        k[3, 0, 5], k[4, 1, 7], k[9, 0, 63] = np.nan, np.inf, -np.inf
    pool = Pool(ctx, [20], KH, HD, page, bounds=True, values=values)
    b = pool.bounds_of(0, 1)[0]
    assert np.isnan(b[0, :, 5]).all() and b[1, 1, 7] == np.inf and b[0, 0, 63] == -np.inf
    assert not np.isnan(np.delete(b[0], 5, axis=1)).any()
    k = np.zeros((1, KH, HD), F32)
    pool.store([0], [2], [1], None, k, k)  # back to three positions: the later ones no longer count
    part = np.concatenate([pool.K[0][:2], k])
    b = pool.bounds_of(0, 1)[0]
    assert np.array_equal(b[:, 0], part.min(0)) and np.array_equal(b[:, 1], part.max(0))


# ------------------------------------------------------------------------------------- attention

SHAPES = [(8, 8, 64, 16), (8, 2, 64, 32), (16, 2, 128, 64), (6, 2, 128, 16), (12, 1, 128, 256), (32, 2, 64, 128)]


@pytest.mark.parametrize("H,KH,HD,page", SHAPES)
def test_rows_of_many_lengths(ctx, H, KH, HD, page):
    rng = np.random.default_rng(H + HD + page)
    lengths = [1, 16, 17, 33, 140, 130, 334, 700, 255]
    pool = Pool(ctx, lengths, KH, HD, page, seed=1)
    seq, rows = [8, 0, 1, 2, 3, 4, 5, 6, 7], [0, 1, 1, 2, 7, 40, 130, 1, 16]
    pos = [lengths[s] - t for s, t in zip(seq, rows)]
    q = normal(rng, sum(rows), H, HD, scale=2)
    want, tol = entries_ref(pool, seq, pos, rows, q, HD ** -0.5)
    got = pool.attend(seq, pos, rows, q)
    near(got, want, tol, "rows")
    assert same(got, pool.attend(seq, pos, rows, q))
    at = 0
    for s, p, t in zip(seq, pos, rows):  # an entry's bits do not depend on the others
        if t:
            assert same(pool.attend([s], [p], [t], q[at:at + t]), got[at:at + t]), (s, t)
        at += t


def many_columns(T, H, pos):
    """More products than the entries that take few columns at a time have."""
    return T * H * (pos + T / 2) > 1 << 23


@pytest.mark.parametrize("H,KH,HD,page", [(64, 1, 64, 16), (64, 8, 128, 64), (96, 2, 128, 256), (130, 10, 64, 32)])
def test_rows_of_many_columns(ctx, H, KH, HD, page):
    rng = np.random.default_rng(H + HD)
    lengths = [700, 1500, 333, 1467, 20]
    pool = Pool(ctx, lengths, KH, HD, page, seed=1)
    seq, rows = [3, 0, 4, 1, 2, 1], [131, 700, 1, 400, 0, 5]
    pos = [lengths[s] - t for s, t in zip(seq, rows)]
    assert all(many_columns(t, H, p) for t, p in zip(rows, pos) if t > 100)
    q = normal(rng, sum(rows), H, HD, scale=2)
    got = pool.attend(seq, pos, rows, q)
    assert same(got, pool.attend(seq, pos, rows, q))
    at = 0
    for s, p, t in zip(seq, pos, rows):
        if t:
            assert same(pool.attend([s], [p], [t], q[at:at + t]), got[at:at + t]), (s, t)
        for i in sorted({0, t - 1, *rng.permutation(t)[:8].tolist()}) if t else ():
            want, tol = attend_ref(q[at + i:at + i + 1], pool.K[s], pool.V[s], [[np.arange(p + i + 1)] * KH], HD ** -0.5)
            near(got[at + i:at + i + 1], want, tol, (s, i))
        at += t


@pytest.mark.parametrize("H,KH,HD,page,n,T", [(8, 1, 128, 64, 20000, 1), (4, 1, 64, 16, 33001, 3), (8, 2, 128, 32, 9000, 100)])
def test_long_contexts(ctx, H, KH, HD, page, n, T):
    rng = np.random.default_rng(n)
    pool = Pool(ctx, [n], KH, HD, page, seed=2)
    q = normal(rng, T, H, HD, scale=2)
    want, tol = entries_ref(pool, [0], [n - T], [T], q, HD ** -0.5)
    near(pool.attend([0], [n - T], [T], q), want, tol, "long")


@pytest.mark.parametrize("T", [1, 3, 40])
def test_a_sequence_twice_and_a_page_shared(ctx, T):
    """Attention only reads: the same sequence in two entries, at other positions, and sequences of one beginning."""
    rng = np.random.default_rng(T)
    H, KH, HD, page = 8, 2, 64, 16
    pool = Pool(ctx, [200, 150], KH, HD, page, shared=64)
    seq, pos, rows = [0, 1, 0], [200 - T, 150 - T, 77], [T, T, T]
    q = normal(rng, 3 * T, H, HD)
    want, tol = entries_ref(pool, seq, pos, rows, q, HD ** -0.5)
    near(pool.attend(seq, pos, rows, q), want, tol, "twice")


@pytest.mark.parametrize("H,KH,HD,page", [(8, 2, 64, 32), (16, 2, 128, 16), (1200, 2, 64, 32), (1200, 4, 128, 16)])
@pytest.mark.parametrize("T", [1, 6, 50])
def test_missing_pages_are_not_seen(ctx, H, KH, HD, page, T):
    """Ids outside the pool: their positions are not seen, nothing is stored there, and a row that sees nothing gives zeros."""
    rng = np.random.default_rng(page + T)
    n = 180
    pool = Pool(ctx, [n, n, n], KH, HD, page, seed=4)
    far = (ctypes.c_int32 * 3)(2 ** 31 - 1, pool.pages, -2 ** 31)
    gone = {0: [1], 1: range(pool.table.shape[1]), 2: [n // page - 1, n // page]}
    import torch
    for s, js in gone.items():
        for i, j in enumerate(js):  # past what assign takes: written by another program
            pool.d_table[s, j] = far[i % 3]
    torch.cuda.synchronize()
    seq, pos, rows = [0, 1, 2], [n - T] * 3, [T] * 3
    q = normal(rng, 3 * T, H, HD)
    got = pool.attend(seq, pos, rows, q)
    for i, s in enumerate(seq):
        sees = []
        for t in range(T):
            at = np.arange(pos[i] + t + 1)
            at = at[~np.isin(at // page, list(gone[s]))]
            sees.append([at] * KH)
        want, tol = attend_ref(q[i * T:(i + 1) * T], pool.K[s], pool.V[s], sees, HD ** -0.5)
        near(got[i * T:(i + 1) * T], want, tol, "seq %d" % s)
    assert not got[T:2 * T].any()
    k = normal(rng, 3 * T, KH, HD)
    raw = pool.dK.clone()
    pool.store([1], [0], [T], None, k[:T], k[:T])
    assert torch.equal(raw.view(torch.int16), pool.dK.view(torch.int16))
    gk, gv = pool.read(1, 0, n)
    assert not gk.any() and not gv.any()


@pytest.mark.parametrize("H,KH,HD,page,T", [(8, 2, 64, 16, 1), (8, 2, 64, 16, 40), (8, 1, 128, 64, 1), (8, 1, 128, 64, 100),
                                            (4, 4, 128, 32, 5), (1024, 1, 64, 16, 90), (1024, 2, 128, 64, 100)])
def test_masked_infinities_and_visible_ones(ctx, H, KH, HD, page, T):
    """Values that no row sees may be anything; one that some rows see makes its column of those infinite or NaN, and of no
    others. Keys of -inf weigh nothing."""
    rng = np.random.default_rng(T + HD)
    n, x = 150, 11

    def values(s, k, v):
        v[n - 1, :, x] = np.inf          # the last row alone sees it
        v[40, 0, 3] = np.nan             # every row does
        k[20:30, :, 0] = -np.inf         # with positive queries there: scores of -inf
    pool = Pool(ctx, [n + 30], KH, HD, page, values=values)
    q = normal(rng, T, H, HD)
    q[..., 0] = np.abs(q[..., 0]) + 0.5
    got = pool.attend([0], [n - T], [T], q)
    K, V = pool.K[0].copy(), pool.V[0].copy()
    V[n - 1, :, x], V[40, 0, 3] = 0, 0
    sees = [[np.setdiff1d(np.arange(n - T + t + 1), np.arange(20, 30))] * KH for t in range(T)]
    want, tol = attend_ref(q, K, V, sees, HD ** -0.5)
    G = H // KH
    odd = np.zeros(got.shape, bool)
    odd[-1, :, x] = True
    odd[:, :G, 3] = True
    assert not np.isfinite(got[odd]).any()
    near(got[~odd], want[~odd], np.broadcast_to(tol, got.shape)[~odd], "the rest")


@pytest.mark.parametrize("H,T", [(4, 1), (4, 30), (4096, 30)])
@pytest.mark.parametrize("HD", [64, 128])
def test_scores_of_any_size(ctx, HD, H, T):
    """Scales of 0, below 0, huge and tiny; queries of very large and small values; infinite ones give what the formula does."""
    KH, n = 2, 90
    rng = np.random.default_rng(HD)
    pool = Pool(ctx, [n], KH, HD, 32)
    q = normal(rng, T, H, HD)
    args = ([0], [n - T], [T])
    for scale, f in ((0.0, 1.0), (-0.3, 1.0), (1e-30, 1e25), (1e4, 1.0), (1.0, 1e-40), (3e-38, 1e36)):
        x = (q * F32(f)).astype(F32)
        want, tol = entries_ref(pool, *args, x, float(F32(scale)))
        near(pool.attend(*args, x, scale=scale), want, np.minimum(tol, 2 * np.abs(pool.V[0]).max()), (scale, f))
    got = pool.attend(*args, np.full_like(q, np.nan))
    assert np.isnan(got).all() or not got.any()
    x = np.zeros_like(q)
    x[..., 0] = np.inf  # scores of +-inf: NaN where one is +inf
    assert np.isnan(pool.attend(*args, x)).all()


def test_pools_past_four_gigabytes(ctx):
    """Pages whose halves pass 2^31, keys and values and bounds' places in 64 bits."""
    import torch
    KH, HD, page, H, n, T = 8, 128, 256, 8, 700, 3
    pages = 2 ** 31 // (KH * HD * page) + 8  # 4.3 GB of keys
    rng = np.random.default_rng(0)
    small = Pool(ctx, [n], KH, HD, page, seed=8, bounds=True)
    big = [torch.empty(pages * KH * HD * page, dtype=torch.float16, device="cuda") for _ in range(2)]
    db = torch.zeros(pages * KH * 2 * HD, dtype=torch.float16, device="cuda")
    small.desc.d_K, small.desc.d_V, small.desc.d_bounds = big[0].data_ptr(), big[1].data_ptr(), db.data_ptr()
    small.desc.pages = small.pages = pages
    small.dB = db
    ids = [pages - 1, pages - 5, pages - 3]
    small.table[0, :3] = ids
    torch.cuda.synchronize()
    small.assign(0, 0, ids)
    small.store([0], [0], [n], None, small.K[0], small.V[0])
    q = normal(rng, T, H, HD)
    want, tol = entries_ref(small, [0], [n - T], [T], q, HD ** -0.5)
    near(small.attend([0], [n - T], [T], q), want, tol, "few rows")
    qm = normal(rng, 100, H, HD)
    want, tol = entries_ref(small, [0], [n - 100], [100], qm, HD ** -0.5)
    near(small.attend([0], [n - 100], [100], qm), want, tol, "rows")
    got, blocks = small.attend([0], [n - T], [T], q, sparse=(0, 1, 1))
    b = small.bounds_of(0, 3)
    for t in range(T):
        for g in range(KH):
            assert blocks[t, g].tolist() == blocks_ref(q[t, g:g + 1], b[:, g, 0], b[:, g, 1], 2, 0, 1, 1)


# ------------------------------------------------------------------------------------- a shared prefix


@pytest.mark.parametrize("H,KH,HD,page", SHAPES)
@pytest.mark.parametrize("prefix,N,T", [(256, 2, 1), (512, 5, 3), (2048, 40, 1), (256, 3, 50)])
def test_shared_prefix(ctx, H, KH, HD, page, prefix, N, T):
    rng = np.random.default_rng(prefix + H)
    lengths = [prefix + T + (13 * i) % 90 for i in range(N)]
    pool = Pool(ctx, lengths, KH, HD, page, seed=6, shared=prefix, room=1)
    seq = [(3 * i + 1) % N if N % 3 else N - 1 - i for i in range(N)]
    rows = [T] * N
    pos = [lengths[s] - T for s in seq]
    q = normal(rng, N * T, H, HD, scale=2)
    some = sorted(rng.permutation(N * T)[:12].tolist()) if N * T > 12 else list(range(N * T))
    got = pool.attend(seq, pos, rows, q, prefix=prefix)
    for r in some:
        s, p = seq[r // T], pos[r // T] + r % T
        want, tol = attend_ref(q[r:r + 1], pool.K[s], pool.V[s], [[np.arange(p + 1)] * KH], HD ** -0.5)
        near(got[r:r + 1], want, tol, "row %d" % r)
    assert same(got, pool.attend(seq, pos, rows, q, prefix=prefix))


@pytest.mark.parametrize("H,KH,HD,page", [(8, 2, 64, 32), (16, 2, 128, 256), (5, 1, 128, 16)])
@pytest.mark.parametrize("prefix,N,T", [(8192, 36, 1), (16384, 20, 3), (8192, 4, 50), (65536, 5, 1)])
def test_shared_prefix_that_is_read_once(ctx, H, KH, HD, page, prefix, N, T):
    rng = np.random.default_rng(prefix + H)
    lengths = [prefix + T + (13 * i) % 90 for i in range(N)]
    pool = Pool(ctx, lengths, KH, HD, page, seed=6, shared=prefix, room=1)
    pos = [n - T for n in lengths]
    q = normal(rng, N * T, H, HD, scale=2)
    got = pool.attend(list(range(N)), pos, [T] * N, q, prefix=prefix)
    for r in sorted({0, N * T - 1, *rng.permutation(N * T)[:6].tolist()}):
        p = pos[r // T] + r % T
        want, tol = attend_ref(q[r:r + 1], pool.K[r // T], pool.V[r // T], [[np.arange(p + 1)] * KH], HD ** -0.5)
        near(got[r:r + 1], want, tol, "row %d" % r)
    assert same(got, pool.attend(list(range(N)), pos, [T] * N, q, prefix=prefix))


@pytest.mark.parametrize("prefix", [320, 3200])
def test_prefix_with_more_entries_than_a_launch_takes(ctx, prefix):
    rng = np.random.default_rng(1)
    H, KH, HD, page, N = 4, 1, 64, 16, 200
    pool = Pool(ctx, [prefix + 1 + i % 20 for i in range(N)], KH, HD, page, shared=prefix, room=1)
    seq, pos = list(range(N)), [prefix + i % 20 for i in range(N)]
    q = normal(rng, N, H, HD)
    want, tol = entries_ref(pool, seq, pos, [1] * N, q, HD ** -0.5)
    near(pool.attend(seq, pos, None, q, prefix=prefix), want, tol, "prefix")


@pytest.mark.parametrize("N,T,prefix", [(3, 1, 128), (4, 40, 128), (9, 1, 16384), (4, 40, 4096), (4, 40, 8192)])
def test_prefix_with_missing_and_odd_pages(ctx, N, T, prefix):
    """A prefix whose pages are missing in part or all, an infinity in it, and rows that then see little."""
    import torch
    rng = np.random.default_rng(N)
    H, KH, HD, page = 8, 2, 128, 32

    def values(s, k, v):
        v[70, :, 4] = np.inf
    pool = Pool(ctx, [prefix + 60] * N, KH, HD, page, shared=prefix, values=values)
    q = normal(rng, N * T, H, HD)
    seq, pos, rows = list(range(N)), [prefix + 60 - T] * N, [T] * N
    for gone in ([1], list(range(prefix // page)), list(range(pool.table.shape[1]))):
        pool.d_table[:, gone] = -1
        torch.cuda.synchronize()
        got = pool.attend(seq, pos, rows, q, prefix=prefix)
        for i in range(N):
            V = pool.V[i].copy()
            V[70, :, 4] = 0
            ats = [np.arange(pos[i] + t + 1) for t in range(T)]
            sees = [[a[~np.isin(a // page, gone)]] * KH for a in ats]
            want, tol = attend_ref(q[i * T:(i + 1) * T], pool.K[i], V, sees, HD ** -0.5)
            odd = np.zeros(want.shape, bool)
            odd[..., 4] = 70 // page not in gone
            g = got[i * T:(i + 1) * T]
            assert not np.isfinite(g[odd]).any()
            near(g[~odd], want[~odd], np.broadcast_to(tol, want.shape)[~odd], gone)


# ------------------------------------------------------------------------------------- pages chosen by their bounds


def sparse_ref(pool, seq, pos, rows, q, opts, scale, gone=()):
    KH, G, page = pool.KH, q.shape[1] // pool.KH, pool.page
    out, tol, blocks, at = [], [], np.full((q.shape[0], KH, sum(opts)), -1, np.int32), 0
    for s, p, t in zip(seq, pos, rows):
        nb = (p + t + page - 1) // page
        b = pool.bounds_of(s, nb)
        sees = []
        for i in range(t):
            row = []
            for g in range(KH):
                lo = [None if j in gone else b[j, g, 0] for j in range(nb)]
                got = blocks_ref(q[at + i, g * G:(g + 1) * G], lo, b[:, g, 1], (p + i) // page, *opts)
                blocks[at + i, g, :len(got)] = got
                a = np.arange(p + i + 1)
                row.append(a[np.isin(a // page, got) & ~np.isin(a // page, gone)])
            sees.append(row)
        o, e = attend_ref(q[at:at + t], pool.K[s], pool.V[s], sees, scale)
        out.append(o)
        tol.append(e)
        at += t
    return np.concatenate(out), np.concatenate(tol), blocks


@pytest.mark.parametrize("H,KH,HD,page", SHAPES)
@pytest.mark.parametrize("opts", [(1, 2, 5), (0, 1, 0), (3, 1, 1), (0, 3, 40), (2, 100, 3)])
def test_chosen_pages(ctx, H, KH, HD, page, opts):
    rng = np.random.default_rng(H + page)
    lengths = [1, 900, 333, 17]
    pool = Pool(ctx, lengths, KH, HD, page, seed=7, bounds=True)
    seq, pos, rows = [1, 3, 0, 2], [890, 16, 0, 320], [3, 1, 1, 13]
    q = normal(rng, sum(rows), H, HD)
    want, tol, blocks = sparse_ref(pool, seq, pos, rows, q, opts, HD ** -0.5)
    got, taken = pool.attend(seq, pos, rows, q, sparse=opts)
    assert np.array_equal(taken, blocks)
    near(got, want, tol, "sparse")
    assert same(got, pool.attend(seq, pos, rows, q, sparse=opts)[0])
    one, t1 = pool.attend([1], [891], [1], q[1:2], sparse=opts)  # a row's choice and bits do not depend on the others
    assert same(one, got[1:2]) and np.array_equal(t1, taken[1:2])


@pytest.mark.parametrize("page,n,top", [(16, 20000, 100), (16, 70000, 2000), (64, 40000, 7), (16, 140000, 300)])
def test_chosen_pages_of_long_contexts(ctx, page, n, top):
    rng = np.random.default_rng(n)
    H, KH, HD = 4, 1, 64
    pool = Pool(ctx, [n], KH, HD, page, seed=1, bounds=True)
    q = normal(rng, 2, H, HD)
    want, tol, blocks = sparse_ref(pool, [0], [n - 2], [2], q, (1, 2, top), HD ** -0.5)
    got, taken = pool.attend([0], [n - 2], [2], q, sparse=(1, 2, top))
    assert np.array_equal(taken, blocks)
    near(got, want, tol, "sparse")


@pytest.mark.parametrize("n", [400, 5000])
def test_ties_go_to_the_lowest_page(ctx, n):
    """Pages of the same keys, a query of zeros, and bounds with infinities and NaN (first)."""
    H, KH, HD, page = 4, 1, 64, 16
    some = np.random.default_rng(0).standard_normal((page, KH, HD)).astype(np.float16).astype(F32)

    def values(s, k, v):
        for j in range(0, n, page):
            k[j:j + page] = some[:len(k[j:j + page])]
        k[5 * page:6 * page] *= 0.5
        k[9 * page + 2, 0, 7] = np.nan
        k[15 * page + 2, 0, 9] = np.inf
    pool = Pool(ctx, [n], KH, HD, page, bounds=True, values=values)
    q = normal(np.random.default_rng(1), 2, H, HD)
    q[1] = 0
    _, taken = pool.attend([0], [n - 2], [2], q, sparse=(1, 1, 6))
    last = (n - 1) // page
    assert taken[0, 0].tolist() == [0, 1, 2, 3, 4, 9, 15, last] and taken[1, 0].tolist() == [0, 1, 2, 3, 4, 9, 15, last]


def test_missing_pages_are_not_taken(ctx):
    import torch
    rng = np.random.default_rng(2)
    H, KH, HD, page, n = 8, 2, 64, 16, 300
    pool = Pool(ctx, [n], KH, HD, page, bounds=True)
    gone = [2, 3, 7, 11, 17]
    pool.d_table[0, gone] = -1
    torch.cuda.synchronize()
    q = normal(rng, 2, H, HD)
    for opts in ((1, 2, 4), (3, 3, 30)):
        want, tol, blocks = sparse_ref(pool, [0], [n - 2], [2], q, opts, HD ** -0.5, gone)
        got, taken = pool.attend([0], [n - 2], [2], q, sparse=opts)
        assert np.array_equal(taken, blocks)
        near(got, want, tol, opts)


# ------------------------------------------------------------------------------------- together


@pytest.mark.parametrize("prefix", [512, 24576])
def test_a_recorded_step_and_its_replays(ctx, prefix):
    """Store, attention with and without a prefix and the sparse choice, recorded, replayed over other values, with eager calls
    between the replays."""
    import torch
    from windlass_amd.backend import PageRows, SparseOpts
    L, H, KH, HD, page, N = load(), 16, 2, 128, 16, 6
    rng = np.random.default_rng(3)
    lengths = [prefix + 20 + 31 * i for i in range(N)]
    pool = Pool(ctx, lengths, KH, HD, page, shared=prefix, bounds=True)
    r = PageRows(list(range(N)), lengths)
    q, qr, out = (torch.zeros((N, H, HD), device="cuda") for _ in range(3))
    k, v = (torch.zeros((N, KH, HD), device="cuda") for _ in range(2))
    o = {x: torch.zeros_like(q) for x in ("plain", "prefix", "sparse")}
    opts = SparseOpts(1, 2, 9)
    d, rr, h = ctypes.byref(pool.desc), ctypes.byref(r), ctx.handle

    def step():
        check(L.wl_paged_store_dev(h, d, rr, q.data_ptr(), H, k.data_ptr(), v.data_ptr(), HD, 0, 10000.0, 1.0, None,
                                   qr.data_ptr()))
        check(L.wl_paged_attention_dev(h, d, rr, qr.data_ptr(), H, 0, 0.09, o["plain"].data_ptr()))
        check(L.wl_paged_attention_dev(h, d, rr, qr.data_ptr(), H, prefix, 0.09, o["prefix"].data_ptr()))
        check(L.wl_paged_sparse_dev(h, d, rr, qr.data_ptr(), H, ctypes.byref(opts), 0.09, o["sparse"].data_ptr(), None))

    def fill(seed):
        g = np.random.default_rng(seed)
        for t in (q, k, v):
            t.copy_(torch.from_numpy(normal(g, *t.shape)))
        torch.cuda.synchronize()
    fill(0)
    step()
    ctx.sync()
    graph = ctx.capture(step)
    for seed in (1, 2, 3):
        fill(seed)
        step()
        ctx.sync()
        want = {x: t.clone() for x, t in o.items()}
        for t in o.values():
            t.fill_(7.0)
        torch.cuda.synchronize()
        pool.attend([2], [lengths[2] - 300], [300], normal(rng, 300, H, HD))  # other scratch in between
        graph.launch()
        ctx.sync()
        for x, t in o.items():
            assert torch.equal(want[x].view(torch.int32), t.view(torch.int32)), (seed, x)
    graph.free()


def test_other_streams_and_two_contexts(ctx):
    """Two contexts read one pool at once, each with its own scratch."""
    rng = np.random.default_rng(4)
    H, KH, HD, page, n = 16, 2, 128, 64, 6000
    pool = Pool(ctx, [n], KH, HD, page)
    q = [normal(rng, 1, H, HD) for _ in range(2)]
    want = [pool.attend([0], [n - 1], [1], x) for x in q]
    import torch
    from windlass_amd.backend import PageRows
    with Context(0) as other:
        r = PageRows([0], [n - 1])
        dq, out = [pool.dev(x) for x in q], [torch.zeros((1, H, HD), device="cuda") for _ in q]
        torch.cuda.synchronize()
        for _ in range(20):
            for c, a, b in ((ctx, dq[0], out[0]), (other, dq[1], out[1])):
                check(load().wl_paged_attention_dev(c.handle, ctypes.byref(pool.desc), ctypes.byref(r), a.data_ptr(), H, 0,
                                                    HD ** -0.5, b.data_ptr()))
        ctx.sync()
        other.sync()
    assert same(out[0].cpu().numpy(), want[0]) and same(out[1].cpu().numpy(), want[1])


# ------------------------------------------------------------------------------------- large calls


def test_more_rows_than_a_launch_takes(ctx):
    """16,400 rows of 256 heads: two launches, the second of 16 rows."""
    import torch
    H, HD, page, n = 256, 64, 64, 16400
    pool = Pool(ctx, [n], 1, HD, page, seed=2)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((n, H, HD), generator=g, device="cuda")
    out = torch.full_like(q, float("nan"))
    one = torch.full_like(q[:16], float("nan"))
    torch.cuda.synchronize()
    for r, a, o in ((PageRows([0], [0], [n]), q, out), (PageRows([0], [16384], [16]), q[16384:], one)):
        check(load().wl_paged_attention_dev(ctx.handle, ctypes.byref(pool.desc), ctypes.byref(r), a.data_ptr(), H, 0, HD ** -0.5,
                                            o.data_ptr()))
    ctx.sync()
    assert same(out[16384:].cpu().numpy(), one.cpu().numpy())
    for row in (0, 5, 8000, 16383, 16384, 16399):
        want, tol = attend_ref(q[row:row + 1].cpu().numpy(), pool.K[0], pool.V[0], [[np.arange(row + 1)]], HD ** -0.5)
        near(out[row:row + 1].cpu().numpy(), want, tol, "row %d" % row)


def test_reading_more_values_than_a_launch_takes(ctx):
    """2^32 + 2^16 values of keys: positions that all name the same pages."""
    import torch
    KH, HD, page, T = 8, 128, 256, (1 << 22) + 64
    pool = Pool(ctx, [4 * page], KH, HD, page, seed=3)
    width = T // page + 1
    table = torch.from_numpy(np.tile(pool.table[0, :4], width // 4 + 1)[:width].copy()).to("cuda")
    pool.desc.d_table, pool.desc.sequences, pool.desc.table_pages = table.data_ptr(), 1, width
    k, v = (torch.full((T, KH, HD), float("nan"), device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    check(load().wl_paged_read_dev(ctx.handle, ctypes.byref(pool.desc), 0, 0, T, k.data_ptr(), v.data_ptr()))
    ctx.sync()
    for row in (0, 1500, (1 << 21) - 1, 1 << 21, (1 << 21) + 1025, (1 << 22) + 63):
        assert same(k[row].cpu().numpy(), pool.K[0][row % (4 * page)]) and same(v[row].cpu().numpy(), pool.V[0][row % (4 * page)])


def test_chosen_pages_of_many_rows(ctx):
    """Rows of many runs, whose records come a part of the rows at a time."""
    H, KH, HD, page, n, T = 32, 8, 128, 256, 40000, 1100
    pool = Pool(ctx, [n], KH, HD, page, seed=4, bounds=True)
    q = normal(np.random.default_rng(5), T, H, HD)
    opts = (1, 2, 125)
    got, taken = pool.attend([0], [n - T], [T], q, sparse=opts)
    for row in (0, 777, 1000, T - 1):
        one, t1 = pool.attend([0], [n - T + row], [1], q[row:row + 1], sparse=opts)
        assert same(one, got[row:row + 1]) and np.array_equal(t1, taken[row:row + 1])
    want, tol, blocks = sparse_ref(pool, [0], [n - 1], [1], q[T - 1:], opts, HD ** -0.5)
    assert np.array_equal(taken[T - 1:], blocks)
    near(got[T - 1:], want, tol, "the last row")


@pytest.mark.parametrize("H,T", [(8, 3), (8, 60), (240, 60)])
def test_a_query_that_is_not_a_number(ctx, H, T):
    """Gives a row that is not, beside others that are what they were."""
    KH, HD, page, n = 2, 64, 32, 700
    pool = Pool(ctx, [n], KH, HD, page, seed=6, bounds=True)
    q = normal(np.random.default_rng(7), T, H, HD)
    bad = q.copy()
    bad[1, 3, 5] = np.nan
    want, tol = entries_ref(pool, [0], [n - T], [T], q, HD ** -0.5)
    for prefix in (0, 128):
        got = pool.attend([0], [n - T], [T], bad, prefix=prefix)
        assert np.isnan(got[1, 3]).all()
        got[1, 3] = want[1, 3]
        near(got, want, tol, "prefix %d" % prefix)
    want, tol, _ = sparse_ref(pool, [0], [n - T], [T], q, (1, 1, 4), HD ** -0.5)
    got, _ = pool.attend([0], [n - T], [T], bad, sparse=(1, 1, 4))
    assert np.isnan(got[1, 3]).all()
    got[1, :H // KH] = want[1, :H // KH]  # its group's choice may be another
    near(got, want, tol, "sparse")
