"""The KV cache in 4 bits (wl_kv4_store_dev, _batch_dev, wl_kv4_read_dev), the attention that reads it
(wl_kv4_attention_dev, _batch_dev) and attention over fp16 caches with a window
(wl_attention_window_dev), against restatements in 64 bits (long_ref.py).

What the cache holds is compared bit for bit. Attention's bound is long_ref's: what rounding in 32
bits may be off, from the sizes of the scores and values."""
import ctypes
import math

import numpy as np
import pytest
import torch

from layer_ref import to_half_ref
from long_ref import attention_span_ref, held_ref
from windlass_amd._lib import check, load
from windlass_amd.backend import Context

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def P(t):
    return ctypes.c_void_p(t.data_ptr())


def dev(a):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    return t


def host(ctx, t):
    ctx.sync()
    return t.cpu().numpy()


class Cache:
    """4-bit caches of `slots` sequences, filled with a pattern that reads as NaN until rows are stored."""

    def __init__(self, ctx, positions, KH, HD, slots=1):
        self.ctx, self.n, self.KH, self.HD = ctx, positions, KH, HD
        b = load().wl_kv4_bytes(positions, KH, HD)
        assert b == KH * -(-positions // 32) * 18 * HD
        self.K = torch.full((slots, b), 0xff, dtype=torch.uint8, device=DEV)
        self.V = torch.full((slots, b), 0xff, dtype=torch.uint8, device=DEV)
        torch.cuda.synchronize()

    def store(self, k, v, pos0, slot=0):
        dk, dv = dev(k), dev(v)
        check(load().wl_kv4_store_dev(self.ctx.handle, P(dk), P(dv), len(k), self.KH, self.HD, P(self.K[slot]),
                                      P(self.V[slot]), self.n, pos0))
        self.ctx.sync()

    def read(self, pos0, T, slot=0):
        out = [torch.full((T, self.KH, self.HD), 7.0, device=DEV) for _ in range(2)]
        torch.cuda.synchronize()
        check(load().wl_kv4_read_dev(self.ctx.handle, P(self.K[slot]), P(self.V[slot]), self.n, self.KH, self.HD, pos0, T,
                                     P(out[0]), P(out[1])))
        return [host(self.ctx, t) for t in out]

    def attention(self, q, pos0, window=0, sinks=0, scale=None, slot=0):
        dq = dev(q)
        out = torch.full(q.shape, 7.0, device=DEV)
        torch.cuda.synchronize()
        check(load().wl_kv4_attention_dev(self.ctx.handle, P(dq), q.shape[0], q.shape[1], self.KH, self.HD,
                                          P(self.K[slot]), P(self.V[slot]), self.n, pos0, window, sinks,
                                          scale or 1 / math.sqrt(self.HD), P(out)))
        return host(self.ctx, out)


def rows(rng, n, KH, HD):
    x = rng.standard_normal((n, KH, HD), dtype=F32)
    x[:, rng.random((KH, HD)) < 0.03] *= F32(6)
    return x


def bits(a):
    return np.ascontiguousarray(a, F32).view(np.uint32)


@pytest.mark.parametrize("KH,HD", [(1, 64), (3, 64), (8, 128), (5, 128)])
@pytest.mark.parametrize("T,pos0,positions", [(1, 0, 1), (1, 31, 33), (70, 0, 70), (37, 29, 66), (33, 95, 200)])
def test_store_holds_the_nearest_values(ctx, KH, HD, T, pos0, positions):
    rng = np.random.default_rng(T * HD + KH)
    k, v = rows(rng, T, KH, HD), rows(rng, T, KH, HD)
    c = Cache(ctx, positions, KH, HD)
    c.store(k, v, pos0)
    gk, gv = c.read(pos0, T)
    assert np.array_equal(gk, held_ref(k)) and np.array_equal(gv, held_ref(v))


def test_blocks_of_every_size_and_kind(ctx):
    KH, HD = 2, 64
    rng = np.random.default_rng(5)
    r = []
    for e in range(-40, 18):  # largest values from below the smallest scale to past the largest
        r.append(rng.standard_normal((KH, HD)).astype(F32) * F32(2.0 ** e))
    x = np.stack(r)
    x[3, 0, :32] = 0                                  # a block of zeros
    x[4, 0, :32] = F32(-0.0)
    x[5, 0, :32] = F32(1.25)                          # equal values
    x[6, 0, :32] = np.where(np.arange(32) % 2, 3, -3)  # equal magnitudes: the first one's sign
    x[7, 0, :32] = np.where(np.arange(32) < 17, 0, np.where(np.arange(32) % 2, 5, -5))
    x[8, 0, :32] = np.arange(32) - 15.5               # ties of the rounding
    x[9, 0, :32] = (np.arange(32) - 16) / 2
    x[10, 1, 32:] = 1e30                              # past the largest scale
    x[11, 1, 32:] = np.linspace(-21760, 21760, 32)
    x[12, 0, 5] = np.inf
    x[13, 1, 40] = np.nan
    x[14, 1, 63] = -np.inf
    x[15, 0, :32] = F32(1e-45)
    c = Cache(ctx, len(x), KH, HD)
    c.store(x, x[::-1], 0)
    gk, gv = c.read(0, len(x))
    assert np.array_equal(gk, held_ref(x), equal_nan=True)
    assert np.array_equal(gv, held_ref(x[::-1]), equal_nan=True)
    assert np.isnan(gk[12, 0, :32]).all() and np.isfinite(gk[12, 0, 32:]).all()


def test_store_leaves_other_positions_as_they_were(ctx):
    KH, HD, n = 2, 128, 100
    rng = np.random.default_rng(9)
    c = Cache(ctx, n, KH, HD)
    k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
    c.store(k, v, 0)
    before = c.read(0, n)
    k2, v2 = rows(rng, 7, KH, HD), rows(rng, 7, KH, HD)
    c.store(k2, v2, 61)
    after = c.read(0, n)
    for b, a, new in zip(before, after, (k2, v2)):
        assert np.array_equal(a[:61], b[:61]) and np.array_equal(a[68:], b[68:]) and np.array_equal(a[61:68], held_ref(new))
    raw = c.K.cpu().clone()
    c.store(k2[:0], v2[:0], 61)  # no rows
    assert torch.equal(raw, c.K.cpu())


def test_batch_store_equals_single_stores(ctx):
    KH, HD, slots, cap, N = 2, 64, 90, 70, 81  # more rows than one launch takes
    rng = np.random.default_rng(2)
    one, many = Cache(ctx, cap, KH, HD, slots), Cache(ctx, cap, KH, HD, slots)
    k, v = rows(rng, N, KH, HD), rows(rng, N, KH, HD)
    slot = rng.permutation(slots)[:N].astype(np.int32)
    pos = rng.integers(0, cap, N).astype(np.int32)
    dk, dv = dev(k), dev(v)
    check(load().wl_kv4_store_batch_dev(ctx.handle, P(dk), P(dv), N, KH, HD, P(many.K), P(many.V),
                                        pos.ctypes.data, slot.ctypes.data, slots, cap))
    for i in range(N):
        one.store(k[i:i + 1], v[i:i + 1], int(pos[i]), int(slot[i]))
    ctx.sync()
    assert torch.equal(one.K, many.K) and torch.equal(one.V, many.V)


# rows of one call, positions before them; head counts from one per KV head to more than a wave's columns
SHAPES = [(8, 2, 64), (8, 8, 128), (28, 4, 128), (64, 8, 128), (20, 1, 64), (5, 1, 128)]


def kv4_case(ctx, rng, T, pos0, H, KH, HD, window, sinks, qscale=2.0):
    n = pos0 + T
    c = Cache(ctx, n + 5, KH, HD)  # positions past the last are never written
    k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
    c.store(k, v, 0)
    q = rng.standard_normal((T, H, HD), dtype=F32) * F32(qscale)
    got = c.attention(q, pos0, window, sinks)
    want, tol = attention_span_ref(q, held_ref(k), held_ref(v), pos0 + np.arange(T), window, sinks, 1 / math.sqrt(HD))
    err = np.abs(got - want)
    assert (err <= tol).all(), "worst %.3g of its bound" % float((err / tol).max())


@pytest.mark.parametrize("H,KH,HD", SHAPES)
@pytest.mark.parametrize("T,pos0", [(1, 0), (1, 1), (1, 31), (1, 32), (1, 700), (2, 0), (7, 333), (15, 64)])
def test_kv4_attention_few_rows(ctx, H, KH, HD, T, pos0):
    kv4_case(ctx, np.random.default_rng(T + pos0 + H), T, pos0, H, KH, HD, 0, 0)


@pytest.mark.parametrize("H,KH,HD", [(8, 2, 64), (14, 2, 128), (3, 3, 128), (24, 1, 64)])
@pytest.mark.parametrize("T,pos0", [(16, 0), (17, 3), (64, 0), (65, 100), (130, 31), (33, 900)])
def test_kv4_attention_prompts(ctx, H, KH, HD, T, pos0):
    kv4_case(ctx, np.random.default_rng(T + pos0 + H), T, pos0, H, KH, HD, 0, 0)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (32, 0), (33, 4), (64, 64), (100, 33), (5000, 7),
                                          (40, 5000), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("T,pos0,H,KH,HD", [(1, 0, 4, 2, 64), (1, 500, 8, 1, 128), (9, 180, 4, 4, 64), (50, 0, 4, 2, 64),
                                            (40, 300, 6, 2, 128)])
def test_kv4_attention_window(ctx, T, pos0, H, KH, HD, window, sinks):
    kv4_case(ctx, np.random.default_rng(T + pos0), T, pos0, H, KH, HD, window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_kv4_attention_long_row(ctx, window, sinks):
    kv4_case(ctx, np.random.default_rng(8), 1, 9000, 8, 1, 128, window, sinks)
    kv4_case(ctx, np.random.default_rng(9), 1, 2200, 16, 8, 64, window, sinks)


@pytest.mark.parametrize("T", [1, 20])
@pytest.mark.parametrize("slots", [1, 3])
def test_offsets_past_32_bits(ctx, slots, T):
    """Caches of 4.6 GB each, whose last slot's window and first positions are compared with a short cache's."""
    H, KH, HD, n, last = 16, 8, 128, 8 * 10**6 // slots, 60
    rng = np.random.default_rng(T)
    c = Cache(ctx, n, KH, HD, slots)
    k, v = rows(rng, 3 + last, KH, HD), rows(rng, 3 + last, KH, HD)
    q = rng.standard_normal((T, H, HD), dtype=F32)
    c.store(k[:3], v[:3], 0, slots - 1)
    c.store(k[3:], v[3:], n - last, slots - 1)
    gk, gv = c.read(n - last, last, slots - 1)
    assert np.array_equal(gk, held_ref(k[3:])) and np.array_equal(gv, held_ref(v[3:]))
    got = c.attention(q, n - T, 30, 3, slot=slots - 1)
    want, tol = attention_span_ref(q, held_ref(k), held_ref(v), 3 + last - T + np.arange(T), 30, 3, 1 / math.sqrt(HD))
    assert (np.abs(got - want) <= tol).all()
    if T == 1:
        dq, out, pos, slot = dev(q), torch.empty((1, H, HD), device=DEV), np.array([n - 1], np.int32), np.array([slots - 1], np.int32)
        check(load().wl_kv4_attention_batch_dev(ctx.handle, P(dq), 1, H, KH, HD, P(c.K), P(c.V), pos.ctypes.data,
                                                slot.ctypes.data, slots, n, 30, 3, 1 / math.sqrt(HD), P(out)))
        assert np.array_equal(bits(host(ctx, out)), bits(got))


@pytest.mark.parametrize("T", [1, 20])
def test_fp16_offsets_past_32_bits(ctx, T):
    H, KH, HD, n, last = 16, 8, 128, 22 * 10**5, 60  # 4.5 GB each
    rng = np.random.default_rng(T)
    k, v = to_half_ref(rows(rng, 3 + last, KH, HD)), to_half_ref(rows(rng, 3 + last, KH, HD))
    K, V = [torch.full((n, KH * HD), 0x7e00, dtype=torch.int16, device=DEV) for _ in range(2)]
    for t, x in ((K, k), (V, v)):
        x = torch.from_numpy(x.view(np.int16).reshape(3 + last, -1)).to(DEV)
        t[:3], t[n - last:] = x[:3], x[3:]
    q = rng.standard_normal((T, H, HD), dtype=F32)
    dq, out = dev(q), torch.empty((T, H, HD), device=DEV)
    check(load().wl_attention_window_dev(ctx.handle, P(dq), T, H, KH, HD, P(K), P(V), n - T, 30, 3, 1 / math.sqrt(HD),
                                         P(out)))
    want, tol = attention_span_ref(q, k.view(np.float16), v.view(np.float16), 3 + last - T + np.arange(T), 30, 3,
                                   1 / math.sqrt(HD))
    assert (np.abs(host(ctx, out) - want) <= tol).all()


def fp16_case(ctx, rng, T, pos0, H, KH, HD, window, sinks):
    n = pos0 + T
    k, v = to_half_ref(rows(rng, n, KH, HD)), to_half_ref(rows(rng, n, KH, HD))
    pad = np.full((3, KH, HD), 0x7e00, np.uint16)  # positions past the last hold NaN
    dk, dv = dev(np.concatenate([k, pad]).view(np.int16)), dev(np.concatenate([v, pad]).view(np.int16))
    q = rng.standard_normal((T, H, HD), dtype=F32) * F32(2)
    dq, out = dev(q), torch.full(q.shape, 7.0, device=DEV)
    torch.cuda.synchronize()
    check(load().wl_attention_window_dev(ctx.handle, P(dq), T, H, KH, HD, P(dk), P(dv), pos0, window, sinks,
                                         1 / math.sqrt(HD), P(out)))
    got = host(ctx, out)
    want, tol = attention_span_ref(q, k.view(np.float16), v.view(np.float16), pos0 + np.arange(T), window, sinks,
                                   1 / math.sqrt(HD))
    err = np.abs(got - want)
    assert (err <= tol).all(), "worst %.3g of its bound" % float((err / tol).max())


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 3), (33, 4), (100, 33), (40, 5000)])
@pytest.mark.parametrize("T,pos0,H,KH,HD", [(1, 0, 4, 2, 64), (1, 500, 8, 1, 128), (1, 3000, 4, 4, 128), (9, 180, 4, 4, 64),
                                            (50, 0, 4, 2, 64), (40, 300, 6, 2, 128), (130, 90, 20, 1, 128),
                                            (3, 70, 4, 2, 80), (20, 50, 3, 1, 5)])
def test_window_attention_fp16(ctx, T, pos0, H, KH, HD, window, sinks):
    fp16_case(ctx, np.random.default_rng(T + pos0), T, pos0, H, KH, HD, window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
@pytest.mark.parametrize("H,KH,HD", [(8, 2, 64), (16, 2, 128), (3, 3, 64)])
def test_batch_rows_equal_single_rows_bitwise(ctx, H, KH, HD, window, sinks):
    slots, cap, N = 75, 400, 70
    rng = np.random.default_rng(H)
    c = Cache(ctx, cap, KH, HD, slots)
    slot = rng.permutation(slots)[:N].astype(np.int32)
    pos = np.concatenate([[0, 31, 32, cap - 1], rng.integers(0, cap, N - 4)]).astype(np.int32)
    for i in range(N):
        c.store(rows(rng, pos[i] + 1, KH, HD), rows(rng, pos[i] + 1, KH, HD), 0, int(slot[i]))
    q = rng.standard_normal((N, H, HD), dtype=F32)
    dq, out = dev(q), torch.full(q.shape, 7.0, device=DEV)
    torch.cuda.synchronize()
    check(load().wl_kv4_attention_batch_dev(ctx.handle, P(dq), N, H, KH, HD, P(c.K), P(c.V), pos.ctypes.data,
                                            slot.ctypes.data, slots, cap, window, sinks, 1 / math.sqrt(HD), P(out)))
    got = host(ctx, out)
    for i in range(N):
        one = c.attention(q[i:i + 1], int(pos[i]), window, sinks, slot=int(slot[i]))
        assert np.array_equal(bits(got[i]), bits(one[0])), i


def test_few_rows_equal_single_rows_bitwise(ctx):
    rng = np.random.default_rng(3)
    for T, pos0, H, KH, HD, window in [(8, 500, 8, 2, 128, 0), (15, 1200, 4, 4, 64, 0), (5, 300, 8, 1, 64, 90)]:
        c = Cache(ctx, pos0 + T, KH, HD)
        c.store(rows(rng, pos0 + T, KH, HD), rows(rng, pos0 + T, KH, HD), 0)
        q = rng.standard_normal((T, H, HD), dtype=F32)
        got = c.attention(q, pos0, window, 4)
        for t in range(T):
            assert np.array_equal(bits(got[t]), bits(c.attention(q[t:t + 1], pos0 + t, window, 4)[0])), (T, t)


@pytest.mark.parametrize("T,pos0", [(1, 400), (1, 5000), (40, 200)])
def test_a_nan_block_reaches_only_the_rows_that_see_it(ctx, T, pos0):
    H, KH, HD, window, sinks = 4, 2, 64, 60, 3
    n = pos0 + T
    rng = np.random.default_rng(1)
    k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
    q = rng.standard_normal((T, H, HD), dtype=F32)
    clean = Cache(ctx, n, KH, HD)
    clean.store(k, v, 0)
    want = clean.attention(q, pos0, window, sinks)
    for what in "kv":
        # a position just before the first row's window, one no row sees, and one the later rows do not
        for at in (pos0 - window, pos0 // 2, pos0 - window + 5):
            x, y = k.copy(), v.copy()
            (x if what == "k" else y)[at, 0, 3] = np.inf
            c = Cache(ctx, n, KH, HD)
            c.store(x, y, 0)
            got = c.attention(q, pos0, window, sinks)
            for t in range(T):
                sees = at < sinks or pos0 + t - window < at <= pos0 + t
                for h in range(H):
                    if sees and h < H // KH:
                        assert np.isnan(got[t, h, :32]).all()
                        assert what == "v" or np.isnan(got[t, h]).all()
                    else:
                        assert np.array_equal(bits(got[t, h]), bits(want[t, h])), (what, at, t, h)


@pytest.mark.parametrize("scale", [1e-3, 0.5, -0.3, 40.0])
def test_scales_and_large_scores(ctx, scale):
    rng = np.random.default_rng(6)
    for T, pos0 in [(1, 300), (20, 100)]:
        KH, H, HD, n = 1, 4, 64, pos0 + T
        c = Cache(ctx, n, KH, HD)
        k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
        c.store(k, v, 0)
        q = rng.standard_normal((T, H, HD), dtype=F32)
        q[:, 1] *= F32(1e4)
        q[:, 2] *= F32(1e-20)
        q[:, 3] = 0
        got = c.attention(q, pos0, 0, 0, scale)
        want, tol = attention_span_ref(q, held_ref(k), held_ref(v), pos0 + np.arange(T), 0, 0, float(F32(scale)))
        assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("T", [1, 3, 30])
def test_scores_past_2_to_the_26(ctx, T):
    """Scores whose units in the last place are whole powers of e: the largest key's weight is 1 all the same."""
    KH, H, HD, pos0 = 2, 4, 64, 200
    n = pos0 + T
    rng = np.random.default_rng(T)
    k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
    q = rng.standard_normal((T, H, HD), dtype=F32) * F32(1e9)
    c = Cache(ctx, n, KH, HD)
    c.store(k, v, 0)
    got = c.attention(q, pos0)
    K, V = held_ref(k).astype(np.float64), held_ref(v)
    for t in range(T):
        for h in range(H):
            s = K[:pos0 + t + 1, h // 2] @ q[t, h].astype(np.float64) / 8
            best = np.argsort(s)[-2:]
            assert s[best[1]] - s[best[0]] > 1e4  # nothing else weighs anything
            assert np.array_equal(got[t, h], V[best[1], h // 2])


@pytest.mark.parametrize("T,pos0,HD", [(1, 300, 64), (1, 5000, 128), (5, 90, 128), (40, 200, 64), (33, 100, 128)])
def test_fp16_infinities_and_nans(ctx, T, pos0, HD):
    """In masked places they change no bit; a visible one reaches the rows that see it, and there its own column (a
    value) or, as a score of -inf, none."""
    H, KH, window, sinks = 4, 2, 60, 3
    n, G = pos0 + T, 2
    rng = np.random.default_rng(pos0)
    k, v = (to_half_ref(rows(rng, n, KH, HD)).view(np.float16) for _ in range(2))
    k[:, 0, 7] = np.abs(k[:, 0, 7])
    q = rng.standard_normal((T, H, HD), dtype=F32)
    q[:, :, 7] = np.abs(q[:, :, 7]) + F32(0.5)
    dq = dev(q)

    def run(x, y):
        dk, dv, out = dev(x.view(np.int16)), dev(y.view(np.int16)), torch.full(q.shape, 7.0, device=DEV)
        torch.cuda.synchronize()
        check(load().wl_attention_window_dev(ctx.handle, P(dq), T, H, KH, HD, P(dk), P(dv), pos0, window, sinks,
                                             1 / math.sqrt(HD), P(out)))
        return host(ctx, out)

    want = run(k, v)
    for what, bad in (("v", np.inf), ("v", np.nan), ("k", -np.inf), ("k", np.nan)):
        for at in (1, pos0 - window, pos0 // 2, pos0 - window + 7, pos0):
            x, y = k.copy(), v.copy()
            (x if what == "k" else y)[at, 0, 7] = bad
            got = run(x, y)
            less, tol = attention_span_ref(q, np.where(np.isfinite(x), x, 0), np.where(np.isfinite(y), y, 0),
                                           pos0 + np.arange(T), window, sinks, 1 / math.sqrt(HD))
            for t in range(T):
                sees = at <= pos0 + t and (at < sinks or at > pos0 + t - window)
                for h in range(H):
                    if not sees or h >= G:
                        assert np.array_equal(bits(got[t, h]), bits(want[t, h])), (what, bad, at, t, h)
                    elif what == "v":
                        rest = np.arange(HD) != 7
                        assert np.array_equal(bits(got[t, h][rest]), bits(want[t, h][rest]))
                        assert np.isnan(got[t, h, 7]) if np.isnan(bad) else got[t, h, 7] == np.inf
                    elif np.isnan(bad):
                        assert np.isnan(got[t, h]).all()
                    else:  # the key weighs nothing: the rows without it
                        m = [j for j in range(pos0 + t + 1) if j != at and (j < sinks or j > pos0 + t - window)]
                        s = k[m, 0].astype(np.float64) @ q[t, h] / math.sqrt(HD)
                        p = np.exp(s - s.max())
                        ref = (p / p.sum()) @ v[m, 0].astype(np.float64)
                        assert (np.abs(got[t, h] - ref) <= tol[t, h]).all()


def test_many_rows_of_another_head_dim(ctx):
    """Scores of more than one launch's scratch."""
    T, pos0, H, KH, HD = 3000, 3000, 4, 1, 8
    n = pos0 + T
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn((n, KH, HD), device=DEV, generator=g).half() for _ in range(2))
    q, out = torch.randn((T, H, HD), device=DEV, generator=g), torch.empty((T, H, HD), device=DEV)
    torch.cuda.synchronize()
    check(load().wl_attention_window_dev(ctx.handle, P(q), T, H, KH, HD, P(k), P(v), pos0, 0, 0, 0.3, P(out)))
    ctx.sync()
    K, V = k[:, 0].double(), v[:, 0].double()
    at = torch.arange(n, device=DEV)
    for h in range(H):
        s = torch.mm(q[:, h].double(), K.t().contiguous()) * 0.3
        s.masked_fill_(at > pos0 + torch.arange(T, device=DEV)[:, None], -math.inf)
        want = torch.mm(torch.softmax(s, 1), V)
        # long_ref's bound, with scores of at most 8 * 4.5^2 * 0.3 in size and values of at most 4.5
        assert float((out[:, h] - want).abs().max()) <= 4.5 * (8 * 2.0**-24 * 8**0.5 * 49 + 4 * 2.0**-24 * n**0.5)


def test_a_graph_outlives_its_scratch(ctx):
    """A later, larger call makes the context take larger scratch; the graph's own stays with it."""
    H, KH, HD, n = 64, 8, 128, 40000
    rng = np.random.default_rng(8)
    with Context(0) as own:
        c = Cache(own, n, KH, HD)
        k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
        c.store(k, v, 0)
        q, out = dev(rng.standard_normal((1, H, HD), dtype=F32)), torch.zeros((1, H, HD), device=DEV)
        logits, u, tok = dev(rng.standard_normal((2, 30000), dtype=F32)), dev(np.array([0.3, 0.8], F32)), dev(np.zeros(2, np.int32))
        from windlass_amd.backend import SampleParams
        ps = (SampleParams * 70)(*[SampleParams(1.0, 0, 0.9, 0.0)] * 70)
        L, h = load(), own.handle

        def step():
            check(L.wl_kv4_attention_dev(h, P(q), 1, H, KH, HD, P(c.K), P(c.V), n, 2000, 0, 0, 0.1, P(out)))
            check(L.wl_sample_dev(h, P(logits), 2, 30000, ps, P(u), P(tok)))

        step()
        own.sync()
        g = own.capture(step)
        big, many = torch.empty((15, H, HD), device=DEV).normal_(), torch.randn((70, 128000), device=DEV)
        bo, bu, bt = torch.empty_like(big), torch.rand(70, device=DEV), torch.zeros(70, dtype=torch.int32, device=DEV)
        for i in range(3):
            q.normal_()
            torch.cuda.synchronize()
            step()
            want = [host(own, t).copy() for t in (out, tok)]
            check(L.wl_kv4_attention_dev(h, P(big), 15, H, KH, HD, P(c.K), P(c.V), n, n - 15, 0, 0, 0.1, P(bo)))
            check(L.wl_sample_dev(h, P(many), 70, 128000, ps, P(bu), P(bt)))
            own.sync()
            junk = [torch.full((1 << 22,), float("nan"), device=DEV) for _ in range(20)]  # where freed scratch would be
            out.zero_()
            tok.zero_()
            torch.cuda.synchronize()
            g.launch()
            assert np.array_equal(bits(host(own, out)), bits(want[0])) and np.array_equal(host(own, tok), want[1]), i
            del junk
        g.free()


def test_kept_scratch_stays_small():
    """Once anything was captured, scratch that a longer context outgrows is kept: all of it stays below three times the
    last's 130 MB and half as much again (one call's growth at a time would keep 40 sizes, 2.6 GB)."""
    H, KH, HD, n, T = 64, 8, 128, 1 << 17, 15
    with Context(0) as own:
        L, h = load(), own.handle
        K, V = [torch.zeros(L.wl_kv4_bytes(n, KH, HD), dtype=torch.uint8, device=DEV) for _ in range(2)]
        q, out = torch.randn((T, H, HD), device=DEV), torch.empty((T, H, HD), device=DEV)
        torch.cuda.synchronize()

        def at(pos):
            check(L.wl_kv4_attention_dev(h, P(q), T, H, KH, HD, P(K), P(V), n, pos, 0, 0, 0.1, P(out)))

        at(1000)
        own.sync()
        own.capture(lambda: at(1000)).free()
        before = torch.cuda.mem_get_info()[0]
        for i in range(1, 41):
            at(i * (n - T) // 40)
        own.sync()
        last = T * H * 256 * (HD + 4) * 4
        assert before - torch.cuda.mem_get_info()[0] < 3 * 1.5 * last + (64 << 20)


def test_captured_calls_replay(ctx):
    """A step's store, attention over both caches and the draw, captured and replayed between eager work."""
    H, KH, HD, n = 8, 2, 128, 1500
    rng = np.random.default_rng(4)
    c = Cache(ctx, n, KH, HD)
    k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
    c.store(k, v, 0)
    h16 = dev(to_half_ref(k).view(np.int16))
    kn, vn, q = dev(k[-1:]), dev(v[-1:]), dev(rng.standard_normal((1, H, HD), dtype=F32))
    o4, o16 = torch.empty((1, H, HD), device=DEV), torch.empty((1, H, HD), device=DEV)
    L, h, sc = load(), ctx.handle, 1 / math.sqrt(HD)

    def step():
        check(L.wl_kv4_store_dev(h, P(kn), P(vn), 1, KH, HD, P(c.K), P(c.V), n, n - 1))
        check(L.wl_kv4_attention_dev(h, P(q), 1, H, KH, HD, P(c.K), P(c.V), n, n - 1, 0, 0, sc, P(o4)))
        check(L.wl_attention_window_dev(h, P(q), 1, H, KH, HD, P(h16), P(h16), n - 1, 700, 4, sc, P(o16)))

    step()
    ctx.sync()
    g = ctx.capture(step)
    for i in range(4):
        kn.copy_(torch.randn_like(kn))
        q.copy_(torch.randn_like(q))
        torch.cuda.synchronize()
        step()
        want = [bits(host(ctx, t)) for t in (o4, o16)]
        o4.zero_()
        o16.zero_()
        torch.cuda.synchronize()
        g.launch()
        assert all(np.array_equal(bits(host(ctx, t)), w) for t, w in zip((o4, o16), want)), i
    g.free()
