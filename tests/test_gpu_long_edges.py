"""Edges of attention over 4-bit caches and windows. Bounds are long_ref's, or stand at the test."""
import ctypes
import math

import numpy as np
import pytest
import torch

from layer_ref import to_half_ref
from long_ref import attention_span_ref, held_ref
from test_gpu_kv4 import Cache, P, bits, dev, host, rows
from test_gpu_long_models import E, H, KH, Layer, caches, same
from windlass_amd._lib import check, load
from windlass_amd.backend import Context, KvOpts

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def window16(ctx, q, k, v, pos0, window, sinks, scale):
    """wl_attention_window_dev of q [T][H][HD] over k, v [n][KH][HD] (float16)."""
    dq, dk, dv = dev(q), dev(k.view(np.int16)), dev(v.view(np.int16))
    out = torch.full(q.shape, 7.0, device=DEV)
    torch.cuda.synchronize()
    check(load().wl_attention_window_dev(ctx.handle, P(dq), q.shape[0], q.shape[1], k.shape[1], q.shape[2], P(dk), P(dv),
                                         pos0, window, sinks, ctypes.c_float(scale), P(out)))
    return host(ctx, out)


def halves(rng, n, KH, HD):
    return to_half_ref(rows(rng, n, KH, HD)).view(np.float16)


@pytest.mark.parametrize("hidden", [(0, 128), (128, 640), (0, 512), (7, 1000)])
@pytest.mark.parametrize("T,HD,window,sinks", [(1, 64, 0, 0), (1, 128, 0, 0), (5, 128, 0, 0), (15, 64, 0, 0), (16, 128, 0, 0),
                                               (1, 128, 1020, 3), (5, 64, 1000, 40), (20, 64, 1010, 1)])
def test_runs_of_keys_at_minus_infinity(ctx, T, HD, window, sinks, hidden):
    """Keys whose scores are all -inf, a tile or whole runs of them, weigh nothing: the outputs are those of the rows without
    them, and to the bit those of keys so low that their weights are zeros."""
    H, KH, pos0 = 4, 2, 1024
    rng = np.random.default_rng(hidden[1] + T)
    k, v = halves(rng, pos0 + T, KH, HD), halves(rng, pos0 + T, KH, HD)
    q = rng.standard_normal((T, H, HD), dtype=F32)
    q[:, :, 7] = np.abs(q[:, :, 7]) + F32(0.5)
    low = k.copy()
    k[hidden[0]:hidden[1], 0, 7] = -np.inf
    low[hidden[0]:hidden[1], 0, 7] = -60000
    got = window16(ctx, q, k, v, pos0, window, sinks, 0.1)
    assert np.array_equal(bits(got), bits(window16(ctx, q, low, v, pos0, window, sinks, 0.1)))
    # the bound from the finite keys; scores near -3000 with weights of e^-3000 are zeros in 64 bits too
    want, _ = attention_span_ref(q, low, v, pos0 + np.arange(T), window, sinks, 0.1)
    zero = np.where(np.isfinite(k), k, 0)
    _, tol = attention_span_ref(q, zero, v, pos0 + np.arange(T), window, sinks, 0.1)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("T", [1, 3, 20])
def test_a_row_without_a_key_is_nan(ctx, T):
    """Every visible score -inf: 0 / 0, for the heads of that KV head alone."""
    H, KH, HD, pos0 = 4, 2, 64, 900
    rng = np.random.default_rng(T)
    k, v = halves(rng, pos0 + T, KH, HD), halves(rng, pos0 + T, KH, HD)
    k[:, 1, 3] = -np.inf
    q = np.abs(rng.standard_normal((T, H, HD), dtype=F32)) + F32(0.1)
    got = window16(ctx, q, k, v, pos0, 800, 2, 0.1)
    assert np.isnan(got[:, 2:]).all() and np.isfinite(got[:, :2]).all()


@pytest.mark.parametrize("N", [1, 5])
def test_layer_rows_with_keys_at_minus_infinity(ctx, N):
    """Batch rows over fp16 pools with a window: a stretch of keys at -inf is one of keys too low to weigh anything."""
    rng = np.random.default_rng(N)
    HD, cap, slots = 64, 1300, N + 1
    l = Layer(ctx, HD, 32, 0)
    bias = torch.zeros(H * HD, device=DEV)
    bias[HD - 1::HD] = 1000.0  # past the rotated values, and above what the product adds: positive in every head
    torch.cuda.synchronize()
    l.d.d_q_bias = bias.data_ptr()
    K, V = caches(ctx, rng, cap, HD, 16, (slots,))
    K.reshape(slots, cap, KH, HD)[:, 100:800, :, HD - 1] = int(np.float16(-np.inf).view(np.int16))
    low = K.clone()
    low.reshape(slots, cap, KH, HD)[:, 100:800, :, HD - 1] = int(np.float16(-60000).view(np.int16))
    pos = (1100 + 17 * np.arange(N)).astype(np.int32)
    slot = rng.permutation(slots)[:N].astype(np.int32)
    x = dev(rng.standard_normal((N, E), dtype=F32) * F32(0.1))
    y, K2, V2 = x.clone(), low, V.clone()
    torch.cuda.synchronize()
    o = KvOpts(16, 1090, 2, 0)
    for xx, kk, vv in ((x, K, V), (y, K2, V2)):
        check(load().wl_layer_batch_kv_dev(ctx.handle, ctypes.byref(l.d), P(xx), N, pos.ctypes.data, slot.ctypes.data, slots,
                                           cap, P(kk), P(vv), ctypes.byref(o)))
    assert np.isfinite(host(ctx, x)).all() and same(ctx, x, y)
    l.free()


# a scale of zero, and queries so small that the scores' unit is the smallest there is
@pytest.mark.parametrize("scale,qsize", [(0.0, 1.0), (0.1, 1e-35), (-0.1, 1e-37), (0.1, 1e-42)])
@pytest.mark.parametrize("kind", [4, 16])
@pytest.mark.parametrize("T,pos0,H,KH,HD,window,sinks", [(40, 300, 6, 2, 128, 100, 0), (130, 500, 4, 4, 64, 70, 3),
                                                         (70, 10, 8, 1, 128, 33, 5), (1, 900, 4, 2, 64, 700, 4),
                                                         (9, 300, 8, 2, 128, 40, 0), (1, 3000, 8, 1, 64, 0, 0)])
def test_equal_scores(ctx, T, pos0, H, KH, HD, window, sinks, kind, scale, qsize):
    """Scores that differ by nothing: every visible position weighs the same, wherever a row's first one lies in a step."""
    rng = np.random.default_rng(T + pos0)
    n = pos0 + T
    q = rng.standard_normal((T, H, HD)).astype(F32) * F32(qsize)
    if kind == 4:
        k, v = rows(rng, n, KH, HD), rows(rng, n, KH, HD)
        c = Cache(ctx, n, KH, HD)
        c.store(k, v, 0)
        k, v = held_ref(k), held_ref(v)
        dq, out = dev(q), torch.full(q.shape, 7.0, device=DEV)
        torch.cuda.synchronize()
        check(load().wl_kv4_attention_dev(ctx.handle, P(dq), T, H, KH, HD, P(c.K), P(c.V), n, pos0, window, sinks,
                                          ctypes.c_float(scale), P(out)))
        got = host(ctx, out)
    else:
        k, v = halves(rng, n, KH, HD), halves(rng, n, KH, HD)
        got = window16(ctx, q, k, v, pos0, window, sinks, scale)
    want, tol = attention_span_ref(q, k, v, pos0 + np.arange(T), window, sinks, float(F32(scale)))
    err = np.abs(got - want)
    assert (err <= tol).all(), "worst %.3g of its bound" % float((err / tol).max())


@pytest.mark.parametrize("T", [1, 4])
def test_small_queries_beside_a_head_without_a_maximum(ctx, T):
    """Two heads of one KV head, their queries of 1e-35: a first tile of keys at -inf for one of them is at +inf for the other,
    whose output is NaN; the first weighs the other positions the same."""
    H, KH, HD, pos0 = 2, 1, 64, 200
    rng = np.random.default_rng(T)
    k, v = halves(rng, pos0 + T, KH, HD), halves(rng, pos0 + T, KH, HD)
    k[:32, 0, 7] = -np.inf
    q = rng.standard_normal((T, H, HD), dtype=F32)
    q[:, 0, 7], q[:, 1, 7] = F32(1.0), F32(-1.0)
    got = window16(ctx, q * F32(1e-35), k, v, pos0, 0, 0, 0.1)
    assert np.isnan(got[:, 1]).all()
    want = np.stack([v[32:pos0 + t + 1, 0].astype(np.float64).mean(0) for t in range(T)])
    u = 2.0 ** -24
    assert (np.abs(got[:, 0] - want) <= np.abs(v.astype(F32)).max() * (4 * u * math.sqrt(pos0 + T) + 4 * u)).all()
