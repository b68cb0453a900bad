"""What the 4-bit cache's, the window's and the sampler's entries refuse, before anything is launched (no GPU:
the context is never touched by a refused call)."""
import ctypes

import pytest

from windlass_amd._lib import WL_E_ARG, WL_E_SHAPE, WL_E_UNSUPPORTED, load
from windlass_amd.backend import SampleParams

CTX = ctypes.create_string_buffer(1 << 14)  # stands for a context: refusals come before its first use
BUF = (ctypes.c_char * 256)()
X = ctypes.c_void_p((ctypes.addressof(BUF) + 63) // 64 * 64)
ODD = ctypes.c_void_p(X.value + 8)


def ints(*v):
    return (ctypes.c_int32 * len(v))(*v)


def store(ctx=CTX, k=X, v=X, T=1, KH=2, HD=64, K=X, V=X, positions=10, pos0=0):
    return load().wl_kv4_store_dev(ctx, k, v, T, KH, HD, K, V, positions, pos0)


def read(ctx=CTX, K=X, V=X, positions=10, KH=2, HD=64, pos0=0, T=1, k=X, v=X):
    return load().wl_kv4_read_dev(ctx, K, V, positions, KH, HD, pos0, T, k, v)


def attend(ctx=CTX, q=X, T=1, H=4, KH=2, HD=64, K=X, V=X, positions=10, pos0=0, window=0, sinks=0, out=X):
    return load().wl_kv4_attention_dev(ctx, q, T, H, KH, HD, K, V, positions, pos0, window, sinks, 1.0, out)


def window(ctx=CTX, q=X, T=1, H=4, KH=2, HD=64, K=X, V=X, pos0=0, window=0, sinks=0, out=X):
    return load().wl_attention_window_dev(ctx, q, T, H, KH, HD, K, V, pos0, window, sinks, 1.0, out)


def batch(ctx=CTX, q=X, N=2, H=4, KH=2, HD=64, K=X, V=X, pos=ints(3, 4), slot=ints(0, 1), slots=3, cap=10, window=0,
          sinks=0, out=X):
    return load().wl_kv4_attention_batch_dev(ctx, q, N, H, KH, HD, K, V, pos, slot, slots, cap, window, sinks, 1.0, out)


def batch_store(ctx=CTX, k=X, v=X, N=2, KH=2, HD=64, K=X, V=X, pos=ints(3, 4), slot=ints(0, 1), slots=3, cap=10):
    return load().wl_kv4_store_batch_dev(ctx, k, v, N, KH, HD, K, V, pos, slot, slots, cap)


def sample(ctx=CTX, logits=X, rows=1, n=10, params=None, u=X, out=X, **kw):
    params = (SampleParams * 1)(SampleParams(**kw)) if params is None else params
    return load().wl_sample_dev(ctx, logits, rows, n, params, u, out)


def test_sizes():
    f = load().wl_kv4_bytes
    assert f(1, 1, 64) == 18 * 64 and f(33, 8, 128) == 2 * 8 * 18 * 128
    assert f(2**31 - 1, 8, 128) == 2**26 * 8 * 18 * 128  # past 32 bits
    assert [f(0, 1, 64), f(-5, 1, 64), f(32, 0, 64), f(32, 1, 96), f(32, 1, 256)] == [0] * 5


@pytest.mark.parametrize("call,names", [(store, "ctx k v K V"), (read, "ctx k v K V"), (attend, "ctx q K V out"),
                                        (window, "ctx q K V out"), (batch, "ctx q K V pos slot out"),
                                        (batch_store, "ctx k v K V pos slot"), (sample, "ctx logits u out")])
def test_null_arguments(call, names):
    for n in names.split():
        assert call(**{n: ctypes.c_void_p()}) == WL_E_ARG, n


@pytest.mark.parametrize("call", [store, read, attend, batch, batch_store])
def test_cache_shapes(call):
    for hd in (32, 80, 96, 192, 256):
        assert call(HD=hd) == WL_E_UNSUPPORTED
    for kw in (dict(HD=0), dict(HD=-64), dict(KH=0), dict(KH=-1), dict(KH=2**30)):
        if call in (attend, batch) and "KH" in kw:
            kw["H"] = 2**30
        assert call(**kw) in (WL_E_SHAPE, WL_E_UNSUPPORTED), kw
    assert call(K=ODD) == WL_E_ARG and call(V=ODD) == WL_E_ARG


@pytest.mark.parametrize("call", [store, read, attend])
def test_rows_outside_the_cache(call):
    assert call(T=-1) == WL_E_SHAPE and call(pos0=-1) == WL_E_SHAPE and call(positions=0) == WL_E_SHAPE
    assert call(T=11) == WL_E_ARG and call(T=1, pos0=10) == WL_E_ARG
    assert call(T=2**31 - 1, pos0=2**31 - 1, positions=2**31 - 1) == WL_E_ARG  # the sum passes 32 bits


def test_window_rows():
    assert window(T=-1) == WL_E_SHAPE and window(pos0=-1) == WL_E_SHAPE and window(HD=0) == WL_E_SHAPE
    assert window(T=2, pos0=2**31 - 2) == WL_E_ARG


@pytest.mark.parametrize("call", [attend, window, batch])
def test_heads_and_spans(call):
    assert call(H=5) == WL_E_SHAPE and call(H=0) == WL_E_SHAPE and call(H=-4) == WL_E_SHAPE
    assert call(window=-1) == WL_E_ARG and call(sinks=-1) == WL_E_ARG


@pytest.mark.parametrize("call", [batch, batch_store])
def test_batch_rows(call):
    assert call(N=-1) == WL_E_SHAPE and call(slots=0) == WL_E_SHAPE and call(cap=0) == WL_E_SHAPE
    for kw in (dict(slot=ints(0, 3)), dict(slot=ints(-1, 0)), dict(slot=ints(1, 1)), dict(pos=ints(10, 0)),
               dict(pos=ints(0, -1))):
        assert call(**kw) == WL_E_ARG, kw


def test_sampling_settings():
    nan = float("nan")
    assert sample(rows=-1) == WL_E_SHAPE and sample(n=0) == WL_E_SHAPE and sample(n=2**24 + 1) == WL_E_SHAPE
    for kw in (dict(temperature=-0.5), dict(temperature=nan), dict(temperature=float("inf")), dict(top_k=-1),
               dict(top_p=-0.1), dict(top_p=1.5), dict(top_p=nan), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=nan)):
        assert sample(**kw) == WL_E_ARG, kw
    assert load().wl_sample_dev(CTX, X, 1, 10, None, X, X) == WL_E_ARG
