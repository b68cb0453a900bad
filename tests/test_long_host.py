"""What the host plans for attention over 4-bit caches and windows at the largest positions (no GPU): the scratch a call takes
follows from the tiles its rows read."""
import ctypes

import pytest

from windlass_amd._lib import load


class KvCache(ctypes.Structure):
    _fields_ = [("K", ctypes.c_void_p), ("V", ctypes.c_void_p), ("bits", ctypes.c_int), ("KH", ctypes.c_int),
                ("HD", ctypes.c_int), ("positions", ctypes.c_int64), ("slot_bytes", ctypes.c_int64)]


class Span(ctypes.Structure):
    _fields_ = [("window", ctypes.c_int), ("sinks", ctypes.c_int)]


class KvRows(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int), ("pos0", ctypes.c_int), ("batch", ctypes.c_int), ("pos", ctypes.c_int * 64),
                ("slot", ctypes.c_int * 64)]


def scratch(T, pos0, H, KH, HD, window, sinks):
    """attention_span_scratch_floats of wl_attention_span.h."""
    f = load()._ZN2wl29attention_span_scratch_floatsERKNS_7KvCacheEiRKNS_4SpanERKNS_6KvRowsE
    f.restype = ctypes.c_int64
    c = KvCache(None, None, 4, KH, HD, pos0 + T, 0)
    return f(ctypes.byref(c), H, ctypes.byref(Span(window, sinks)), ctypes.byref(KvRows(T, pos0)))


@pytest.mark.parametrize("T", [1, 15, 16, 40])
@pytest.mark.parametrize("window", [1, 2, 17, 33, 70])
def test_first_tokens_up_to_the_last_position(T, window):
    """First tokens that reach the window are the whole context: the same tiles, and the same runs, as without a window."""
    top = 2**31 - 1 - T
    want = scratch(T, top, 8, 1, 64, 0, 0)
    assert want > 8 * T * 68  # more than one run of a row
    assert scratch(T, top, 8, 1, 64, window, 2**31 - 1) == want
    assert scratch(T, 40, 8, 1, 64, window, 2**31 - 1) == scratch(T, 40, 8, 1, 64, 0, 0)


def test_no_bytes_for_caches_that_no_call_takes():
    f = load().wl_kv4_bytes
    assert f(2**31 - 1, 1 << 18, 64) == 2**26 * 2**18 * 18 * 64 and f(33, 1 << 17, 128) == 2 * 2**17 * 18 * 128
    assert f(1, (1 << 18) + 1, 64) == f(1, (1 << 17) + 1, 128) == f(2**31 - 1, 2**31 - 1, 128) == f(64, 2**31 - 1, 64) == 0
