"""Paged calls that store, where host memory has run out: an error code, as for any other shortage (no GPU: the call is refused
before it touches its context)."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import ctypes, resource
import numpy as np
from windlass_amd._lib import load
from windlass_amd.backend import LayerDesc, PageRows, Pages
L = load()
ctx, buf = ctypes.create_string_buffer(1 << 14), ctypes.create_string_buffer(256)
x = (ctypes.addressof(buf) + 63) // 64 * 64
p = Pages(x, x, None, x, 9, 16, 2, 64, 4, 5)
r = PageRows([0], [0])
zeros = np.zeros(1 << 25, np.int32)  # as many entries without rows
r.n = zeros.size
r.seq = r.pos = r.rows = zeros.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
d = LayerDesc(heads=4, kv_heads=2, head_dim=64)
now = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (now + (32 << 20),) * 2)
a = L.wl_paged_store_dev(ctx, ctypes.byref(p), ctypes.byref(r), None, 0, None, None, 0, 0, 1.0, 1.0, None, None)
b = L.wl_layer_paged_dev(ctx, ctypes.byref(d), x, ctypes.byref(p), ctypes.byref(r), 0, None)
print(a, b, L.wl_last_error().decode())
"""


def test_no_host_memory_for_the_entries():
    from windlass_amd._lib import WL_E_NOMEM
    r = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    a, b, what = r.stdout.split(None, 2)
    assert int(a) == int(b) == WL_E_NOMEM and "entries" in what
