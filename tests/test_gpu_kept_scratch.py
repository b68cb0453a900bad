"""Scratch that a context keeps once anything was captured (a graph may name it): growing by half each time, all that was
outgrown is less than two of the last, and the last less than one and a half of what its call needs. So what is kept stays
below 4.5 times that, where buffers of just what each call needs would add up to far more (each test says how much)."""
import ctypes

import numpy as np
import pytest
import torch

from gpu_common import blocks
from test_gpu_long_models import E, KH, Layer, P, dev
from windlass_amd._lib import check, load
from windlass_amd.backend import Context, GgmlType

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")


def test_scratch_of_a_growing_context_stays_small():
    """64 rows of a batch over one KV head, whose runs, and so the scratch, grow to 131,000 positions."""
    H, KH, HD, N, cap, steps = 8, 1, 128, 64, 1 << 17, 40
    with Context(0) as own:
        L, h = load(), own.handle
        K, V = [torch.zeros(N * L.wl_kv4_bytes(cap, KH, HD), dtype=torch.uint8, device=DEV) for _ in range(2)]
        q, out = torch.randn((N, H, HD), device=DEV), torch.empty((N, H, HD), device=DEV)
        torch.cuda.synchronize()
        slot = np.arange(N, dtype=np.int32)

        def at(p):
            pos = np.full(N, p, np.int32)
            check(L.wl_kv4_attention_batch_dev(h, P(q), N, H, KH, HD, P(K), P(V), pos.ctypes.data, slot.ctypes.data, N, cap, 0,
                                               0, 0.1, P(out)))

        def need(p):  # the runs of a row: 16 tiles each past 160 tiles, 256 at most
            tiles = p // 32 + 1
            per = max(16, -(-tiles // 512), -(-tiles // 256))
            return N * H * -(-tiles // per) * (HD + 4) * 4

        at(6000)
        own.sync()
        own.capture(lambda: at(6000)).free()
        before = torch.cuda.mem_get_info()[0]
        where = [6000 + i * (cap - 1 - 6000) // steps for i in range(1, steps + 1)]
        for p in where:
            at(p)
        own.sync()
        bound = 3 * 1.5 * need(where[-1]) + (64 << 20)
        assert sum(sorted({need(p) for p in where})) > 1.5 * bound  # one call's growth at a time
        assert before - torch.cuda.mem_get_info()[0] < bound


def test_large_kept_scratch_stays_small():
    """Prompts' operands of 256 MB to 3.5 GB, 256 MB more at a time."""
    rows_, cols, unit = 32, 256, 1 << 19  # 2 bytes a value: unit rows of x are 256 MB
    with Context(0) as own:
        L, h = load(), own.handle
        w = own.upload(GgmlType.Q4_K, blocks(GgmlType.Q4_K, rows_, cols, seed=1), rows_, cols)
        x, y = torch.zeros((14 * unit, cols), device=DEV), torch.empty((14 * unit, rows_), device=DEV)
        torch.cuda.synchronize()

        def run(T):
            check(L.wl_matmul_dev(h, w.handle, -1, P(x), T, P(y)))

        run(unit)
        own.sync()
        own.capture(lambda: run(unit)).free()
        before = torch.cuda.mem_get_info()[0]
        for i in range(2, 15):
            run(i * unit)
        own.sync()
        taken = before - torch.cuda.mem_get_info()[0]
        bound = 3 * 1.5 * 14 * unit * cols * 2
        assert sum(i * unit * cols * 2 for i in range(2, 15)) > 1.5 * bound
        assert 14 * unit * cols * 2 - (1 << 30) <= taken < bound, (taken, bound)
        w.free()


def test_kept_rope_tables_stay_small():
    """Angles of 64 pairs, 1 KB a position, to 131,000 positions, 4,096 more at a time: no recording names their table."""
    cap, step = 1 << 17, 4096
    with Context(0) as own:
        l = Layer(own, 64, 64, 0)
        K, V = [torch.zeros((cap, KH * 64), dtype=torch.int16, device=DEV) for _ in range(2)]
        x = dev(np.ones((1, E), F32))

        def at(p):
            check(load().wl_layer_dev(own.handle, ctypes.byref(l.d), P(x), 1, p, P(K), P(V)))

        at(0)
        own.sync()
        own.capture(lambda: at(0)).free()
        before = torch.cuda.mem_get_info()[0]
        for p in range(step, cap, step):
            at(p)
        own.sync()
        bound = 3 * 1.5 * cap * 1024 + (64 << 20)  # attention's scratch: 512 chunks of one row
        assert sum(range(2 * step, cap + 1, step)) * 1024 > 3 * bound
        assert before - torch.cuda.mem_get_info()[0] < bound
        l.free()
