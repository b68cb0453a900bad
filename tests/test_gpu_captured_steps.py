"""Recorded layer steps over whole fp16 caches: a replay repeats what was recorded (its angles; its tokens, positions and slots),
whatever the program has run since."""
import ctypes

import numpy as np
import pytest
import torch

from gpu_common import blocks
from test_gpu_long_models import E, Layer, P, caches, dev, host
from windlass_amd._lib import check, load
from windlass_amd.backend import Context, GgmlType, KvOpts

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")
VOCAB = 700


@pytest.mark.parametrize("before", [True, False])
def test_a_recorded_step_keeps_its_angles(before):
    """Layers of two RoPE bases, one of them recorded (with or without its own call at that position first), replayed between
    calls of the other at the same position, which take their angles from the same table."""
    with Context(0) as ctx:
        rng = np.random.default_rng(0)
        K0, V0 = caches(ctx, rng, 50, 64, 16)
        x0 = dev(rng.standard_normal((1, E), dtype=F32))
        a, b = Layer(ctx, 64, 64, 0), Layer(ctx, 64, 64, 0)
        b.d.rope_base = 500.0
        x, K, V = x0.clone(), K0.clone(), V0.clone()

        def fresh():
            for t, t0 in ((x, x0), (K, K0), (V, V0)):
                t.copy_(t0)
            torch.cuda.synchronize()

        def step(l, pos=7):
            l.run(x, 1, pos, K, V, 50, 16, 0, 0)

        def eager(l, pos=7):
            fresh()
            step(l, pos)
            return [host(ctx, t).copy().view(np.uint8) for t in (x, K, V)]

        with Context(0) as other:  # the outputs, from a context of their own
            own = Layer(other, 64, 64, 0), Layer(other, 64, 64, 0)
            own[1].d.rope_base = 500.0
            want = []
            for l in own:
                fresh()
                l.run(x, 1, 7, K, V, 50, 16, 0, 0)
                want.append([host(other, t).copy().view(np.uint8) for t in (x, K, V)])
        assert not np.array_equal(want[0][1], want[1][1])  # the stored keys
        eager(a, 7 if before else 9)
        fresh()
        g = ctx.capture(lambda: step(a))
        for rep in range(3):
            assert all(np.array_equal(p, q) for p, q in zip(eager(b), want[1])), rep
            fresh()
            g.launch()
            assert all(np.array_equal(host(ctx, t).view(np.uint8), q) for t, q in zip((x, K, V), want[0])), rep
            assert all(np.array_equal(p, q) for p, q in zip(eager(a if rep % 2 else b), want[0 if rep % 2 else 1])), rep
        g.free()


class Step:
    """Tokens, positions and slots of N rows; run() embeds the tokens and takes them through a layer."""

    def __init__(self, ctx, seed, N, entry):
        rng = np.random.default_rng(seed)
        self.ctx, self.N, self.entry, self.cap, self.slots = ctx, N, entry, 90, N + 2
        self.l = Layer(ctx, 64, 64, 0)
        self.embd = ctx.upload(GgmlType.Q8_0, blocks(GgmlType.Q8_0, VOCAB, E, seed=1), VOCAB, E)
        self.tokens = (ctypes.c_int32 * N)(*rng.integers(0, VOCAB, N))
        self.pos = (ctypes.c_int32 * N)(*rng.integers(0, self.cap, N))
        self.slot = (ctypes.c_int32 * N)(*rng.permutation(self.slots)[:N])
        self.K0, self.V0 = caches(ctx, rng, self.cap, 64, 16, (self.slots,))
        self.K, self.V, self.x = self.K0.clone(), self.V0.clone(), torch.empty((N, E), device=DEV)

    def run(self):
        L, h, d, o = load(), self.ctx.handle, ctypes.byref(self.l.d), KvOpts(16, 0, 0, 0)
        check(L.wl_embed_dev(h, self.embd.handle, self.tokens, self.N, P(self.x)))
        a = (h, d, P(self.x), self.N, self.pos, self.slot, self.slots, self.cap, P(self.K), P(self.V))
        check(L.wl_layer_batch_kv_dev(*a, ctypes.byref(o)) if self.entry == "kv" else L.wl_layer_batch_dev(*a))

    def reset(self):
        self.K.copy_(self.K0)
        self.V.copy_(self.V0)
        self.x.fill_(float("nan"))
        torch.cuda.synchronize()

    def outputs(self):
        return [host(self.ctx, t).copy().view(np.uint8) for t in (self.x, self.K, self.V)]


@pytest.mark.parametrize("entry", ["kv", "plain"])
@pytest.mark.parametrize("N", [1, 5, 150])
def test_recorded_batch_steps_repeat_their_rows(N, entry):
    with Context(0) as ctx:
        a, other = Step(ctx, N, N, entry), Step(ctx, N + 1, N, entry)
        wants = []
        for s in (a, other):
            s.reset()
            s.run()
            wants.append(s.outputs())
        assert np.isfinite(wants[0][0].view(F32)).all()
        a.reset()
        g = ctx.capture(a.run)
        tokens = list(a.tokens)
        for arr in (a.tokens, a.pos, a.slot):  # the recording holds their values
            ctypes.memset(arr, 0x7f, ctypes.sizeof(arr))
        for rep in range(4):
            for _ in range(rep + 1):
                other.reset()
                other.run()
                assert all(np.array_equal(x, y) for x, y in zip(other.outputs(), wants[1]))
            a.reset()
            g.launch()
            assert all(np.array_equal(x, y) for x, y in zip(a.outputs(), wants[0])), (rep, tokens[:4])
        g.free()
