"""Recorded layer steps over whole fp16 caches: a replay repeats what was recorded, whatever the program has run since."""
import numpy as np
import pytest
import torch

from test_gpu_long_models import E, Layer, caches, dev, host
from windlass_amd.backend import Context

pytestmark = pytest.mark.gpu
F32 = np.float32


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
