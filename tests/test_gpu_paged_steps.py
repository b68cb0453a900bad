"""Greedy steps over pages against the slots', one by one, and queries that are not numbers."""
import numpy as np
import pytest

from paged_ref import F32, Pool
from test_gpu_long_models import VOCAB, model
from windlass_amd import DeviceBatch, PagedBatch, SparseOpts
from windlass_amd.backend import Context

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with Context(0) as c:
        yield c


@pytest.mark.parametrize("sparse", [None, SparseOpts(1, 1, 50)])
def test_greedy_steps_are_the_slots(ctx, sparse):
    """Every step's logits and token, up to a sequence's first step whose two largest logits are too near for their order to be
    told: logits are within 2^-9 of the largest (two small layers by another order of sums), so tokens whose margin is four
    times that are the same."""
    rng = np.random.default_rng(3)
    m, w = model(ctx)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (5, 30, 17, 1)]
    N, steps = len(prompts), 6
    a, seen_a = DeviceBatch(m, N, 60).greedy(prompts, steps, keep_logits=True)
    b, seen_b = PagedBatch(m, 16, N, 60, page=16, sparse=sparse).greedy(prompts, steps, keep_logits=True)
    compared = 0
    for i in range(N):
        for s in range(steps + 1):
            x, y = seen_a[s][i], seen_b[s][i]
            most = float(np.abs(x).max())
            assert float(np.abs(x - y).max()) <= 2.0 ** -9 * most, (i, s)
            compared += s > 0  # after a decode step
            top = np.sort(x)[-2:]
            if s == steps or top[1] - top[0] <= 2.0 ** -7 * most:
                break
            assert a[i][s] == b[i][s] == int(np.argmax(x)), (i, s)
    assert compared >= 2 * N
    for x in w.values():
        x.free()


@pytest.mark.parametrize("H,T", [(4, 1), (4, 30), (4096, 30)])
@pytest.mark.parametrize("HD", [64, 128])
def test_queries_of_nan_give_nan(ctx, HD, H, T):
    n = 90
    pool = Pool(ctx, [n], 2, HD, 32, bounds=True)
    q = np.full((T, H, HD), np.nan, F32)
    assert np.isnan(pool.attend([0], [n - T], [T], q)).all()
    assert np.isnan(pool.attend([0], [n - T], [T], q, sparse=(1, 1, 1))[0]).all()
