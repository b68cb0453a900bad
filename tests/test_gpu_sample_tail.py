"""Draws from the tails of long rows of logits (wl_sample_dev), against 64-bit sums."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import P, dev, host
from windlass_amd._lib import check, load
from windlass_amd.backend import Context, SampleParams

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


TAIL = [(1 << 24, 20.0, 2.0, 1.0), (1 << 24, 30.0, 2.0, 1.3), (1 << 22, 25.0, 3.0, 1.0), (1 << 20, 18.0, 2.0, 1.0),
        (128256, 16.0, 2.0, 1.0), (1 << 18, 16.0, 2.0, 1.0), ((1 << 18) + 1, 16.0, 2.0, 1.0), (3 << 17, 1e30, 2.0, 1.0), (1 << 24, 0.0, 1.0, 5.0), (40000, 300.0, 1.0, 20.0)]


@pytest.mark.parametrize("n,peak,sigma,t", TAIL)
def test_draws_from_the_tail(ctx, n, peak, sigma, t):
    """One logit far above a bulk whose tokens weigh next to nothing each, and together much more than the numbers' unit. The
    drawn token lies where the exact sum passes u of the weight, to within what cutting n weights to the row's unit may take: n
    2^-52; up to 2^18 logits n 2^(bits - 63); past them n 2^-49 of the weight (n units, each 2^-62 of a bound on the weight at
    most, which is 1.01 times 4,096 times it at most). And what the reference's own sums of n take, n 2^-53 of the weight, and
    the weights' last places."""
    t = float(F32(t))
    rng = np.random.default_rng(n)
    l = rng.standard_normal(n).astype(F32) * F32(sigma)
    l[n // 3] = F32(peak)
    order = np.argsort(-l, kind="stable")
    w = np.exp((l[order].astype(np.float64) - float(l[order[0]])) / t)
    c = np.cumsum(w)
    rank = np.empty(n, np.int64)
    rank[order] = np.arange(n)
    head = 1.0 / c[-1]
    us = np.array([0.0, 0.5, head + (1 - head) * 0.01, head + (1 - head) * 0.3, head + (1 - head) * 0.8, 1 - 2.0 ** -24,
                   1 - 2.0 ** -22, 1 - 2.0 ** -20], F32)
    us = us[us < 1]
    dl, du = dev(l), dev(us)
    out = torch.full((len(us),), -7, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    ps = (SampleParams * 1)(SampleParams(t))
    for i in range(len(us)):
        check(load().wl_sample_dev(ctx.handle, P(dl), 1, n, ps, P(du[i:]), P(out[i:])))
    got = host(ctx, out)
    cut = n * 2.0 ** ((n - 1).bit_length() - 63) if n <= 1 << 18 else n * 2.0 ** -49 * c[-1]
    near = n * 2.0 ** -52 + cut + (n * 2.0 ** -53 + 2.0 ** -40) * c[-1]
    for u, g in zip(us.astype(np.float64), got):
        r = rank[g]
        x = u * c[-1]
        assert c[r] > x - near and c[r] - w[r] <= x + near, (u, r, (c[r] - x) / c[-1])
