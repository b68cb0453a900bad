"""wl_sample_dev against a restatement in 64 bits (long_ref.sample_ref).

Tokens are compared exactly. Where the given number or a filter's sum lies nearer to a border between two
tokens than 1e-9 of the weight (double sums of up to 130,000 weights are off by less), the case
says nothing and its number is drawn again before the library is asked."""
import ctypes

import numpy as np
import pytest
import torch

from long_ref import sample_ref
from windlass_amd._lib import ShapeError, check, load
from windlass_amd.backend import Context, SampleParams

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")
NEAR = 1e-9


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def P(t):
    return ctypes.c_void_p(t.data_ptr())


def sample(ctx, logits, u, sets):
    dl = torch.from_numpy(np.ascontiguousarray(logits, F32)).to(DEV)
    du = torch.from_numpy(np.asarray(u, F32)).to(DEV)
    out = torch.full((len(logits),), -7, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    ps = (SampleParams * len(logits))(*[SampleParams(**s) for s in sets])
    check(load().wl_sample_dev(ctx.handle, P(dl), len(logits), logits.shape[1], ps, P(du), P(out)))
    ctx.sync()
    return out.cpu().numpy()


def compare(ctx, logits, rng, sets, us=None):
    want, u = [], []
    for i, s in enumerate(sets):
        for _ in range(20):
            x = F32(rng.random()) if us is None else F32(us[i])
            t, near = sample_ref(logits[i], x, **s)
            if near > NEAR or us is not None:
                break
        want.append(t)
        u.append(x)
    got = sample(ctx, logits, u, sets)
    assert np.array_equal(got, want), [(i, int(g), w, sets[i]) for i, (g, w) in enumerate(zip(got, want)) if g != w][:4]


def peaked(rng, rows, n, bulk=2.0, up=60):
    l = rng.standard_normal((rows, n), dtype=F32) * F32(bulk)
    l[rng.random((rows, n)) < up / n] += F32(8)
    return l


SETS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=40, top_p=0.95, min_p=0.05), dict(top_p=0.9),
        dict(top_k=1), dict(top_k=3), dict(min_p=0.1), dict(min_p=1.0), dict(top_p=0.0), dict(temperature=1.6, top_p=0.999),
        dict(temperature=0.05, top_k=500), dict(temperature=30.0), dict(temperature=30.0, top_p=0.5, top_k=900),
        dict(temperature=1e-6), dict(top_k=10**9, top_p=1.0), dict(temperature=0.3, min_p=1e-3, top_p=0.8)]


@pytest.mark.parametrize("n", [1, 2, 63, 64, 1000, 4095, 4096, 4097, 32003, 128256])
def test_every_setting(ctx, n):
    rng = np.random.default_rng(n)
    compare(ctx, peaked(rng, len(SETS), n), rng, SETS)


def test_the_longest_rows(ctx):
    rng = np.random.default_rng(24)
    compare(ctx, peaked(rng, 2, 1 << 24), rng, [dict(temperature=0.7, top_k=300, top_p=0.95), dict(min_p=0.2)])
    with pytest.raises(ShapeError):
        sample(ctx, np.zeros((1, (1 << 24) + 1), F32), [0.5], [dict()])


@pytest.mark.parametrize("rows", [1, 2, 64, 65, 131])
def test_row_counts(ctx, rows):
    rng = np.random.default_rng(rows)
    compare(ctx, peaked(rng, rows, 5001), rng, [SETS[i % len(SETS)] for i in range(rows)])


@pytest.mark.parametrize("levels", [1, 2, 5, 300])
def test_equal_logits(ctx, levels):
    """Many equal logits: the lower ids first, also past what one pass gathers."""
    rng = np.random.default_rng(levels)
    n = 50001
    l = rng.integers(0, levels, (len(SETS), n)).astype(F32) / F32(max(levels, 1)) - F32(0.3)
    compare(ctx, l, rng, SETS)


def test_borders_of_equal_weights(ctx):
    """Weights that are exact: the number on a border belongs to the next token."""
    n = 8192
    l = np.zeros((6, n), F32)
    us = [0.0, 0.5, 0.25, 1.0 - 2.0**-24, 4095 / 8192, 1 / 8192]
    sets = [dict()] * 3 + [dict()] + [dict(top_p=0.5)] * 2
    # of 8192 equal tokens u picks floor(8192 u); of the first half floor(4096 u)
    got = sample(ctx, l, us, sets)
    assert got.tolist() == [0, 4096, 2048, 8191, 2047, 0]


def test_masked_and_non_finite_logits(ctx):
    rng = np.random.default_rng(0)
    n = 20000
    l = peaked(rng, 12, n)
    l[0, rng.random(n) < 0.99] = -np.inf
    l[1, rng.random(n) < 0.999] = np.finfo(F32).min
    l[2, :] = -np.inf
    l[2, 777] = F32(-3)
    l[3, :] = -np.inf                      # nothing: token 0
    l[4, :] = np.nan
    l[5, rng.random(n) < 0.5] = np.nan
    l[6, [5, 900]] = np.inf                # only these two weigh anything
    l[7] *= F32(1e30)
    l[8] = l[8] * F32(1e-30)
    l[9, :] = np.where(np.arange(n) % 2, F32(0.0), F32(-0.0))
    l[10, 0] = np.nan
    l[11, :] = np.finfo(F32).max
    l[11, 7] = -np.finfo(F32).max
    for s in (dict(), dict(temperature=0.8, top_k=50, top_p=0.9), dict(min_p=0.02), dict(temperature=0.0)):
        compare(ctx, l, rng, [s] * len(l))


@pytest.mark.parametrize("masked", [0.0, 0.5, 0.97])
def test_counts_past_the_bins(ctx, masked):
    """A low temperature leaves most tokens below the bins' reach: top_k ends among them, or among masked ones."""
    rng = np.random.default_rng(int(masked * 100))
    n, ks = 50001, [20, 300, 1400, 5000, 26000, 45000, 50000]
    l = peaked(rng, 3 * len(ks), n)
    l[rng.random(l.shape) < masked] = -np.inf
    l[2::3] = np.rint(l[2::3] * F32(2)) / F32(2)  # many equal
    l[:, 17] = np.finfo(F32).min
    compare(ctx, l, rng, [dict(temperature=t, top_k=k, top_p=p) for k in ks for t, p in [(0.002, 1.0), (0.03, 0.9), (0.3, 0.99)]])


def test_numbers_outside_the_range(ctx):
    l = np.array([[1.0, 5.0, 3.0, 3.0]] * 4, F32)
    got = sample(ctx, l, [-1.0, np.nan, 1.0, np.inf], [dict(top_k=3)] * 4)
    assert got.tolist() == [1, 1, 3, 3]


def test_frequencies(ctx):
    """Numbers evenly over [0, 1): each token as often as its weight says, to within one."""
    rng = np.random.default_rng(11)
    n, N = 37, 4096
    l = rng.standard_normal(n).astype(F32)
    u = ((np.arange(N) + 0.5) / N).astype(F32)
    got = sample(ctx, np.repeat(l[None], N, 0), u, [dict(top_k=20)] * N)
    w = np.exp(l.astype(np.float64) - l.max())
    w[np.argsort(-l, kind="stable")[20:]] = 0
    assert np.abs(np.bincount(got, minlength=n) - N * w / w.sum()).max() <= 1.0


def test_greedy_equals_argmax(ctx):
    rng = np.random.default_rng(12)
    l = np.round(rng.standard_normal((9, 30011)) * 4).astype(F32)
    dl = torch.from_numpy(l).to(DEV)
    out = torch.empty(9, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    check(load().wl_argmax_dev(ctx.handle, P(dl), 9, l.shape[1], P(out)))
    ctx.sync()
    assert np.array_equal(sample(ctx, l, [0.99] * 9, [dict(temperature=0.0)] * 9), out.cpu().numpy())


def test_captured_draws_replay_with_new_numbers(ctx):
    rng = np.random.default_rng(13)
    l = peaked(rng, 3, 40000)
    dl, du = torch.from_numpy(l).to(DEV), torch.zeros(3, device=DEV)
    out = torch.zeros(3, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    sets = [dict(top_p=0.9), dict(temperature=0.8, top_k=40), dict()]
    ps = (SampleParams * 3)(*[SampleParams(**s) for s in sets])
    call = lambda: check(load().wl_sample_dev(ctx.handle, P(dl), 3, l.shape[1], ps, P(du), P(out)))  # noqa: E731
    call()
    ctx.sync()
    g = ctx.capture(call)
    for i in range(4):
        u = rng.random(3).astype(F32)
        du.copy_(torch.from_numpy(u))
        torch.cuda.synchronize()
        call()
        ctx.sync()
        want = out.cpu().numpy().copy()
        out.zero_()
        torch.cuda.synchronize()
        g.launch()
        ctx.sync()
        assert np.array_equal(out.cpu().numpy(), want)
        assert np.array_equal(want, [sample_ref(l[r], u[r], **sets[r])[0] for r in range(3)]), i
    g.free()
