"""Pages chosen by bounds that are infinite: the definition's sum over channels of max(q lo, q hi), where only a score that is
infinite or NaN itself comes before all others."""
import numpy as np
import pytest

from paged_ref import F32, Pool
from windlass_amd.backend import Context

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with Context(0) as c:
        yield c


def blocks_by_maximum(q, b, cur, first, recent, top):
    """The pages a row takes of one KV head: q [G][HD], b [pages][2][HD]."""
    start = min(first, cur + 1)
    end = max(start, cur + 1 - recent)
    q, score = q.astype(np.float64), {}
    with np.errstate(invalid="ignore"):
        for j in range(start, end):
            lo, hi = b[j].astype(np.float64)
            s = np.maximum(q * lo, q * hi).sum(1)  # a NaN of either stays
            score[j] = max(x if np.isfinite(x) else np.inf for x in s)
    pick = sorted(score, key=lambda j: (-score[j], j))[:top]
    return sorted(list(range(start)) + pick + list(range(end, cur + 1)))


# channels by the sign of every head's query, and one whose sign is the head's own
UP, DOWN, MIXED, ZERO = 3, 37, 20, 50


@pytest.mark.parametrize("G,KH,HD", [(1, 2, 64), (3, 2, 64), (8, 1, 128), (11, 3, 128), (16, 1, 64), (40, 2, 128)])
@pytest.mark.parametrize("page,n", [(16, 16 * 40), (64, 64 * 90 + 7)])
def test_infinite_bounds(ctx, G, KH, HD, page, n):
    rng = np.random.default_rng(G * HD + page)
    last = (n - 1) // page
    put = {}  # page: (channel, key), of one position of it, or of all
    for j, (c, key) in enumerate([(UP, -np.inf), (DOWN, np.inf), (UP, np.inf), (DOWN, -np.inf), (MIXED, -np.inf), (MIXED, np.inf),
                                  (ZERO, np.inf), (ZERO, -np.inf)]):
        put[3 + 3 * j] = [(c, key, False)]
    put[28] = [(UP, -np.inf, False), (DOWN, np.inf, False)]  # on the side that no head takes
    put[29] = [(UP, -np.inf, False), (UP, np.inf, False)]
    put[31] = [(UP, -np.inf, True)]  # both bounds: a score of -inf
    put[32] = [(DOWN, np.inf, True)]

    def values(s, k, v):
        k[28 * page:29 * page] *= 2.0  # of large scores by itself; pages 3 and 6 have small ones
        for j in (3, 6):
            k[j * page:(j + 1) * page] *= 0.25
        for j, what in put.items():
            for i, (c, key, every) in enumerate(what):
                k[slice(j * page, (j + 1) * page) if every else j * page + (5 + 3 * i) % page, :, c] = key
    pool = Pool(ctx, [n], KH, HD, page, bounds=True, values=values)
    T = 4
    q = rng.standard_normal((T, KH * G, HD)).astype(F32)
    q[..., UP], q[..., DOWN] = np.abs(q[..., UP]) + F32(0.1), -np.abs(q[..., DOWN]) - F32(0.1)
    q[1:, :, ZERO] = 0.0
    q[2] *= F32(1e-38)  # among them numbers below the normal range
    q[3, :, ZERO] = -0.0
    b = pool.bounds_of(0, last + 1)
    for opts in ((1, 1, 5), (0, 2, 12), (2, 1, 17), (0, 1, 30)):
        _, taken = pool.attend([0], [n - T], [T], q, sparse=opts)
        for t in range(T):
            for g in range(KH):
                want = blocks_by_maximum(q[t, g * G:(g + 1) * G], b[:, g], (n - T + t) // page, *opts)
                want += [-1] * (sum(opts) - len(want))
                assert taken[t, g].tolist() == want, (opts, t, g)


@pytest.mark.parametrize("G,KH,HD", [(1, 1, 64), (8, 2, 128), (18, 1, 64)])
def test_queries_that_are_infinite_or_nan(ctx, G, KH, HD):
    """Of one head of a group, over finite bounds of both signs, of one sign and of zero, and over infinite ones."""
    page, n, T = 16, 16 * 50 + 3, 5

    def values(s, k, v):
        k[5 * page:6 * page, :, 9] = np.abs(k[5 * page:6 * page, :, 9]) + 1  # lo above 0
        k[7 * page:8 * page, :, 9] = 0
        k[11 * page:12 * page, :, 9] = np.minimum(k[11 * page:12 * page, :, 9], 0)
        k[11 * page, :, 9] = 0  # hi of 0
        k[13 * page + 1, :, 9], k[17 * page + 1, :, 9], k[19 * page + 1, :, 30] = np.inf, -np.inf, -np.inf
    pool = Pool(ctx, [n], KH, HD, page, bounds=True, values=values)
    q = np.random.default_rng(HD).standard_normal((T, KH * G, HD)).astype(F32)
    q[0, 0, 9], q[1, 0, 9], q[2, 0, 9] = np.inf, -np.inf, np.nan
    q[3, :, 9], q[3, :, 30] = 3e38, 1e-45  # the largest and smallest numbers
    b = pool.bounds_of(0, (n - 1) // page + 1)
    for opts in ((0, 1, 4), (1, 2, 20)):
        _, taken = pool.attend([0], [n - T], [T], q, sparse=opts)
        for t in range(T):
            for g in range(KH):
                want = blocks_by_maximum(q[t, g * G:(g + 1) * G], b[:, g], (n - T + t) // page, *opts)
                assert taken[t, g].tolist() == want + [-1] * (sum(opts) - len(want)), (opts, t, g)
