"""Calls of more rows than a launch takes are cut at entries: a row's bits do not depend on the entries beside its own."""
import ctypes

import pytest

from paged_ref import Pool
from windlass_amd._lib import check, load
from windlass_amd.backend import Context, PageRows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with Context(0) as c:
        yield c


@pytest.mark.parametrize("H,KH,rows", [(256, 1, [10, 16380, 30, 0, 5]), (96, 2, [7, 1, 43685, 50])])
def test_rows_past_a_launch_have_their_own_calls_bits(ctx, H, KH, rows):
    """2^22 (row, head) pairs are a launch's: 16,384 rows of 256 heads, 43,690 of 96."""
    import torch
    HD, page, most = 64, 64, (1 << 22) // H
    assert sum(rows) > most > max(rows)
    seq = list(range(len(rows)))
    pos = [3 * i for i in range(len(rows))]
    pool = Pool(ctx, [max(p + t, 1) for p, t in zip(pos, rows)], KH, HD, page, seed=2)
    q = torch.randn((sum(rows), H, HD), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    out, one = (torch.full_like(q, float("nan")) for _ in range(2))
    torch.cuda.synchronize()

    def attend(r, a, o):
        check(load().wl_paged_attention_dev(ctx.handle, ctypes.byref(pool.desc), ctypes.byref(r), a.data_ptr(), H, 0, HD ** -0.5,
                                            o.data_ptr()))
    attend(PageRows(seq, pos, rows), q, out)
    at = 0
    for s, p, t in zip(seq, pos, rows):
        if t:
            attend(PageRows([s], [p], [t]), q[at:], one[at:])
        at += t
    ctx.sync()
    at = 0
    for s, t in zip(seq, rows):
        a, b = out[at:at + t].view(torch.int32), one[at:at + t].view(torch.int32)
        assert torch.equal(a, b), (s, int((a != b).any(2).any(1).sum()), t)
        at += t
