"""Layers and models over caches in pages: wl_layer_paged_dev against its operations and against the fp16 slots' layers, and a
small model's PagedBatch against DeviceBatch."""
import ctypes

import numpy as np
import pytest
import torch

from paged_ref import attend_ref
from test_gpu_long_models import BASE, DEV, E, EPS, FF, H, KH, VOCAB, Layer, P, dev, host, model, same
from windlass_amd import DeviceBatch, PagedBatch, SampleParams
from windlass_amd._lib import ArgumentOutOfRangeError, NotSupportedError, ShapeError, check, load
from windlass_amd.backend import Context, PageRows, Pages, SparseOpts

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


class PagedLayer(Layer):
    def pool(self, rng, lengths, page=16, room=300):
        """A pool of NaN, `lengths` positions of each sequence stored, with bounds."""
        HD, N = self.HD, len(lengths)
        width = (max(lengths) + room + page - 1) // page
        pages = N * width + 2
        self.t = [torch.full((pages * KH * page * HD,), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2)]
        self.t.append(torch.full((pages * KH * 2 * HD,), float("nan"), dtype=torch.float16, device=DEV))
        self.t.append(dev(rng.permutation(pages)[:N * width].reshape(N, width).astype(np.int32)))
        self.p = Pages(*(x.data_ptr() for x in self.t), pages, page, KH, HD, N, width)
        k, v = (dev(rng.standard_normal((sum(lengths), KH, HD), dtype=F32)) for _ in range(2))
        r = PageRows(list(range(N)), [0] * N, lengths)
        check(load().wl_paged_store_dev(self.ctx.handle, ctypes.byref(self.p), ctypes.byref(r), None, 0, P(k), P(v), 0, 0,
                                        1.0, 1.0, None, None))
        self.ctx.sync()

    def state(self):
        return [x.clone() for x in self.t]

    def paged(self, x, seq, pos, rows=None, prefix=0, sparse=None):
        check(load().wl_layer_paged_dev(self.ctx.handle, ctypes.byref(self.d), P(x), ctypes.byref(self.p),
                                        ctypes.byref(PageRows(seq, pos, rows)), prefix,
                                        ctypes.byref(SparseOpts(*sparse)) if sparse else None))

    def paged_operations(self, x, seq, pos, rows=None, prefix=0, sparse=None):
        """The layer one operation at a time; 8 rows at most."""
        L, h, c, HD, T = load(), self.ctx.handle, ctypes.c_float, self.HD, x.shape[0]
        QD, KD = H * HD, KH * HD
        xn, g = (torch.empty((T, n), device=DEV) for n in (E, FF))
        q, k, v, qr, att = (torch.empty((T, n), device=DEV) for n in (QD, KD, KD, QD, QD))
        r, p = PageRows(seq, pos, rows), ctypes.byref(self.p)
        check(L.wl_rms_norm_dev(h, P(x), T, E, P(self.norms[0]), c(EPS), P(xn)))
        ws = (ctypes.c_void_p * 3)(*(self.w[n].handle.value for n in ("attn_q", "attn_k", "attn_v")))
        check(L.wl_matmul_multi_dev(h, 3, ws, P(xn), T, (ctypes.c_void_p * 3)(*(t.data_ptr() for t in (q, k, v)))))
        check(L.wl_paged_store_dev(h, p, ctypes.byref(r), P(q), H, P(k), P(v), self.rd, self.neox, BASE, 0.5, P(self.freqs),
                                   P(qr)))
        if sparse:
            check(L.wl_paged_sparse_dev(h, p, ctypes.byref(r), P(qr), H, ctypes.byref(SparseOpts(*sparse)), c(0.1), P(att),
                                        None))
        else:
            check(L.wl_paged_attention_dev(h, p, ctypes.byref(r), P(qr), H, prefix, c(0.1), P(att)))
        check(L.wl_matmul_add_dev(h, self.w["attn_output"].handle, -1, P(att), T, P(x), c(0.5)))
        check(L.wl_rms_norm_dev(h, P(x), T, E, P(self.norms[1]), c(EPS), P(xn)))
        check(L.wl_gate_up_dev(h, self.w["ffn_gate"].handle, self.w["ffn_up"].handle, -1, P(xn), T, P(g)))
        check(L.wl_matmul_add_dev(h, self.w["ffn_down"].handle, -1, P(g), T, P(x), c(0.5)))
        self.ctx.sync()


@pytest.mark.parametrize("HD,rd,neox", [(64, 32, 1), (128, 128, 0)])
@pytest.mark.parametrize("seq,pos,rows,prefix,sparse", [
    ([2, 0, 1], [90, 100, 41], None, 0, None), ([1, 2], [60, 90], [3, 5], 0, None), ([0, 1], [100, 200], None, 0, (1, 2, 3)),
    ([2, 1], [90, 60], [2, 4], 0, (0, 1, 2)), ([1], [60], [8], 0, None), ([1], [64], [1], 48, None)])
def test_layer_equals_its_operations(ctx, HD, rd, neox, seq, pos, rows, prefix, sparse):
    rng = np.random.default_rng(HD + len(seq))
    l = PagedLayer(ctx, HD, rd, neox)
    l.pool(rng, [100, 200, 90])
    T = sum(rows) if rows else len(seq)
    x = dev(rng.standard_normal((T, E), dtype=F32))
    xb, was = x.clone(), l.state()
    torch.cuda.synchronize()
    l.paged(x, seq, pos, rows, prefix, sparse)
    ctx.sync()
    now = l.state()
    for a, b in zip(l.t, was):
        a.copy_(b)
    torch.cuda.synchronize()
    l.paged_operations(xb, seq, pos, rows, prefix, sparse)
    assert same(ctx, x, xb) and all(same(ctx, a, b) for a, b in zip(l.t, now))
    assert np.isfinite(host(ctx, x)).all() and not same(ctx, now[0], was[0])
    l.free()


@pytest.mark.parametrize("seq,pos,rows,prefix,sparse", [
    ([2, 0, 1], [90, 100, 41], None, 0, None), ([0, 1], [100, 200], None, 0, (1, 2, 3)), ([1, 2], [60, 90], [3, 40], 48, None)])
def test_a_recorded_layer_reads_the_table_as_it_is(ctx, seq, pos, rows, prefix, sparse):
    """Replays over other rows and after pages have moved, with eager calls between."""
    rng = np.random.default_rng(11)
    l = PagedLayer(ctx, 64, 64, 1)
    l.pool(rng, [100, 200, 90])
    if prefix:
        l.t[3][2, :3] = l.t[3][1, :3]
        torch.cuda.synchronize()
    T = sum(rows) if rows else len(seq)
    x = torch.zeros((T, E), device=DEV)
    r, o = PageRows(seq, pos, rows), SparseOpts(*sparse) if sparse else None

    def step():
        check(load().wl_layer_paged_dev(ctx.handle, ctypes.byref(l.d), P(x), ctypes.byref(l.p), ctypes.byref(r), prefix,
                                        ctypes.byref(o) if o else None))
    step()
    ctx.sync()
    graph = ctx.capture(step)
    free = sorted(set(range(l.p.pages)) - set(l.t[3].cpu().numpy().reshape(-1).tolist()))[0]
    for i in range(3):
        new = dev(rng.standard_normal((T, E), dtype=F32))
        # the page before the last entry's own goes to a free place
        j = pos[-1] // 16 - 1
        old = int(l.t[3][seq[-1], j])
        for t, n in ((l.t[0], KH * 16 * 64), (l.t[1], KH * 16 * 64), (l.t[2], KH * 2 * 64)):
            t[free * n:free * n + n] = t[old * n:old * n + n]
            t[old * n:old * n + n] = 3.0
        torch.cuda.synchronize()
        check(load().wl_paged_assign_dev(ctx.handle, ctypes.byref(l.p), seq[-1], j, 1, (ctypes.c_int32 * 1)(free)))
        ctx.sync()
        free = old
        was = l.state()
        x.copy_(new)
        torch.cuda.synchronize()
        step()
        ctx.sync()
        want, now = x.clone(), l.state()
        for a, b in zip(l.t, was):
            a.copy_(b)
        x.copy_(new)
        torch.cuda.synchronize()
        graph.launch()
        ctx.sync()
        assert same(ctx, x, want) and all(same(ctx, a, b) for a, b in zip(l.t, now)), i
    graph.free()
    l.free()


@pytest.mark.parametrize("N", [1, 5, 70, 140])
@pytest.mark.parametrize("sparse", [None, (1, 1, 3)])
def test_batch_rows_equal_single_tokens(ctx, N, sparse):
    rng = np.random.default_rng(N)
    l = PagedLayer(ctx, 64, 64, 0)
    lengths = [int(n) for n in rng.integers(1, 200, N + 2)]
    l.pool(rng, lengths, room=20)
    seq = [int(s) for s in rng.permutation(N + 2)[:N]]
    pos = [lengths[s] for s in seq]
    x = dev(rng.standard_normal((N, E), dtype=F32))
    xb, was = x.clone(), l.state()
    torch.cuda.synchronize()
    l.paged(x, seq, pos, None, 0, sparse)
    ctx.sync()
    now = l.state()
    for a, b in zip(l.t, was):
        a.copy_(b)
    torch.cuda.synchronize()
    for i in range(N):
        l.paged(xb[i:i + 1], seq[i:i + 1], pos[i:i + 1], None, 0, sparse)
    assert same(ctx, x, xb) and all(same(ctx, a, b) for a, b in zip(l.t, now))
    l.free()


def test_prompts_and_steps_in_one_call_are_near_their_own(ctx):
    """Rows of several prompts as one prompt's: against the fp16 slots' layer, within what the products' other tiles and the
    attention's other order change: its outputs' fp32 roundings, and operands that round to the other side in bf16 (2^-9 each,
    of sums of which x's residual is the largest part)."""
    rng = np.random.default_rng(6)
    l = PagedLayer(ctx, 64, 64, 0)
    l.pool(rng, [0, 0, 0])
    rows = [40, 9, 100]
    x = dev(rng.standard_normal((149, E), dtype=F32))
    xb = x.clone()
    torch.cuda.synchronize()
    l.paged(x, [2, 0, 1], [0, 0, 0], rows)
    at = 0
    for t in rows:
        K, V = (torch.zeros((t, KH * 64), dtype=torch.int16, device=DEV) for _ in range(2))
        torch.cuda.synchronize()
        check(load().wl_layer_dev(ctx.handle, ctypes.byref(l.d), P(xb[at:at + t]), t, 0, P(K), P(V)))
        ctx.sync()
        at += t
    a, b = host(ctx, x), host(ctx, xb)
    assert np.abs(a - b).max() <= 2.0 ** -8 * np.abs(b).max()
    l.free()


# ------------------------------------------------------------------------------------- models


def logits_near(a, b, what):
    """Logits of one sequence by two orders of the attention's sums (fp32 roundings, through two small layers)."""
    off, most = float(np.abs(a - b).max()), float(np.abs(b).max())
    assert off <= 2.0 ** -9 * most, (what, off, most)


def test_steps_equal_a_sequence_alone(ctx):
    rng = np.random.default_rng(0)
    m, w = model(ctx)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (3, 40, 17)]
    params = [SampleParams(0.9, 50, 0.95, 0.02), SampleParams(1.3), SampleParams(0.0)]
    u = rng.random((12, 3)).astype(F32)
    got = PagedBatch(m, 12, 4, 80, page=16).generate(prompts, 12, params, u)
    for i, p in enumerate(prompts):
        one = PagedBatch(m, 6, 1, 80, page=16)
        assert one.generate([p], 12, params[i:i + 1], u[:, i:i + 1]) == got[i:i + 1]
    for x in w.values():
        x.free()


@pytest.mark.parametrize("sparse", [None, SparseOpts(1, 1, 50)])
def test_logits_are_near_the_slots(ctx, sparse):
    """Pages, a shared beginning and a choice of every page give the slots' logits, but for the order of sums."""
    rng = np.random.default_rng(1)
    m, w = model(ctx)
    beginning = rng.integers(0, VOCAB, 50).tolist()
    prompts = [beginning + rng.integers(0, VOCAB, n).tolist() for n in (3, 20, 1)]
    want = DeviceBatch(m, 3, 120)
    got = PagedBatch(m, 20, 3, 120, page=16, sparse=sparse)
    a = [host(ctx, want.prefill(i, p)) for i, p in enumerate(prompts)]
    b = [host(ctx, got.prefill(0, prompts[0]))]
    for i in (1, 2):
        got.share(0, i, 48)
        b.append(host(ctx, got.prefill(i, prompts[i][48:])))
    for i in range(3):
        logits_near(b[i], a[i], i)
    ids = dev(np.array([5, 6, 7], np.int32))
    for s in range(3):
        x, y = host(ctx, got.step([0, 1, 2], ids)), host(ctx, want.step([0, 1, 2], ids))
        logits_near(x, y, s)
    assert got.length == want.length and got._shared([0, 1, 2]) == 48 and got._shared([1]) == 0
    for x in w.values():
        x.free()


def test_generate_with_a_shared_beginning(ctx):
    rng = np.random.default_rng(2)
    m, w = model(ctx)
    beginning = rng.integers(0, VOCAB, 70).tolist()
    prompts = [beginning + rng.integers(0, VOCAB, n).tolist() for n in (3, 0, 9)]
    params, u = [SampleParams(0.0)] * 3, np.full((6, 3), 0.5, F32)
    b = PagedBatch(m, 4 + 3 * 2, 3, 100, page=16)
    got = b.generate(prompts, 6, params, u, shared=70)
    assert b._shared([0, 1, 2]) == 64 and len(b.free_pages) == 2  # four pages once; 14, 11 and 20 positions more
    # greedy tokens from the same steps one at a time
    one = PagedBatch(m, 30, 3, 100, page=16)
    one.prefill(0, beginning[:64])
    for i in (1, 2):
        one.share(0, i, 64)
    lg = [host(ctx, one.prefill(i, p[64:]))[0] for i, p in enumerate(prompts)]
    ids = [int(np.argmax(x)) for x in lg]
    for t in range(6):
        assert ids == [g[t] for g in got], t
        if t < 5:
            ids = [int(np.argmax(x)) for x in host(ctx, one.step([0, 1, 2], dev(np.array(ids, np.int32))))]
    for i in range(3):
        b.release(i)
    assert len(b.free_pages) == 10 and not any(b.users) and b.generate(prompts, 6, params, u, shared=70) == got
    for x in w.values():
        x.free()


def test_greedy_is_the_slots(ctx):
    rng = np.random.default_rng(3)
    m, w = model(ctx)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (5, 30)]
    a, seen_a = DeviceBatch(m, 2, 60).greedy(prompts, 5, keep_logits=True)
    b, seen_b = PagedBatch(m, 8, 2, 60, page=16).greedy(prompts, 5, keep_logits=True)
    logits_near(seen_b[0], seen_a[0], "prompts")
    top = np.sort(seen_a[0], 1)
    if (top[:, -1] - top[:, -2]).min() > 2.0 ** -7 * np.abs(seen_a[0]).max():
        assert [x[0] for x in a] == [x[0] for x in b]
    for x in w.values():
        x.free()
