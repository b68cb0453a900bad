"""KV caches in pages for the tests: a pool whose unwritten places hold NaN, its sequences, and plain restatements in 64 bits
of the rotation, the bounds, the choice of pages and attention."""
import ctypes

import numpy as np

from windlass_amd._lib import check, load
from windlass_amd.backend import PageRows, Pages, SparseOpts

F32, U = np.float32, 2.0 ** -24


def key_at(off, d, HD):
    return off // 16 * 16 * HD + off // 4 % 2 * 8 * HD + d // 8 * 64 + (off // 8 % 2 * 4 + off % 4) * 8 + d % 8


def val_at(off, d, HD):
    return off // 8 * 8 * HD + d * 8 + off % 8


def attend_ref(q, K, V, sees, scale):
    """Rows q [T][H][HD] over K, V [n][KH][HD] in 64 bits; sees[t][kvh]: the positions row t sees. Outputs (zeros for a row
    that sees none) and a bound of what 32-bit arithmetic may be off: a score's error is taken as 4 u sqrt(HD) of its sum
    of |q k| (a random walk of rounded additions, four deviations), its parts' as 2^-22 of it and the exponential's
    argument's as u of its size; an output's as the largest |v| times twice the largest of these, and 4 u sqrt(n)."""
    T, H, HD = q.shape
    G = H // K.shape[1]
    q, K, V = q.astype(np.float64), K.astype(np.float64), V.astype(np.float64)
    out, tol = np.zeros_like(q), np.zeros((T, H, 1))
    for t in range(T):
        for h in range(H):
            at = sees[t][h // G]
            if not len(at):
                continue
            k, v = K[at, h // G], V[at, h // G]
            s = k @ q[t, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ v
            size = float((np.abs(k) @ np.abs(q[t, h])).max() * abs(scale))
            d = (4 * U * np.sqrt(HD) + 2.0 ** -22) * size + U * float(s.max() - s.min())
            tol[t, h] = np.abs(v).max() * (2 * d + 4 * U * np.sqrt(len(at)) + 4 * U)
    return out, tol


def rope_ref(x, pos, n, neox, base, freq_scale, freqs):
    """x [T][heads][HD] rotated at positions pos in 64 bits, and a bound of what 32-bit arithmetic is off: the cosine and sine
    (half a step each, and the angle's own error: n / 2 + 2 roundings in 64 bits), two products and a sum."""
    y, tol = x.astype(np.float64), np.zeros(x.shape)
    half = n // 2
    i = np.arange(half)
    a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
    ang = np.asarray(pos, np.float64)[:, None] * freq_scale * float(base) ** (-2.0 * i / max(n, 1))
    if freqs is not None:
        ang = ang / freqs.astype(np.float64)
    ang = ang[:, None]
    x0, x1 = y[..., a].copy(), y[..., b].copy()
    y[..., a] = x0 * np.cos(ang) - x1 * np.sin(ang)
    y[..., b] = x0 * np.sin(ang) + x1 * np.cos(ang)
    d = (np.abs(x0) + np.abs(x1)) * (3 * U + np.abs(ang) * (half + 2) * 2.0 ** -53)
    tol[..., a] = tol[..., b] = d
    return y, tol


def blocks_ref(q, lo, hi, cur, first, recent, top):
    """The pages a row takes of one KV head: q [G][HD], lo, hi [pages][HD] (a row of None where there is no page)."""
    start = min(first, cur + 1)
    end = max(start, cur + 1 - recent)
    sc = {}
    with np.errstate(invalid="ignore"):
        for j in range(start, end):
            if lo[j] is None:
                continue
            l, h = lo[j].astype(np.float64), hi[j].astype(np.float64)
            s = [float(np.sum(np.maximum(x, 0) * h + np.minimum(x, 0) * l)) for x in q.astype(np.float64)]
            sc[j] = max(v if np.isfinite(v) else np.inf for v in s)
    pick = sorted(sc, key=lambda j: (-sc[j], j))[:top]
    return sorted(list(range(start)) + pick + list(range(end, cur + 1)))


class Pool:
    """Sequences of `lengths` positions of random keys and values (fp16 numbers) in a pool of pages in random order; every other
    place of the pool holds NaN."""

    def __init__(self, ctx, lengths, KH, HD, page, seed=0, shared=0, bounds=False, room=64, spare=3, values=None):
        import torch
        self.torch, self.ctx, self.KH, self.HD, self.page = torch, ctx, KH, HD, page
        rng = np.random.default_rng(seed)
        N = len(lengths)
        width = (max(lengths) + room + page - 1) // page
        sh = shared // page
        self.pages = sh + N * (width - sh) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((N, width), -1, np.int32)
        self.table[:, :sh] = order[:sh]
        self.table[:, sh:] = order[sh:sh + N * (width - sh)].reshape(N, width - sh)
        self.d_table = torch.full((N, width), -7, dtype=torch.int32, device="cuda")
        n = self.pages * KH * page * HD
        self.dK, self.dV = (torch.full((n,), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
        self.dB = torch.full((self.pages * KH * 2 * HD,), float("nan"), dtype=torch.float16, device="cuda") if bounds else None
        self.desc = Pages(self.dK.data_ptr(), self.dV.data_ptr(), self.dB.data_ptr() if bounds else None,
                          self.d_table.data_ptr(), self.pages, page, KH, HD, N, width)
        torch.cuda.synchronize()
        for s in range(N):
            self.assign(s, 0, self.table[s])
        self.K, self.V = [], []
        for s in range(N):
            k, v = ((rng.standard_normal((lengths[s], KH, HD)) * m).astype(np.float16).astype(F32) for m in (1.5, 1.0))
            if values is not None:
                values(s, k, v)
            if s:
                k[:shared], v[:shared] = self.K[0][:shared], self.V[0][:shared]
            self.K.append(k)
            self.V.append(v)
        for s in range(N):
            self.store([s], [0], [lengths[s]], None, self.K[s], self.V[s])

    def dev(self, a):
        return None if a is None else self.torch.from_numpy(np.ascontiguousarray(a)).to("cuda")

    def assign(self, seq, first, ids):
        ids = (ctypes.c_int32 * len(ids))(*[int(i) for i in ids])
        check(load().wl_paged_assign_dev(self.ctx.handle, ctypes.byref(self.desc), seq, first, len(ids), ids))

    def store(self, seq, pos, rows, q, k, v, n=0, neox=0, base=10000.0, fs=1.0, freqs=None, inplace=False):
        p = lambda t: None if t is None else t.data_ptr()
        dq, dk, dv, df = (self.dev(a) for a in (q, k, v, freqs))
        out = dq if inplace or dq is None else self.torch.full_like(dq, float("nan"))
        self.torch.cuda.synchronize()
        check(load().wl_paged_store_dev(self.ctx.handle, ctypes.byref(self.desc), ctypes.byref(PageRows(seq, pos, rows)),
                                        p(dq), q.shape[1] if q is not None else 0, p(dk), p(dv), n, neox, base, fs, p(df),
                                        p(out)))
        self.ctx.sync()
        return None if out is None else out.cpu().numpy()

    def read(self, seq, pos0, T):
        k, v = (self.torch.full((T, self.KH, self.HD), float("nan"), device="cuda") for _ in range(2))
        self.torch.cuda.synchronize()
        check(load().wl_paged_read_dev(self.ctx.handle, ctypes.byref(self.desc), seq, pos0, T, k.data_ptr(), v.data_ptr()))
        self.ctx.sync()
        return k.cpu().numpy(), v.cpu().numpy()

    def attend(self, seq, pos, rows, q, prefix=0, scale=None, sparse=None):
        """Outputs; with sparse (first, recent, top) also the pages taken."""
        dq = self.dev(q)
        out = self.torch.full_like(dq, float("nan"))
        scale = self.HD ** -0.5 if scale is None else scale
        r = PageRows(seq, pos, rows)
        blocks = None
        if sparse:
            blocks = self.torch.full((q.shape[0], self.KH, sum(sparse)), -9, dtype=self.torch.int32, device="cuda")
        self.torch.cuda.synchronize()
        if sparse:
            check(load().wl_paged_sparse_dev(self.ctx.handle, ctypes.byref(self.desc), ctypes.byref(r), dq.data_ptr(),
                                             q.shape[1], ctypes.byref(SparseOpts(*sparse)), scale, out.data_ptr(),
                                             blocks.data_ptr()))
        else:
            check(load().wl_paged_attention_dev(self.ctx.handle, ctypes.byref(self.desc), ctypes.byref(r), dq.data_ptr(),
                                                q.shape[1], prefix, scale, out.data_ptr()))
        self.ctx.sync()
        return (out.cpu().numpy(), blocks.cpu().numpy()) if sparse else out.cpu().numpy()

    def bounds_of(self, seq, n):
        """Bounds [pages][KH][2][HD] of a sequence's first n pages, as the pool holds them."""
        b = self.dB.reshape(self.pages, self.KH, 2, self.HD).cpu().numpy().astype(F32)
        return b[self.table[seq, :n]]
