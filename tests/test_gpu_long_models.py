"""The 4-bit caches, windows and sampling together, as a model uses them: wl_layer_kv_dev and wl_layer_batch_kv_dev
against their operations one at a time, and a small model's generate() alone and batched.

Everything is compared bit for bit: the layer calls run the same kernels as the operations, a batch row is its
sequence's own step, and a drawn token follows from the logits and the given number (long_ref.sample_ref)."""
import ctypes

import numpy as np
import pytest
import torch

from gpu_common import blocks
from long_ref import sample_ref
from windlass_amd import DeviceBatch, DeviceTransformer, LayerDesc, ModelConfig, SampleParams
from windlass_amd._lib import ArgumentOutOfRangeError, NotSupportedError, ShapeError, check, load
from windlass_amd.backend import Context, GgmlType, KvOpts

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")
E, H, KH, FF, EPS, BASE = 256, 4, 2, 512, 1e-6, 10000.0


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


def P(t):
    return ctypes.c_void_p(t.data_ptr())


def dev(a):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    return t


def host(ctx, t):
    ctx.sync()
    return t.cpu().numpy()


class Layer:
    def __init__(self, ctx, HD, rd, neox, seed=0):
        QD, KD = H * HD, KH * HD
        rng = np.random.default_rng(seed)
        mats = {"attn_q": (GgmlType.Q4_K, QD, E), "attn_k": (GgmlType.Q8_0, KD, E), "attn_v": (GgmlType.Q6_K, KD, E),
                "attn_output": (GgmlType.Q4_K, E, QD), "ffn_gate": (GgmlType.Q4_K, FF, E),
                "ffn_up": (GgmlType.Q4_K, FF, E), "ffn_down": (GgmlType.Q6_K, E, FF)}
        self.ctx, self.HD, self.rd, self.neox = ctx, HD, rd, neox
        self.w = {n: ctx.upload(t, blocks(t, r, c, seed=i), r, c) for i, (n, (t, r, c)) in enumerate(mats.items())}
        self.norms = [dev((1 + 0.2 * rng.standard_normal(E)).astype(F32)) for _ in range(2)]
        self.freqs = dev((1 + 3 * rng.random(rd // 2)).astype(F32))
        d = self.d = LayerDesc()
        for n in mats:
            setattr(d, n, self.w[n].handle.value)
        d.d_attn_norm, d.d_ffn_norm = self.norms[0].data_ptr(), self.norms[1].data_ptr()
        d.d_rope_freqs = self.freqs.data_ptr()
        d.embd, d.heads, d.kv_heads, d.head_dim, d.rope_dims, d.neox = E, H, KH, HD, rd, neox
        d.rope_base, d.rope_freq_scale, d.eps, d.attention_scale, d.residual_scale = BASE, 0.5, EPS, 0.1, 0.5

    def operations(self, x, T, pos0, K, V, positions, bits, window, sinks):
        """The layer one operation at a time; T <= 8 (the products' fused entries)."""
        L, h, c, HD = load(), self.ctx.handle, ctypes.c_float, self.HD
        QD, KD = H * HD, KH * HD
        xn, g = (torch.empty((T, n), device=DEV) for n in (E, FF))
        q, k, v, att = (torch.empty((T, n), device=DEV) for n in (QD, KD, KD, QD))
        check(L.wl_rms_norm_dev(h, P(x), T, E, P(self.norms[0]), c(EPS), P(xn)))
        ws = (ctypes.c_void_p * 3)(*(self.w[n].handle.value for n in ("attn_q", "attn_k", "attn_v")))
        check(L.wl_matmul_multi_dev(h, 3, ws, P(xn), T, (ctypes.c_void_p * 3)(*(t.data_ptr() for t in (q, k, v)))))
        for y, n in ((q, H), (k, KH)):
            check(L.wl_rope_dev(h, P(y), T, n, HD, self.rd, self.neox, pos0, None, BASE, 0.5, P(self.freqs)))
        if bits == 4:
            check(L.wl_kv4_store_dev(h, P(k), P(v), T, KH, HD, P(K), P(V), positions, pos0))
            check(L.wl_kv4_attention_dev(h, P(q), T, H, KH, HD, P(K), P(V), positions, pos0, window, sinks, c(0.1), P(att)))
        else:
            check(L.wl_kv_store_dev(h, P(k), P(v), T, KD, P(K), P(V), pos0))
            check(L.wl_attention_window_dev(h, P(q), T, H, KH, HD, P(K), P(V), pos0, window, sinks, c(0.1), P(att)))
        check(L.wl_matmul_add_dev(h, self.w["attn_output"].handle, -1, P(att), T, P(x), c(0.5)))
        check(L.wl_rms_norm_dev(h, P(x), T, E, P(self.norms[1]), c(EPS), P(xn)))
        check(L.wl_gate_up_dev(h, self.w["ffn_gate"].handle, self.w["ffn_up"].handle, -1, P(xn), T, P(g)))
        check(L.wl_matmul_add_dev(h, self.w["ffn_down"].handle, -1, P(g), T, P(x), c(0.5)))
        self.ctx.sync()

    def run(self, x, T, pos0, K, V, positions, bits, window, sinks):
        o = KvOpts(bits, window, sinks, positions)
        check(load().wl_layer_kv_dev(self.ctx.handle, ctypes.byref(self.d), P(x), T, pos0, P(K), P(V), ctypes.byref(o)))

    def free(self):
        for w in self.w.values():
            w.free()


def caches(ctx, rng, positions, HD, bits, lead=()):
    """Caches of `positions` positions, all of them stored."""
    if bits == 16:
        shape = tuple(lead) + (positions, KH * HD)
        return [dev(rng.standard_normal(shape, dtype=F32).astype(np.float16).view(np.int16)) for _ in range(2)]
    n = load().wl_kv4_bytes(positions, KH, HD)
    K, V = (torch.zeros(tuple(lead) + (n,), dtype=torch.uint8, device=DEV) for _ in range(2))
    torch.cuda.synchronize()
    for kk, vv in zip(K.reshape(-1, n), V.reshape(-1, n)):
        k, v = (dev(rng.standard_normal((positions, KH, HD), dtype=F32)) for _ in range(2))
        check(load().wl_kv4_store_dev(ctx.handle, P(k), P(v), positions, KH, HD, P(kk), P(vv), positions, 0))
        ctx.sync()
    return [K, V]


def same(ctx, a, b):
    a, b = host(ctx, a), host(ctx, b)
    return np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("bits,window,sinks", [(4, 0, 0), (4, 70, 3), (16, 70, 3)])
@pytest.mark.parametrize("T,pos0,HD,rd,neox", [(1, 0, 64, 64, 0), (1, 300, 128, 64, 1), (5, 37, 64, 32, 1), (8, 0, 128, 128, 0)])
def test_layer_equals_its_operations(ctx, T, pos0, HD, rd, neox, bits, window, sinks):
    rng = np.random.default_rng(T + pos0)
    l = Layer(ctx, HD, rd, neox)
    positions = pos0 + T + 40
    K, V = caches(ctx, rng, positions, HD, bits)
    x0 = dev(rng.standard_normal((T, E), dtype=F32))
    xa, xb, Kb, Vb = x0.clone(), x0.clone(), K.clone(), V.clone()
    torch.cuda.synchronize()
    l.run(xa, T, pos0, K, V, positions, bits, window, sinks)
    l.operations(xb, T, pos0, Kb, Vb, positions, bits, window, sinks)
    assert same(ctx, xa, xb) and same(ctx, K, Kb) and same(ctx, V, Vb)
    assert np.isfinite(host(ctx, xa)).all() and not same(ctx, xa, x0)
    l.free()


@pytest.mark.parametrize("T", [64, 65, 100])
def test_prompt_stores_equal_its_operations(ctx, T):
    """RoPE and the 4-bit stores either side of the rows that share their angles."""
    rng = np.random.default_rng(T)
    HD, positions = 64, T + 9
    l = Layer(ctx, HD, 48, 1)
    K, V = caches(ctx, rng, positions, HD, 4)
    x = dev(rng.standard_normal((T, E), dtype=F32))
    l.run(x, T, 5, K, V, positions, 4, 0, 0)
    k, v = (torch.empty((T, KH, HD), device=DEV) for _ in range(2))
    torch.cuda.synchronize()
    check(load().wl_kv4_read_dev(ctx.handle, P(K), P(V), positions, KH, HD, 5, T, P(k), P(v)))
    gk, gv = host(ctx, k), host(ctx, v)
    assert np.isfinite(gk).all() and np.isfinite(gv).all() and np.abs(gk).max() > 0
    # held values are fixed points of the store
    K2, V2 = torch.zeros_like(K), torch.zeros_like(V)
    torch.cuda.synchronize()
    check(load().wl_kv4_store_dev(ctx.handle, P(k), P(v), T, KH, HD, P(K2), P(V2), positions, 5))
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    torch.cuda.synchronize()
    check(load().wl_kv4_read_dev(ctx.handle, P(K2), P(V2), positions, KH, HD, 5, T, P(k2), P(v2)))
    assert np.array_equal(host(ctx, k2), gk) and np.array_equal(host(ctx, v2), gv)
    l.free()


def test_plain_options_are_wl_layer_dev(ctx):
    rng = np.random.default_rng(3)
    l = Layer(ctx, 64, 64, 0)
    for T, pos0 in ((1, 20), (3, 0), (20, 7)):
        K, V = caches(ctx, rng, 60, 64, 16)
        x = dev(rng.standard_normal((T, E), dtype=F32))
        xb, Kb, Vb = x.clone(), K.clone(), V.clone()
        torch.cuda.synchronize()
        l.run(x, T, pos0, K, V, 60, 16, 0, 5)
        check(load().wl_layer_dev(ctx.handle, ctypes.byref(l.d), P(xb), T, pos0, P(Kb), P(Vb)))
        assert same(ctx, x, xb) and same(ctx, K, Kb) and same(ctx, V, Vb)
    l.free()


@pytest.mark.parametrize("bits,window,sinks", [(4, 0, 0), (4, 33, 2), (16, 33, 2), (16, 0, 0)])
@pytest.mark.parametrize("N", [1, 5, 70])
def test_batch_rows_equal_single_tokens(ctx, N, bits, window, sinks):
    rng = np.random.default_rng(N)
    HD, cap, slots = 64, 120, N + 3
    l = Layer(ctx, HD, HD, 0)
    K, V = caches(ctx, rng, cap, HD, bits, (slots,))
    pos = rng.integers(0, cap, N).astype(np.int32)
    slot = rng.permutation(slots)[:N].astype(np.int32)
    x = dev(rng.standard_normal((N, E), dtype=F32))
    xb, Kb, Vb = x.clone(), K.clone(), V.clone()
    torch.cuda.synchronize()
    o = KvOpts(bits, window, sinks, 0)
    check(load().wl_layer_batch_kv_dev(ctx.handle, ctypes.byref(l.d), P(x), N, pos.ctypes.data, slot.ctypes.data, slots, cap,
                                       P(K), P(V), ctypes.byref(o)))
    for i in range(N):
        l.run(xb[i:i + 1], 1, int(pos[i]), Kb[slot[i]], Vb[slot[i]], cap, bits, window, sinks)
    assert same(ctx, x, xb) and same(ctx, K, Kb) and same(ctx, V, Vb)
    l.free()


def test_layer_refusals(ctx):
    l = Layer(ctx, 64, 64, 0)
    K, V = caches(ctx, np.random.default_rng(0), 10, 64, 4)
    x = torch.zeros((1, E), device=DEV)
    torch.cuda.synchronize()
    with pytest.raises(ArgumentOutOfRangeError):
        l.run(x, 1, 10, K, V, 10, 4, 0, 0)
    with pytest.raises(ArgumentOutOfRangeError):
        l.run(x, 1, 0, K, V, 10, 4, -1, 0)
    with pytest.raises(NotSupportedError):
        l.run(x, 1, 0, K, V, 10, 8, 0, 0)
    with pytest.raises(ShapeError):
        l.run(x, 1, 0, K, V, 0, 4, 0, 0)
    l.d.head_dim = 96
    with pytest.raises(NotSupportedError):
        l.run(x, 1, 0, K, V, 10, 4, 0, 0)
    cfg = ModelConfig(layers=1, embd=E, heads=H, kv_heads=KH, head_dim=96)
    with pytest.raises(NotSupportedError):
        DeviceTransformer(ctx, cfg, {"token_embd": l.w["ffn_gate"]}, {}, 10, kv_bits=4)
    l.free()


VOCAB, HD, LAYERS = 500, 64, 2


def model(ctx, **kw):
    cfg = ModelConfig(layers=LAYERS, embd=E, heads=H, kv_heads=KH, head_dim=HD, rope_base=BASE, eps=EPS)
    up = lambda t, r, c, s: ctx.upload(t, blocks(t, r, c, seed=s), r, c)  # noqa: E731
    w = {"token_embd": up(GgmlType.Q8_0, VOCAB, E, 1), "output": up(GgmlType.Q6_K, VOCAB, E, 2)}
    v = {"output_norm": torch.ones(E, device=DEV)}
    for l in range(LAYERS):
        for i, (n, r, c) in enumerate((("attn_q", H * HD, E), ("attn_k", KH * HD, E), ("attn_v", KH * HD, E),
                                       ("attn_output", E, H * HD), ("ffn_gate", FF, E), ("ffn_up", FF, E),
                                       ("ffn_down", E, FF))):
            w["blk.%d.%s" % (l, n)] = up(GgmlType.Q4_K, r, c, 10 + 10 * l + i)
        v["blk.%d.attn_norm" % l] = torch.ones(E, device=DEV)
        v["blk.%d.ffn_norm" % l] = torch.ones(E, device=DEV)
    return DeviceTransformer(ctx, cfg, w, v, 200, **kw), w


@pytest.mark.parametrize("kw", [dict(), dict(kv_bits=4), dict(kv_bits=4, window=20, sinks=2), dict(window=20, sinks=2)])
def test_generate_alone_and_batched(ctx, kw):
    rng = np.random.default_rng(1)
    m, w = model(ctx, **kw)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (3, 40, 8)]
    params = [SampleParams(0.9, 50, 0.95, 0.02), SampleParams(1.3), SampleParams(0.0)]
    steps = 12
    u = rng.random((steps, 3)).astype(F32)
    alone = [m.generate(p, steps, params[i], u[:, i]) for i, p in enumerate(prompts)]
    assert DeviceBatch(m, 4, 80).generate(prompts, steps, params, u) == alone
    # each token is the draw from the logits that the same steps leave
    for i, p in enumerate(prompts):
        m.forward(p, 0)
        s = params[i]
        for t in range(steps):
            want, _ = sample_ref(m.host_logits()[:], u[t, i], float(s.temperature), s.top_k, float(s.top_p), float(s.min_p))
            assert want == alone[i][t] == m.sample(s, float(u[t, i])), (i, t)
            if t + 1 < steps:
                m.forward([want], len(p) + t)
    assert m.generate(prompts[0], 6, SampleParams(0.0), [0.5] * 6) == m.greedy(prompts[0], 6)
    with pytest.raises(ShapeError):
        m.generate(prompts[0], 6, params[0], [0.5] * 5)
    for x in w.values():
        x.free()


def test_a_window_changes_nothing_before_it_and_something_after(ctx):
    rng = np.random.default_rng(2)
    p = rng.integers(0, VOCAB, 30).tolist()
    full, w1 = model(ctx, kv_bits=4)
    cut, w2 = model(ctx, kv_bits=4, window=31, sinks=0)
    small, w3 = model(ctx, kv_bits=4, window=10, sinks=1)
    for m in (full, cut, small):
        m.forward(p, 0)
    a, b, c = (m.host_logits() for m in (full, cut, small))
    assert np.array_equal(a, b) and not np.array_equal(a, c) and np.isfinite(c).all()
    for x in (*w1.values(), *w2.values(), *w3.values()):
        x.free()
