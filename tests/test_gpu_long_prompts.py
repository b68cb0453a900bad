"""Prompts of wl_layer_kv_dev over 4-bit caches and windows against their operations one at a time, bit for bit."""
import ctypes

import numpy as np
import pytest
import torch

from gpu_common import blocks
from test_gpu_long_models import BASE, E, EPS, FF, H, KH, Layer, P, caches, dev, host, same
from windlass_amd._lib import check, load
from windlass_amd.backend import Context, GgmlType

pytestmark = pytest.mark.gpu
F32 = np.float32
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def ctx():
    c = Context(0)
    yield c
    c.close()


class PromptLayer(Layer):
    """A layer whose down product adds zeros, so that its rows are x plus the attention's product."""

    def __init__(self, ctx, HD, rd, neox, seed=0):
        super().__init__(ctx, HD, rd, neox, seed)
        self.w["ffn_down"].free()
        zeros = np.zeros_like(blocks(GgmlType.Q6_K, E, FF, seed=0))
        self.w["ffn_down"] = ctx.upload(GgmlType.Q6_K, zeros, E, FF)
        self.d.ffn_down = self.w["ffn_down"].handle.value

    def operations(self, x, T, pos0, K, V, positions, bits, window, sinks, rope_from=None):
        """The norm, the products, RoPE (from another position where asked), the store, attention and the sum, each its own
        call, any T."""
        L, h, c, HD = load(), self.ctx.handle, ctypes.c_float, self.HD
        QD, KD = H * HD, KH * HD
        xn = torch.empty((T, E), device=DEV)
        q, k, v, att = (torch.empty((T, n), device=DEV) for n in (QD, KD, KD, QD))
        torch.cuda.synchronize()
        check(L.wl_rms_norm_dev(h, P(x), T, E, P(self.norms[0]), c(EPS), P(xn)))
        for n, y in (("attn_q", q), ("attn_k", k), ("attn_v", v)):
            check(L.wl_matmul_dev(h, self.w[n].handle, -1, P(xn), T, P(y)))
        for y, n in ((q, H), (k, KH)):
            check(L.wl_rope_dev(h, P(y), T, n, HD, self.rd, self.neox, pos0 if rope_from is None else rope_from, None, BASE,
                                0.5, P(self.freqs)))
        if bits == 4:
            check(L.wl_kv4_store_dev(h, P(k), P(v), T, KH, HD, P(K), P(V), positions, pos0))
            check(L.wl_kv4_attention_dev(h, P(q), T, H, KH, HD, P(K), P(V), positions, pos0, window, sinks, c(0.1), P(att)))
        else:
            check(L.wl_kv_store_dev(h, P(k), P(v), T, KD, P(K), P(V), pos0))
            check(L.wl_attention_window_dev(h, P(q), T, H, KH, HD, P(K), P(V), pos0, window, sinks, c(0.1), P(att)))
        check(L.wl_matmul_add_dev(h, self.w["attn_output"].handle, -1, P(att), T, P(x), c(0.5)))
        self.ctx.sync()


@pytest.mark.parametrize("bits,window,sinks", [(4, 0, 0), (4, 70, 3), (16, 70, 3)])
@pytest.mark.parametrize("HD,rd,neox", [(64, 48, 1), (128, 128, 0)])
@pytest.mark.parametrize("T,pos0", [(9, 30), (16, 0), (63, 5), (64, 5), (65, 0), (100, 41), (200, 7)])
def test_layer_prompts_equal_their_operations(ctx, T, pos0, HD, rd, neox, bits, window, sinks):
    """Rows and caches of a prompt's layer, either side of the rows that take RoPE and the store in one launch."""
    rng = np.random.default_rng(T + HD)
    l = PromptLayer(ctx, HD, rd, neox)
    positions = pos0 + T + 33
    K, V = caches(ctx, rng, positions, HD, bits)
    x0 = dev(rng.standard_normal((T, E), dtype=F32))
    xa, xb, xc = x0.clone(), x0.clone(), x0.clone()
    Kb, Vb, Kc, Vc = K.clone(), V.clone(), K.clone(), V.clone()
    torch.cuda.synchronize()
    l.run(xa, T, pos0, K, V, positions, bits, window, sinks)
    l.operations(xb, T, pos0, Kb, Vb, positions, bits, window, sinks)
    assert same(ctx, K, Kb) and same(ctx, V, Vb) and same(ctx, xa, xb)
    assert np.isfinite(host(ctx, xa)).all() and not same(ctx, xa, x0)
    # the comparison tells a wrong angle
    l.operations(xc, T, pos0, Kc, Vc, positions, bits, window, sinks, rope_from=pos0 + 1)
    assert not same(ctx, K, Kc) and same(ctx, V, Vc)
    l.free()
