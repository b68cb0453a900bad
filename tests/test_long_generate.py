"""What generate() and sample() do around the library's calls, with a stand-in for it (no GPU): they wait for the model's own
device, refuse what does not fit before anything is queued, and leave nothing queued when a call fails."""
import types

import pytest
import torch

from windlass_amd import DeviceBatch, DeviceTransformer, KvCaches, ModelConfig, SampleParams
from windlass_amd._lib import WL_E_ARG, ArgumentOutOfRangeError, ShapeError

DEV = torch.device("cpu")  # the stand-in's buffers


class Library:
    """Entries that only write down their names; the one called `fails` refuses after `after` calls."""

    def __init__(self, log, fails=None, after=0):
        self.log, self.fails, self.after = log, fails, after

    def __getattr__(self, name):
        def call(*_):
            self.log.append(name)
            if name == self.fails:
                self.after -= 1
                return WL_E_ARG if self.after < 0 else 0
            return 0
        return call


def model(**kw):
    log = []
    m = object.__new__(DeviceTransformer)
    m.log = log
    m.cfg = ModelConfig(layers=1, embd=4, heads=1, kv_heads=1, head_dim=64)
    m.L = Library(log, **kw)
    m.ctx = types.SimpleNamespace(handle=None, device=0, sync=lambda: log.append("sync"))
    waits = types.SimpleNamespace(synchronize=lambda device=None: log.append(("wait", device)))
    m.torch = types.SimpleNamespace(cuda=waits, **{n: getattr(torch, n) for n in ("full", "empty", "zeros", "as_tensor", "int32",
                                                                                  "uint8", "int16")})
    m.dev, m.vocab, m.max_positions, m.length = DEV, 5, 20, 0
    m.embd_w = m.head_w = types.SimpleNamespace(handle=None)
    m.v, m.descs, m.stream, m._x = {"output_norm": torch.ones(4)}, [], None, {}
    m.logits, m._tok, m._xn = torch.zeros((1, 5)), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 4))
    m.kv = object.__new__(KvCaches)
    m.kv.cfg, m.kv.bits, m.kv.window, m.kv.sinks = m.cfg, 16, 0, 0
    return m


def before(log, first, then):
    return log.index(first) < log.index(then)


def test_the_draw_waits_for_the_models_device():
    """The number is written by a kernel on the model's device, whichever device is current."""
    m = model()
    m.sample(SampleParams(0.8), 0.5)
    assert before(m.log, ("wait", DEV), "wl_sample_dev")
    m = model()
    m.generate([1, 2], 3, SampleParams(0.8), [0.1, 0.2, 0.3])
    assert before(m.log, ("wait", DEV), "wl_embed_dev") and ("wait", None) not in m.log
    m = model()
    b = DeviceBatch(m, 2, 20)
    assert m.log[-1] == ("wait", DEV)  # the pools' zeros
    del m.log[:]
    b.generate([[1], [2, 3]], 2, [SampleParams()] * 2, [0.1] * 4)
    assert before(m.log, ("wait", DEV), "wl_embed_dev") and ("wait", None) not in m.log


def test_what_does_not_fit_is_refused_before_anything_runs():
    p = SampleParams()
    for prompt, steps in (([], 2), ([1] * 21, 0), ([1] * 20, 2), ([1] * 5, 17)):
        for chunk in (None, 3):
            m = model()
            with pytest.raises(ShapeError):
                m.generate(prompt, steps, p, [0.5] * steps, chunk)
            assert not [x for x in m.log if isinstance(x, str)]
    assert len(model().generate([1] * 5, 16, p, [0.5] * 16)) == 16  # the last token takes no position
    for prompts, steps in (([[1], []], 2), ([[1], [1] * 21], 1), ([[1], [1] * 8], 14), ([[1]] * 3, 1)):
        m = model()
        b = DeviceBatch(m, 2, 20)
        with pytest.raises(ShapeError):
            b.generate(prompts, steps, [p] * len(prompts), [0.5] * (steps * len(prompts)))
        assert not [x for x in m.log if isinstance(x, str)]
    m = model()
    b = DeviceBatch(m, 2, 20)
    b.generate([[1], [1] * 8], 13, [p] * 2, [0.5] * 26)
    with pytest.raises(ShapeError):  # the second sequence's slot is full
        b.generate([[1], [1]], 1, [p] * 2, [0.5] * 2)


@pytest.mark.parametrize("fails,after", [("wl_sample_dev", 1), ("wl_embed_dev_ids", 2), ("wl_embed_dev", 0)])
def test_nothing_stays_queued_after_a_failure(fails, after):
    """The numbers and tokens go back to torch's allocator when generate() ends, so their last use is waited for."""
    m = model(fails=fails, after=after)
    with pytest.raises(ArgumentOutOfRangeError):
        m.generate([1, 2], 5, SampleParams(), [0.5] * 5)
    assert m.log[-1] == "sync"
    m = model(fails=fails, after=after)
    b = DeviceBatch(m, 2, 20)
    with pytest.raises(ArgumentOutOfRangeError):
        b.generate([[1, 2], [3]], 5, [SampleParams()] * 2, [0.5] * 10)
    assert m.log[-1] == "sync"


@pytest.mark.parametrize("kw", [dict(window=-1), dict(sinks=-1), dict(window=1 << 31), dict(window=1 << 32), dict(sinks=1 << 32)])
def test_windows_past_32_bits_are_refused(kw):
    """2^32 would reach the library as 0: no window."""
    cfg = ModelConfig(layers=1, embd=4, heads=1, kv_heads=1, head_dim=64)
    assert KvCaches(cfg, window=(1 << 31) - 1, sinks=(1 << 31) - 1).opts(5).window == (1 << 31) - 1
    with pytest.raises(ShapeError):
        KvCaches(cfg, **kw)
