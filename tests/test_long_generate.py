"""What generate() and sample() do around the library's calls, with a stand-in for it (no GPU): they wait for the model's own
device."""
import types

import torch

from windlass_amd import DeviceBatch, DeviceTransformer, KvCaches, ModelConfig, SampleParams

DEV = torch.device("cpu")  # the stand-in's buffers


class Library:
    """Entries that only write down their names."""

    def __init__(self, log):
        self.log = log

    def __getattr__(self, name):
        def call(*_):
            self.log.append(name)
            return 0
        return call


def model():
    log = []
    m = object.__new__(DeviceTransformer)
    m.log = log
    m.cfg = ModelConfig(layers=1, embd=4, heads=1, kv_heads=1, head_dim=64)
    m.L = Library(log)
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
