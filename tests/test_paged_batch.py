"""What PagedBatch keeps of its pages, and refuses, with a stand-in for the library (no GPU)."""
import pytest
import torch

from test_long_generate import DEV, before, model
from windlass_amd import PagedBatch, SampleParams
from windlass_amd._lib import ArgumentOutOfRangeError, NotSupportedError, ShapeError


def batch(m, pages=6, slots=3, cap=100, page=16, **kw):
    return PagedBatch(m, pages, slots, cap, page, **kw)


def queued(m):
    return [x for x in m.log if isinstance(x, str)]


def test_pools_wait_for_the_models_device():
    m = model()
    batch(m)
    assert m.log[-1] == ("wait", DEV)


def test_pages_are_taken_as_sequences_grow_and_come_back():
    m = model()
    b = batch(m)
    b.prefill(0, [1] * 16)
    assert len(b.held[0]) == 1 and len(b.free_pages) == 5
    b.step([0], torch.zeros(1, dtype=torch.int32))
    assert len(b.held[0]) == 2 and b.length[0] == 17
    b.prefill(1, [1] * 40)
    assert len(b.free_pages) == 1
    del m.log[:]
    with pytest.raises(ShapeError):  # two pages, one is free: nothing is taken
        b.prefill(2, [1] * 17)
    assert not m.log and len(b.free_pages) == 1
    b.prefill(2, [1])
    with pytest.raises(ShapeError):  # 17 positions of 32 are held: one more page than there is
        b.prefill(0, [1] * 40)
    assert b.length == [17, 40, 1] and [len(h) for h in b.held] == [2, 3, 1] and not b.free_pages
    b.release(1)
    assert len(b.free_pages) == 3 and b.length[1] == 0
    assert sorted(b.free_pages + b.held[0] + b.held[2]) == list(range(6))


def test_shared_pages_are_free_when_no_sequence_holds_them():
    b = batch(model())
    b.prefill(0, [1] * 40)
    b.share(0, 1, 32)
    b.share(0, 2, 16)
    assert b.held[1] == b.held[0][:2] and b._shared([0, 1]) == 32 and b._shared([0, 1, 2]) == 16 and b._shared([2, 1]) == 16
    b.prefill(1, [1] * 3)
    assert b.held[1][2] != b.held[0][2] and len(b.free_pages) == 2
    b.release(0)
    assert len(b.free_pages) == 3
    b.release(1)
    assert len(b.free_pages) == 5
    b.release(2)
    assert sorted(b.free_pages) == list(range(6)) and not any(b.users)


def test_what_cannot_be_shared():
    b = batch(model())
    b.prefill(0, [1] * 40)
    for src, dst, n in ((0, 1, 17), (0, 1, 48), (0, 1, -16), (1, 0, 0)):
        with pytest.raises(ShapeError):
            b.share(src, dst, n)
    for src, dst in ((0, 0), (0, 3), (-1, 1)):
        with pytest.raises(ArgumentOutOfRangeError):
            b.share(src, dst, 16)
    assert len(b.free_pages) == 3


def test_sequences_out_of_range_or_twice():
    m = model()
    b = batch(m)
    del m.log[:]
    ids = torch.zeros(2, dtype=torch.int32)
    for slots in ([0, 0], [0, 3], [-1, 0]):
        with pytest.raises(ArgumentOutOfRangeError):
            b.step(slots, ids)
    for call in (lambda: b.prefill(3, [1]), lambda: b.release(-1)):
        with pytest.raises(ArgumentOutOfRangeError):
            call()
    with pytest.raises(ShapeError):
        b.prefill(0, [])
    assert not m.log


def test_what_does_not_fit_is_refused_before_anything_runs():
    p = SampleParams()
    for prompts, steps, shared in (([[1] * 90], 1, 0), ([[1] * 40, [1] * 40, [1] * 40], 1, 0), ([[1], []], 2, 0),
                                   ([[1] * 101], 0, 0), ([[1]] * 4, 1, 0), ([[1, 2], [2, 2]], 1, 1), ([[1], [1]], 1, 2),
                                   ([[1] * 40] * 3, 20, 40)):
        m = model()
        b = batch(m, pages=5)
        with pytest.raises(ShapeError):
            b.generate(prompts, steps, [p] * len(prompts), [0.5] * (steps * len(prompts)), shared=shared)
        assert not queued(m), (prompts, steps)
    m = model()
    b = batch(m, pages=5)
    with pytest.raises(ShapeError):
        b.generate([[1] * 40] * 3, 2, [p] * 2, [0.5] * 6, shared=40)
    assert not queued(m)
    b.generate([[1] * 40] * 3, 8, [p] * 3, [0.5] * 24, shared=40)  # two pages once, and one of each
    assert not b.free_pages and b.length == [47] * 3
    with pytest.raises(ShapeError):
        b.generate([[1] * 40] * 3, 1, [p] * 3, [0.5] * 3, shared=40)  # they hold positions


def test_models_that_pages_do_not_hold():
    for name, value in (("bits", 4), ("window", 5)):
        m = model()
        setattr(m.kv, name, value)
        with pytest.raises(NotSupportedError):
            batch(m)
    m = model()
    with pytest.raises(NotSupportedError):
        batch(m, page=24)
    m.cfg.head_dim = 80
    with pytest.raises(NotSupportedError):
        batch(m)
    for kw in (dict(pages=0), dict(slots=0), dict(cap=0), dict(cap=1 << 31), dict(pages=1 << 31)):
        with pytest.raises(ShapeError):
            batch(model(), **kw)


def test_pages_stay_free_when_they_cannot_be_assigned():
    m = model(fails="wl_paged_assign_dev")
    b = batch(m)
    with pytest.raises(ArgumentOutOfRangeError):
        b.prefill(0, [1] * 20)
    assert len(b.free_pages) == 6 and b.held[0] == [] and not any(b.users)


@pytest.mark.parametrize("fails,after", [("wl_sample_dev", 1), ("wl_embed_dev_ids", 2), ("wl_embed_dev", 0), ("wl_embed_dev", 1),
                                         ("wl_paged_assign_dev", 1)])
def test_nothing_stays_queued_after_a_failure(fails, after):
    m = model(fails=fails, after=after)
    b = batch(m)
    with pytest.raises(ArgumentOutOfRangeError):
        b.generate([[1] * 20, [1] * 20], 5, [SampleParams()] * 2, [0.5] * 10, shared=18)
    assert m.log[-1] == "sync"


def test_a_sequence_set_back_does_not_write_into_pages_that_others_hold():
    m = model()
    b = batch(m)
    b.prefill(0, [1] * 40)
    b.share(0, 1, 32)
    b.length[0] = 20
    del m.log[:]
    for call in (lambda: b.prefill(0, [1]), lambda: b.step([0], torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ShapeError):
            call()
    assert not m.log
    b.length[0] = 33
    b.prefill(0, [1])
    b.release(1)
    b.length[0] = 20
    b.prefill(0, [1])
    assert b.length[0] == 21 and len(b.held[0]) == 3


def test_a_shared_beginning_for_sequences_that_hold_pages_is_refused():
    m = model()
    b = batch(m)
    b.prefill(1, [1] * 16)
    b.length[1] = 0
    del m.log[:]
    with pytest.raises(ShapeError):
        b.generate([[1] * 20, [1] * 20], 2, [SampleParams()] * 2, [0.5] * 4, shared=16)
    assert not queued(m)


def test_what_all_of_the_sequences_share():
    """Against its definition, over sequences that begin at one another."""
    import random
    rng = random.Random(0)
    b = batch(model(), pages=200, slots=8, cap=200)
    for s in range(8):
        if s and rng.random() < 0.8:
            src = rng.randrange(s)
            b.share(src, s, rng.randrange(0, b.length[src] // 16 + 1) * 16)
        b.prefill(s, [1] * rng.randrange(1, 80))
    for _ in range(300):
        slots = rng.sample(range(8), rng.randrange(1, 9))
        n = 0
        for ids in zip(*(b.held[s] for s in slots)):
            if len(set(ids)) > 1:
                break
            n += 1
        assert b._shared(slots) == (n * 16 if len(slots) > 1 else 0)
