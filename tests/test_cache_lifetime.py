"""When the storage of dropped caches is let go of: not before the stream has
passed the calls that were queued on it, and at once where a call has waited."""
import gc
import weakref

import numpy as np
import pytest

from krystal_b200 import BankCache, SessionBanks, abi
from krystal_b200 import cache as kc
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.frame import QUERY_BAND
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from tests.test_clip_lifetime import Buffer, Device, be, clip_a_temporary  # noqa: F401 (be: the fixture)

torch = pytest.importorskip("torch")
CFG = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))


def bare_cache():
    """A cache without a device."""
    cache = BankCache.__new__(BankCache)
    cache.storage, cache.device, cache.backends = Buffer(), torch.device("cuda", 0), []
    cache.view = abi.KcCacheView()
    return cache


def write(be, cache):
    be.cache_write(cache, kc.page_table(None, None, 0, 0), kc.cache_rows(None, None, "f32", 0))


def drop(cache_box):
    dead = weakref.ref(cache_box[0].storage)
    cache_box.clear()
    gc.collect()
    return dead


def test_a_cache_dropped_behind_its_call_is_held(be, monkeypatch):
    dev = Device(monkeypatch)
    box = [bare_cache()]
    write(be, box[0])
    dead = drop(box)
    assert dead() is not None
    write(be, bare_cache())  # records its event
    assert dead() is not None
    dev.passed = dev.recorded
    write(be, bare_cache())
    assert dead() is None


def test_a_wait_lets_go_at_once(be, monkeypatch):
    """What was dropped before a synchronize goes with it, without an event of its
    own; a cache dropped after goes by itself; one used again is held."""
    dev = Device(monkeypatch)
    box, second, third = [bare_cache()], [bare_cache()], [bare_cache()]
    for b in (box, second, third):
        write(be, b[0])
    clip, dead = clip_a_temporary(be), drop(box)
    assert drop([bare_cache()])() is None  # never used
    assert dead() is not None and clip() is not None
    be.synchronize()
    assert dead() is None and clip() is None and dev.recorded == 0
    assert drop(second)() is None
    write(be, third[0])
    assert drop(third)() is not None


def test_a_wait_that_began_before_covers_nothing_queued_in_it(be, monkeypatch):
    """A call and a drop by another thread, between the start of a wait and its end."""
    Device(monkeypatch)
    box = [bare_cache()]
    held = []

    class Slow(type(be._lib)):
        def __getattr__(self, name):
            if name == "kc_synchronize":
                def wait(*a):
                    write(be, box[0])
                    held.append(drop(box))
                    return 0
                return wait
            return super().__getattr__(name)

    be._lib = Slow()
    be.synchronize()
    assert held[0]() is not None


def test_a_cache_of_two_backends_waits_for_both(be, monkeypatch):
    Device(monkeypatch)
    other = CudaBrainBackend(CFG, create_brain_forward_weights(CFG, 1), 0)
    other._h = 1
    try:
        box = [bare_cache()]
        write(be, box[0])
        write(other, box[0])
        be.synchronize()
        dead = drop(box)
        assert dead() is not None
        other.synchronize()
        assert dead() is None
    finally:
        other._h = None


def test_a_refused_device_holds_nothing(be):
    cache = bare_cache()
    cache.device = torch.device("cuda", 1)
    with pytest.raises(ValueError, match="lies on"):
        write(be, cache)
    assert cache.backends == []


@pytest.mark.gpu
def test_banks_are_freed_with_their_last_turn():
    """Sessions' caches dropped behind a turn leave the memory at once."""
    b = CudaBrainBackend(CFG, create_brain_forward_weights(CFG, 1), 0)
    try:
        record = dict(schemaId=1, band=0, tokens=[3, 4])
        ask = dict(schemaId=1, band=QUERY_BAND, tokens=[5])
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        banks = SessionBanks(b, 64, 100)
        size = sum(c.storage.numel() for c in (*banks.mixer, banks.selector))
        banks.turn([("a", [record, ask])])
        assert torch.cuda.memory_allocated() >= before + size
        del banks
        gc.collect()
        assert torch.cuda.memory_allocated() <= before + 4096
        # a cache whose call was waited for by synchronize
        cache = BankCache(64)
        x = torch.zeros(1, 4, 32, device="cuda")
        pages, lengths = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated()
        b.cache_write(cache, kc.page_table(pages.data_ptr(), lengths.data_ptr(), 1, 1),
                      kc.cache_rows(x.data_ptr(), x.data_ptr(), "f32", 1))
        b.synchronize()
        del cache
        gc.collect()
        assert torch.cuda.memory_allocated() < held
    finally:
        b.destroy()
