"""A queued clip's list, gradients and workspace live until the stream has
passed them, whoever else drops the list."""
import contextlib
import gc
import weakref

import numpy as np
import pytest

from krystal_b200 import abi
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from krystal_b200.policy import GradList

torch = pytest.importorskip("torch")
CFG = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))


class Buffer:
    def data_ptr(self):
        return 64


def grad_list():
    """A list without a device: its workspace is what has to live."""
    grads = GradList.__new__(GradList)
    grads.device, grads.address, grads.count, grads.workspace_bytes = torch.device("cuda", 0), 64, 1, 64
    grads.workspace, grads.keep, grads.backends = Buffer(), (), []
    return grads


class Device:
    """Events that pass when told to; a stream that may be capturing."""

    def __init__(self, monkeypatch):
        self.passed, self.recorded, self.asked, self.capturing = 0, 0, 0, False
        dev = self

        class Event:
            def record(self, stream):
                assert not dev.capturing
                dev.recorded += 1
                self.n = dev.recorded

            def query(self):
                assert not dev.capturing
                dev.asked += 1
                return self.n <= dev.passed

        monkeypatch.setattr(torch.cuda, "Event", Event)
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda ptr, device=None: ptr)
        monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: dev.capturing)


class Library:
    def __getattr__(self, name):
        return (lambda *a: 1) if name == "kc_get_stream" else (lambda *a: 0)


@pytest.fixture()
def be(monkeypatch):
    monkeypatch.setattr(abi, "load", lambda path=None: Library())
    b = CudaBrainBackend(CFG, create_brain_forward_weights(CFG, 1), 0)
    b._h = 1
    yield b
    b.destroy()


def clip_a_temporary(be):
    grads = grad_list()
    dead = weakref.ref(grads.workspace)
    be.clip_grads(grads, 1.0, 64)
    del grads
    gc.collect()
    return dead


def test_a_temporary_list_outlives_its_call(be, monkeypatch):
    dev = Device(monkeypatch)
    first = clip_a_temporary(be)
    assert first() is not None
    second = clip_a_temporary(be)  # nothing has passed yet
    assert first() is not None and second() is not None
    dev.passed = dev.recorded
    third = clip_a_temporary(be)  # the first one's event was recorded in the second's call
    assert first() is None and second() is not None and third() is not None
    dev.passed = 10 ** 6
    be.synchronize()
    assert second() is None and third() is None


def test_destroy_lets_go_of_every_list(be, monkeypatch):
    Device(monkeypatch)
    lists = [clip_a_temporary(be) for _ in range(3)]
    assert all(x() is not None for x in lists)
    be.destroy()
    assert all(x() is None for x in lists)


def test_lists_used_again_cost_no_event(be, monkeypatch):
    dev = Device(monkeypatch)
    lists = [grad_list(), grad_list()]
    for i in range(6):
        be.clip_grads(lists[i % 2], 1.0, 64)
    assert dev.recorded == 0 and dev.asked == 0


def test_no_event_is_touched_while_a_graph_is_captured(be, monkeypatch):
    dev = Device(monkeypatch)
    before = clip_a_temporary(be)
    dev.capturing = True
    held = [grad_list(), grad_list()]
    for x in held:
        be.clip_grads(x, 1.0, 64)
    assert before() is not None and dev.recorded == 0
    dev.capturing, dev.passed = False, 10 ** 6
    be.clip_grads(held[0], 1.0, 64)
    assert before() is None


def test_a_list_outlives_none_of_its_backends(be, monkeypatch):
    Device(monkeypatch)
    grads = grad_list()
    dead = weakref.ref(grads.workspace)
    be.clip_grads(grads, 1.0, 64)
    be.destroy()  # has waited for the stream
    del grads
    assert dead() is None


@pytest.mark.gpu
def test_a_temporary_lists_workspace_is_not_handed_out_again():
    """Clips of temporary lists queued on the handle's own stream, each behind
    others, while torch's stream takes and fills blocks of the workspace's
    size."""
    be = CudaBrainBackend(CFG, create_brain_forward_weights(CFG, 1), 0)
    try:
        grads = [torch.randn(3_000_000, device="cuda") for _ in range(4)]
        outs = [torch.empty_like(g) for g in grads]
        want = float(torch.cat(grads).double().norm())
        size = GradList(grads).workspace.numel()
        res = torch.zeros(40, 2, dtype=torch.float64, device="cuda")
        torch.cuda.synchronize()
        for i in range(40):
            lst = GradList(grads, outs)
            at = lst.workspace.data_ptr()
            be.clip_grads(lst, want / 2, res[i].data_ptr())
            del lst
            blocks = [torch.full((size,), 1e9, dtype=torch.float64, device="cuda") for _ in range(3)]
            assert at not in [b.data_ptr() for b in blocks]
            del blocks
        be.synchronize()
        assert (res[:, 0] - want).abs().max() <= want * 2.0 ** -28 and torch.equal(res[:, 0], res[:1, 0].expand(40))
    finally:
        be.destroy()
