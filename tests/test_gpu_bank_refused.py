"""Turns over cached banks that are refused: what a call can refuse it refuses
before it appends, and when it has answered nothing of it is left to run."""
import numpy as np
import pytest

from krystal_b200 import SessionBanks, abi
from krystal_b200.cache import page_table
from krystal_b200.frame import pack_frame_batch
from krystal_b200.policy import Sampling
from tests.test_gpu_bank_turn import be, frame_records  # noqa: F401 (be: the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Call:
    """One turn of one session, as SessionBanks makes it, in device arrays."""

    def __init__(self, be, seed=21):
        (bank, asks), = frame_records(seed, 1)
        self.be, self.asks, self.held = be, len(asks), len(bank)
        self.banks = SessionBanks(be, 10, 600)
        b = pack_frame_batch([bank + asks])
        self.frames, self.records = b.frames, b.records
        up = lambda a, t: torch.from_numpy(np.ascontiguousarray(a).view(t)).cuda()  # noqa: E731
        self.batch = [up(b.rec_off.astype(np.uint64), np.int64)]
        self.batch += [up(np.asarray(x, np.uint32), np.int32) for x in (b.token_ids, b.field_roles, b.schema_ids, b.band_ids)]
        self.pages, self.lengths = torch.arange(10, dtype=torch.int32).cuda(), torch.tensor([self.held], dtype=torch.int32).cuda()
        self.p, self.index = torch.full((self.asks, 600), 7.0).cuda(), torch.full((self.asks,), 7, dtype=torch.int32).cuda()
        self.uniforms = torch.full((self.asks + 1,), 0.5, dtype=torch.float64).cuda()
        for c in (*self.banks.mixer, self.banks.selector):
            c.storage.fill_(0x5A)
        self.before = [c.storage.clone() for c in (*self.banks.mixer, self.banks.selector)]
        torch.cuda.synchronize()

    def run(self, uniforms=0, q_capacity=None, sampling=None):
        self.be.bank_turn(self.frames, self.records, *(t.data_ptr() for t in self.batch), self.banks.mixer,
                          self.banks.selector, page_table(self.pages.data_ptr(), self.lengths.data_ptr(), 1, 10, 600),
                          self.p.data_ptr(), self.asks if q_capacity is None else q_capacity, index=self.index.data_ptr(),
                          uniforms=self.uniforms.data_ptr() + uniforms, sampling=sampling)

    def idle(self):
        return torch.cuda.ExternalStream(self.be.stream_ptr(), device=self.be.device).query()

    def untouched(self):
        return (all(torch.equal(c.storage, s) for c, s in zip((*self.banks.mixer, self.banks.selector), self.before))
                and bool((self.p == 7.0).all()) and bool((self.index == 7).all()))


@pytest.mark.parametrize("how,match", [(dict(uniforms=4), "8-byte aligned"), (dict(q_capacity=1), "output rows are fewer"),
                                       (dict(sampling=Sampling(temperature=-1.0)), "temperature")])
def test_a_refused_turn_appends_nothing_and_leaves_nothing_queued(be, how, match):
    call = Call(be)
    with pytest.raises(abi.KrystalCudaError, match=match):
        call.run(**how)
    assert call.idle()
    assert call.untouched()
    call.run()
    assert call.idle() and not call.untouched()
    assert np.allclose(call.p[:, :call.held].sum(1).cpu().numpy(), 1, atol=1e-5) and bool((call.p[:, call.held:] == 0).all())


def test_a_turn_refused_on_the_device_leaves_nothing_queued(be):
    """Records outside the vocabulary: found while the batch is packed."""
    call = Call(be)
    call.batch[1].fill_(2 ** 31 - 1)
    torch.cuda.synchronize()
    with pytest.raises(abi.KrystalCudaError):
        call.run()
    assert call.idle() and call.untouched()
