"""The handle's policy on the framework's paths: targets that it does not hold,
and the learn step's."""
import numpy as np
import pytest

from krystal_b200 import abi
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.learn import BatchLearner, LearnOptions
from krystal_b200.policy import Sampling
from tests.test_gpu_policy_paths import CFG, frame_and_targets, learn_batch, weights

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    b = CudaBrainBackend(CFG, weights(), 0)
    yield b
    b.destroy()


@pytest.mark.parametrize("s", [Sampling(), Sampling(0.5), Sampling(0.8, 9), Sampling(1.7, 0, 0.6, 0.2)])
@pytest.mark.parametrize("away", [0, abi.KC_AWAY_TARGET])
def test_a_target_outside_the_row_moves_nothing_under_a_policy(be, s, away):
    frame, q, r, _ = frame_and_targets(21, False)
    none = np.full(q, abi.KC_NO_TARGET, np.uint32)
    outside = np.array([r, r + 7, 0x7ffffffe], np.uint32)[np.arange(q) % 3] | np.uint32(away)
    free = be.backward(frame, targets=outside)
    quiet = be.backward(frame, targets=none)
    be.set_policy(s)
    try:
        got, want = be.backward(frame, targets=outside), be.backward(frame, targets=none)
    finally:
        be.set_policy(None)
    assert np.array_equal(got.d_selector_wq, want.d_selector_wq)
    assert np.array_equal(got.d_selector_wk, want.d_selector_wk)
    assert np.array_equal(want.d_selector_wq, quiet.d_selector_wq)
    # without a policy such a target pushes the row down, as the reference has it; away from it there is nothing
    assert np.array_equal(free.d_selector_wq, quiet.d_selector_wq) == bool(away)


def learned_page(handle_policy, options):
    batch, rewards, (tok, role, sch, band, tg), off = learn_batch(16)
    w = weights()
    b = CudaBrainBackend(CFG, w, 0)
    try:
        if handle_policy is not None:
            b.set_policy(handle_policy)
        rep = BatchLearner(b, w).step(batch.frames, batch.records, off.data_ptr(), tok.data_ptr(), role.data_ptr(),
                                      sch.data_ptr(), band.data_ptr(), rewards, np.ones(batch.frames, bool),
                                      tg.data_ptr(), options=options)
        assert rep.update_applied and b.policy is handle_policy
        return w.page.copy()
    finally:
        b.destroy()


def test_a_learn_step_keeps_the_policy_the_handle_was_given():
    s, opts = Sampling(0.5, 0, 0.9), LearnOptions(learning_rate=2.0)
    free = learned_page(None, opts)
    asked = learned_page(None, LearnOptions(learning_rate=2.0, sampling=s))
    assert np.array_equal(learned_page(s, opts), asked) and not np.array_equal(free, asked)
    # the options' own policy goes before the handle's, for that step
    whole = learned_page(None, LearnOptions(learning_rate=2.0, sampling=Sampling()))
    assert np.array_equal(learned_page(s, LearnOptions(learning_rate=2.0, sampling=Sampling())), whole)
