"""The handle's policy on the framework's paths: targets that it does not hold."""
import numpy as np
import pytest

from krystal_b200 import abi
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.policy import Sampling
from tests.test_gpu_policy_paths import CFG, frame_and_targets, weights

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
