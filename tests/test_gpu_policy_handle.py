"""The handle's policy on the framework's paths: targets that it does not hold,
the learn step's, and what the certified path's draws keep of its promise."""
import numpy as np
import pytest

from krystal_b200 import abi, synth
from krystal_b200.backend import CudaBrainBackend, MaskRule
from krystal_b200.frame import QUERY_BAND
from krystal_b200.learn import BatchLearner, LearnOptions
from krystal_b200.policy import Sampling
from tests.test_gpu_policy_paths import CFG, WL, blocks_of, frame_and_targets, learn_batch, weights

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


def at_precision(be, precision, call):
    be.set_precision(precision)
    try:
        return call()
    finally:
        be.set_precision("certified")


@pytest.mark.parametrize("again", [False, True])
def test_certified_draws_of_the_whole_distribution_match_the_exact_paths(be, again):
    """Uniforms between an edge of the fast path's running p and the exact
    path's: drawn from either, the answers differ."""
    batch = synth.make_batch(WL, seed=15, frames=24)
    rule = MaskRule(*synth.make_rule(batch, seed=16))
    fast = at_precision(be, "fast", lambda: be.forward_batch(batch, rule=rule))
    exact = at_precision(be, "exact", lambda: be.forward_batch(batch, rule=rule))
    u = np.full(int((batch.band_ids == QUERY_BAND).sum()), 0.5)
    tight = 0
    for i, (at, r) in enumerate(blocks_of(exact)):
        run = [np.cumsum(x["p"][at:at + r].astype(np.float64)) for x in (fast, exact)]
        if run[1][-1] == 0:
            continue
        run = [c / c[-1] for c in run]
        e = int(np.argmax(np.abs(run[0] - run[1])))
        if abs(run[0][e] - run[1][e]) > 1e-9:
            u[i] = (run[0][e] + run[1][e]) / 2
            tight += 1
    assert tight > 50

    def drawn(precision):
        if again:
            be.forward_batch(batch)
            return be.select_batch(rule=rule, uniforms=u, sampling=Sampling())
        return be.forward_batch(batch, rule=rule, uniforms=u, sampling=Sampling())

    by_fast, by_exact, certified = (at_precision(be, x, lambda: drawn(x)) for x in ("fast", "exact", "certified"))
    assert (by_fast["index"] != by_exact["index"]).sum() > tight // 2
    assert np.array_equal(certified["index"], by_exact["index"])
    assert np.array_equal(certified["kept"], by_exact["kept"])


def test_certified_answers_without_uniforms_are_the_exact_paths(be):
    batch = synth.make_batch(WL, seed=17, frames=24)
    got = be.forward_batch(batch, sampling=Sampling(0.6, 12, 0.8))
    want = at_precision(be, "exact", lambda: be.forward_batch(batch, sampling=Sampling(0.6, 12, 0.8)))
    assert np.array_equal(got["index"], want["index"])


def test_uniforms_of_another_length_are_refused(be):
    batch = synth.make_batch(WL, seed=18, frames=3)
    nq = int((batch.band_ids == QUERY_BAND).sum())
    be.forward_batch(batch)
    for s in (Sampling(), Sampling(0.5)):
        for n in (0, nq - 1, nq + 1):
            for call in (lambda **k: be.forward_batch(batch, **k), be.select_batch):
                with pytest.raises(ValueError, match="uniforms"):
                    call(uniforms=np.full(n, 0.5), sampling=s)
