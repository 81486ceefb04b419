"""Drawing, the drawn policy's gradient and clipping on the framework's own
paths: think, packed batches, the backward, the learn step, and all of them in
one go; and what each call refuses."""
import math
import threading
from dataclasses import replace

import numpy as np
import pytest

from krystal_b200 import BrainSession, abi, policy, synth
from krystal_b200.backend import CudaBrainBackend, MaskRule
from krystal_b200.frame import QUERY_BAND, pack_host_frame
from krystal_b200.learn import BatchLearner, LearnOptions
from krystal_b200.policy import GradList, Sampling
from tests import policy_cases as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

WL = synth.WORKLOADS["ragged_4096"]
CFG = synth.workload_config(WL)
HALF = 2.0 ** -24


def weights():
    return synth.workload_weights(CFG, WL.vocab)


@pytest.fixture(scope="module")
def be():
    b = CudaBrainBackend(CFG, weights(), 0)
    yield b
    b.destroy()


def f32(x):
    return float(np.float32(x))


def check_rows(p, got, blocks, s, u):
    """Every row of a batch's draw against the plain form on the p it was drawn from."""
    q = 0
    for at, r in blocks:
        row = ref.policy(p[at:at + r], f32(s.temperature), s.top_k, f32(s.top_p), f32(s.min_p), kind="p")
        want = np.zeros(r)
        want[row[0]] = row[1]
        j, lp = ref.draw(row, None if u is None else u[q])
        assert int(np.int32(got["index"][q])) == j and int(got["kept"][q]) == row[0].size
        assert (np.abs(got["p"][at:at + r] - want) <= 1.001 * HALF * want + 2.0 ** -149).all()
        assert got["logp"][q] == lp or abs(got["logp"][q] - lp) <= 1.001 * HALF * abs(lp) + 2e-12
        q += 1
    assert q == len(got["index"])


def blocks_of(res):
    out = []
    for f in range(len(res["q_off"]) - 1):
        nq = int(res["q_off"][f + 1] - res["q_off"][f])
        for i in range(nq):
            r = int(res["p_off"][f + 1] - res["p_off"][f]) // nq
            out.append((int(res["p_off"][f]) + i * r, r))
    return out


@pytest.mark.parametrize("precision", ["certified", "exact"])
def test_packed_batch_draws(be, precision):
    be.set_precision(precision)
    try:
        batch = synth.make_batch(WL, seed=5, frames=40 if precision == "certified" else 6)
        nq = int((batch.band_ids == QUERY_BAND).sum())
        rule, u = MaskRule(*synth.make_rule(batch, seed=6)), np.random.default_rng(7).random(nq)
        s = Sampling(0.6, 20, 0.9, 0.01)
        plain = be.forward_batch(batch, rule=rule)
        drawn = be.forward_batch(batch, rule=rule, sampling=s, uniforms=u)
        check_rows(plain["p"], drawn, blocks_of(plain), s, u)
        # chosen again from the resident batch, under other masks and policies
        open_p = be.select_batch()
        again = be.select_batch(sampling=Sampling(1.0, 0, 0.5), uniforms=u)
        check_rows(open_p["p"], again, blocks_of(open_p), Sampling(1.0, 0, 0.5), u)
        d = be.draw_batch(Sampling(temperature=0.0))
        assert np.array_equal(d.index, open_p["index"]) and (d.kept == 1).all()
        rows = be.draw_batch(Sampling(row_top_k=np.arange(nq) % 5 + 1, row_temperature=np.full(nq, 2.0)), u)
        assert (rows.kept <= np.arange(nq) % 5 + 1).all()
        # the resident batch is still the selection's
        assert np.array_equal(be.select_batch()["p"], open_p["p"])
    finally:
        be.set_precision("certified")


def test_a_batch_keeps_its_results_beside_a_draw(be):
    batch = synth.make_batch(WL, seed=8, frames=16)
    before = be.forward_batch(batch)
    be.forward_batch(batch, sampling=Sampling(0.5))
    after = be.forward_batch(batch)
    assert np.array_equal(before["p"], after["p"]) and np.array_equal(before["index"], after["index"])


def test_think_draws_from_the_policy():
    rng = np.random.default_rng(4)
    session = BrainSession(np.arange(4096, dtype=np.uint32) % 64, seed=3)
    try:
        recs = [dict(schemaId=int(rng.integers(0, 9)), tokens=[int(t) for t in rng.integers(1, 4000, 5)])
                for _ in range(30)] + [dict(query=True, tokens=[7]), dict(query=True, tokens=[9])]
        thought = session.consider(recs)
        allows = lambda q, slot: slot % 3 != 0  # noqa: E731
        base = thought.choose(allows)
        for s, u in ((Sampling(0.7, 6), [0.2, 0.95]), (Sampling(top_p=0.4), [0.5, 0.01]), (Sampling(temperature=0), None)):
            got = thought.choose(allows, None if u is None else (lambda q: u[q]), s)
            bank = thought.frame.active.bank_records
            for q, (a, b) in enumerate(zip(base.selections, got.selections)):
                row = ref.policy(a.distribution, f32(s.temperature), s.top_k, f32(s.top_p), f32(s.min_p), kind="p")
                j, _ = ref.draw(row, None if u is None else u[q])
                want = np.zeros(len(bank))
                want[row[0]] = row[1]
                assert b.record == int(bank[j]) and allows(q, b.record)
                assert np.abs(b.distribution - want).max() <= 1.001 * HALF
                assert b.probability == b.distribution[j]
        again = session.think(recs, allows=allows, sampling=Sampling(temperature=0))
        assert [s.record for s in again.selections] == [s.record for s in base.selections]
    finally:
        session.destroy()


def frame_and_targets(seed, away):
    batch = synth.make_batch(WL, seed=seed, frames=1)
    g = batch.frame(0)
    from krystal_b200.frame import HostFrame, compile_active_frame
    frame = HostFrame(g, compile_active_frame(g), g.schema_ids.size)
    rng = np.random.default_rng(seed)
    q, r = frame.active.query_records.size, frame.active.bank_records.size
    targets = rng.integers(0, r, q).astype(np.uint32)
    targets[0] = abi.KC_NO_TARGET
    if away and q > 1:
        targets[1] |= abi.KC_AWAY_TARGET
    return frame, q, r, targets


@pytest.mark.parametrize("s", [Sampling(), Sampling(0.5), Sampling(0.8, 9), Sampling(1.7, 0, 0.6, 0.2)])
@pytest.mark.parametrize("away", [False, True])
def test_backward_differentiates_the_policy(be, s, away):
    """dWq and dWk against a 64-bit form from the encoded frame. The policy is
    taken from the stored p (2^-24), raised to 1/T <= 2; dscore, the projected
    gradient and the result are stored in f32 and so is every factor: fewer
    than 16 roundings of 2^-24 of the sum of magnitudes."""
    w = weights()
    frame, q, r, targets = frame_and_targets(21, away)
    enc = be.encode(frame)
    h = CFG.hidden_size
    plain = be.backward(frame, targets=targets)
    top = [int(np.argmax(plain.policy[i * r:(i + 1) * r])) for i in range(q)]
    targets[2::2] = np.array(top, np.uint32)[2::2]  # likely answers, which a cut policy holds
    be.set_policy(s)
    try:
        got = be.backward(frame, targets=targets)
    finally:
        be.set_policy(None)
    assert np.array_equal(got.policy, plain.policy)
    t = f32(s.temperature)
    ds = np.zeros((q, r))
    for i in range(q):
        if targets[i] == abi.KC_NO_TARGET:
            continue
        at = int(targets[i] & 0x7fffffff)
        j, pi, _ = ref.policy(got.policy[i * r:(i + 1) * r], t, s.top_k, f32(s.top_p), f32(s.min_p), kind="p")
        if at not in j:
            continue
        row = np.zeros(r)
        row[j] = pi
        one = (np.arange(r) == at).astype(float)
        sc = row[at] / max(1 - row[at], 1e-6)
        full = sc * (one - row) if targets[i] & abi.KC_AWAY_TARGET else row - one
        ds[i, j] = full[j] / t
    assert (ds != 0).any()
    qo, bk = enc.query_output.astype(float).reshape(q, h), enc.bank_keys.astype(float).reshape(r, h)
    wq, wk = w.selector.wq.astype(float).reshape(h, h), w.selector.wk.astype(float).reshape(h, h)
    scale = 1 / math.sqrt(h)
    kp, qp = bk @ wk.T, qo @ wq.T
    for g, d, x in ((got.d_selector_wq, scale * ds @ kp, qo), (got.d_selector_wk, scale * ds.T @ qp, bk)):
        mag = (scale * np.abs(ds) @ np.abs(kp) if x is qo else scale * np.abs(ds).T @ np.abs(qp)).T @ np.abs(x)
        assert (np.abs(g.reshape(h, h) - d.T @ x) <= 16 * HALF * mag + 1e-30).all()
    # without a policy the backward is what it was
    back = be.backward(frame, targets=targets)
    be.set_policy(Sampling())
    be.set_policy(None)
    assert np.array_equal(back.d_selector_wq, be.backward(frame, targets=targets).d_selector_wq)


def learn_batch(frames=24):
    batch = synth.make_batch(synth.WORKLOADS["learn_1024"], seed=31, frames=frames)
    targets, rewards = synth.make_learn_inputs(batch)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).cuda()  # noqa: E731
    arrays = [dev(a) for a in (batch.token_ids, batch.field_roles, batch.schema_ids, batch.band_ids, targets)]
    off = torch.from_numpy(batch.rec_off.astype(np.int64)).cuda()
    return batch, rewards, arrays, off


def learn_once(options, frames=24, page=None):
    batch, rewards, (tok, role, sch, band, tg), off = learn_batch(frames)
    w = weights()
    b = CudaBrainBackend(CFG, w, 0)
    try:
        rep = BatchLearner(b, w).step(batch.frames, batch.records, off.data_ptr(), tok.data_ptr(), role.data_ptr(),
                                      sch.data_ptr(), band.data_ptr(), rewards, np.ones(batch.frames, bool),
                                      tg.data_ptr(), options=options)
        assert b.policy is None  # the step puts the handle's policy back
        return rep, w.page.copy()
    finally:
        b.destroy()


@pytest.mark.parametrize("extra", [{}, dict(unfreeze_pool=True, unfreeze_tokens=True, token_rate=0.3)])
def test_learn_step_clips_the_actors_update(extra):
    opts = LearnOptions(learning_rate=2.0, **extra)
    start = weights().page.astype(float)
    rep, free = learn_once(opts)
    assert rep.update_applied and rep.update_norm is None
    lay = weights().layout
    critic = slice(lay.total - 3 * CFG.hidden_size, lay.total)  # the value head: the critic's own rate
    actor = np.ones(start.size, bool)
    actor[critic] = False
    step = (start - free)[actor]
    norm = float(np.sqrt((step ** 2).sum()))
    # a weight is stored in f32: its step is off by at most 2^-24 of its size, the norm by that of all of them
    slack = HALF * float(np.sqrt((start[actor][step != 0] ** 2).sum() + (free[actor][step != 0] ** 2).sum())) + 1e-12
    rep2, same = learn_once(replace(opts, max_update_norm=norm * 2))
    assert abs(rep2.update_norm - norm) <= slack
    assert np.abs(same - free).max() <= 1e-6 if extra else np.array_equal(same, free)
    rep3, cut = learn_once(replace(opts, max_update_norm=norm / 5))
    assert abs(rep3.update_norm - norm) <= slack
    want = start[actor] - step * (norm / 5 / rep3.update_norm)
    assert (np.abs(cut[actor] - want) <= 2.5 * HALF * (np.abs(want) + np.abs(start[actor])) + 1e-9).all()
    assert np.array_equal(cut[critic], free[critic])


def test_learn_step_under_a_policy():
    """Learning under a policy that cuts nothing is learning as it was; under a
    tempered one the selector moves otherwise, by the policy's gradient."""
    opts = LearnOptions(learning_rate=2.0)
    _, free = learn_once(opts)
    _, same = learn_once(replace(opts, sampling=Sampling()))
    _, cut = learn_once(replace(opts, sampling=Sampling(0.5, 0, 0.9)))
    start = weights().page
    moved = np.abs(free - start).max()
    assert np.abs(same - free).max() <= 1e-4 * moved + 2 * HALF * np.abs(start).max()
    assert np.abs(cut - free).max() > 1e-2 * moved
    with pytest.raises(abi.KrystalCudaError, match="temperature 0"):
        learn_once(replace(opts, sampling=Sampling(temperature=0.0)))


def test_all_together_on_one_stream(be):
    """A host's exploration round: a device batch, answers drawn from its
    distributions, their loss and gradient by the scores, a linear readout's
    gradient clipped; torch's work and the library's in one stream's order."""
    batch = synth.make_batch(WL, seed=41, frames=32)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int32)).cuda()  # noqa: E731
    tok, role, sch, band = (dev(a) for a in (batch.token_ids, batch.field_roles, batch.schema_ids, batch.band_ids))
    off = torch.from_numpy(batch.rec_off.astype(np.int64)).cuda()
    nq = int((batch.band_ids == QUERY_BAND).sum())
    host = be.forward_batch(batch)
    prev, side = be.stream_ptr(), torch.cuda.Stream()
    torch.cuda.synchronize()
    be.set_stream(side.cuda_stream)
    try:
        with torch.cuda.stream(side):
            res = be.forward_batch_device(batch.frames, batch.records, off.data_ptr(), tok.data_ptr(),
                                          role.data_ptr(), sch.data_ptr(), band.data_ptr())
            s = Sampling(0.8, 30, 0.95)
            u = torch.rand(nq, dtype=torch.float64, device="cuda")
            idx = torch.zeros(nq, dtype=torch.int32, device="cuda")
            pi, logp = torch.zeros(res.total_p, device="cuda"), torch.zeros(nq, device="cuda")
            be.draw(policy.ragged_rows(res.p, "f32", nq, batch.frames, res.q_off, res.p_off, 256, "p"), s,
                    u.data_ptr(), index=idx.data_ptr(), logp=logp.data_ptr(), p=pi.data_ptr())
            p = torch.from_numpy(host["p"]).cuda()
            x = torch.log(p)  # scores with the same policy
            adv = torch.randn(nq, device="cuda")
            lp2, grad = torch.zeros(nq, device="cuda"), torch.zeros_like(x)
            rows = policy.ragged_rows(x.data_ptr(), "f32", nq, batch.frames, res.q_off, res.p_off, 256)
            be.policy_loss(rows, s, idx.data_ptr(), adv.data_ptr(), 0.0, logp=lp2.data_ptr(), grad=grad.data_ptr())
            feats = torch.randn(x.numel(), 8, device="cuda")
            w = (feats.t() @ grad).contiguous()
            b = grad.sum().reshape(1)
            norm = torch.zeros(2, dtype=torch.float64, device="cuda")
            lst = GradList([w, b])
            before = torch.cat([w, b]).double()
            be.clip_grads(lst, 0.1, norm.data_ptr())
        torch.cuda.synchronize()
    finally:
        be.set_stream(prev)
    hu, a = u.cpu().numpy(), adv.double().cpu().numpy()
    got_pi, got_g = pi.cpu().numpy(), grad.double().cpu().numpy()
    for i, (at, r) in enumerate(blocks_of(host)):
        row = ref.policy(host["p"][at:at + r], f32(0.8), 30, f32(0.95), kind="p")
        j, lp = ref.draw(row, hu[i])
        assert int(idx[i]) == j
        assert abs(float(logp[i]) - lp) <= 1.001 * HALF * abs(lp) + 2e-12
        # log p rounded to f32: 2^-24 of up to 20, over T
        assert abs(float(lp2[i]) - lp) <= 3 * 20 * HALF / 0.8
        g = np.zeros(r)
        g[row[0]] = a[i] * row[1]
        g[j] -= a[i]
        assert np.abs(got_g[at:at + r] - g / f32(0.8)).max() <= 4 * 20 * HALF / 0.64 * abs(a[i])
    assert float(norm[0]) == pytest.approx(float(before.norm()), rel=1e-9)
    assert float(torch.cat([w, b]).double().norm()) == pytest.approx(min(0.1, float(before.norm())), rel=1e-6)


def test_two_threads_share_a_handle(be):
    rng = np.random.default_rng(9)
    v = [torch.from_numpy(rng.normal(size=(50, 300)).astype(np.float32)).cuda() for _ in range(2)]
    u = torch.rand(50, dtype=torch.float64, device="cuda")
    want, got = [], [[], []]
    s = Sampling(0.9, 10)
    for x in v:
        idx = torch.zeros(50, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        be.draw(policy.dense_rows(x.data_ptr(), "f32", 50, 300), s, u.data_ptr(), index=idx.data_ptr())
        be.synchronize()
        want.append(idx.clone())

    def work(t):
        for _ in range(30):
            idx = torch.zeros(50, dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            be.draw(policy.dense_rows(v[t].data_ptr(), "f32", 50, 300), s, u.data_ptr(), index=idx.data_ptr())
            be.synchronize()
            got[t].append(idx)

    ts = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert all(len(g) == 30 and all(torch.equal(x, w) for x in g) for g, w in zip(got, want))


def refused(match, call, *a, **k):
    with pytest.raises(abi.KrystalCudaError, match=match):
        call(*a, **k)


def test_refusals(be):
    v = torch.zeros(64, device="cuda")
    i = torch.zeros(8, dtype=torch.int32, device="cuda")
    p, ip = v.data_ptr(), i.data_ptr()
    rows = policy.dense_rows(p, "f32", 2, 8)
    ok = Sampling()
    refused("at least one output", be.draw, rows, ok)
    for s, m in ((Sampling(-1.0), "temperature"), (Sampling(math.nan), "temperature"), (Sampling(math.inf), "temperature"),
                 (Sampling(top_p=-0.1), "top_p"), (Sampling(top_p=math.nan), "top_p"), (Sampling(min_p=1.5), "min_p"),
                 (Sampling(min_p=math.nan), "min_p"), (Sampling(row_top_k=ip + 2), "row limits")):
        refused(m, be.draw, rows, s, index=ip)
    bad = [(policy.dense_rows(p, "f64", 2, 8), "f32, f16 or bf16"), (policy.dense_rows(p, "f16", 2, 8, kind="p"), "f32"),
           (policy.dense_rows(0, "f32", 2, 8), "no values"), (policy.dense_rows(p + 2, "f32", 2, 8), "aligned"),
           (policy.dense_rows(p + 1, "f16", 2, 8), "aligned"), (policy.dense_rows(p, "f32", 2, 8, 7), "row_pitch"),
           (policy.dense_rows(p, "f32", 2, abi.KC_MAX_ROW + 1), "KC_MAX_ROW"),
           (policy.ragged_rows(p, "f32", 2, 1, ip, 0), "p_off"), (policy.ragged_rows(p, "f32", 2, 1, ip + 4, ip), "8-byte")]
    for r, m in bad:
        refused(m, be.draw, r, ok, index=ip)
    odd = policy.dense_rows(p, "f32", 2, 8)
    odd.kind = 5
    refused("kind", be.draw, odd, ok, index=ip)
    refused("pitch", be.draw, rows, ok, p=p, p_pitch=7)
    refused("8-byte", be.draw, rows, ok, p + 4, index=ip)
    refused("4-byte", be.draw, rows, ok, index=ip + 2)
    refused("at least one output", be.policy_loss, rows, ok, ip, p)
    refused("actions", be.policy_loss, rows, ok, 0, p, loss=p)
    refused("temperature 0", be.policy_loss, rows, Sampling(temperature=0.0), ip, p, loss=p)
    refused("scores", be.policy_loss, policy.dense_rows(p, "f32", 2, 8, kind="p"), ok, ip, p, loss=p)
    refused("entropy_coef", be.policy_loss, rows, ok, ip, p, math.nan, loss=p)
    refused("aligned", be.policy_loss, rows, ok, ip, p + 2, loss=p)
    refused("temperature 0", be.set_policy, Sampling(temperature=0.0))
    refused("scalar", be.set_policy, Sampling(row_top_k=ip))
    assert be.policy is None
    with pytest.raises(ValueError, match="rows of one length"):
        be.draw_rows(np.zeros(7), 2, ok)
    with pytest.raises(ValueError, match="uniforms"):
        be.draw_rows(np.zeros(8), 2, ok, uniforms=[0.5])
    fresh = CudaBrainBackend(CFG, weights(), 0)
    try:
        with pytest.raises(RuntimeError, match="forward_batch"):
            fresh.draw_batch(ok)
        batch = synth.make_batch(WL, seed=3, frames=4)
        fresh.forward_batch(batch)
        fresh.sync(weights())
        refused("resident", fresh.draw_batch, ok)
    finally:
        fresh.destroy()
    # nothing to do is no error, and writes nothing
    be.draw(policy.dense_rows(0, "f32", 0, 8), ok, index=ip)
    i.fill_(-5)
    torch.cuda.synchronize()
    be.draw(policy.dense_rows(0, "f32", 3, 0), ok, index=ip)  # rows without entries
    be.synchronize()
    assert i.tolist() == [-1] * 3 + [-5] * 5
    d = be.draw_rows(np.zeros(0), 0, ok)
    assert d.index.size == 0


def test_rows_written_over_themselves_and_too_many_rows_are_refused(be):
    v = torch.zeros(64, device="cuda")
    i = torch.zeros(8, dtype=torch.int32, device="cuda")
    p, ip, ok = v.data_ptr(), i.data_ptr(), Sampling()
    wide = policy.dense_rows(p, "f32", 2, 8, 10)
    refused("one pitch", be.draw, wide, ok, p=p)
    refused("one pitch", be.draw, policy.dense_rows(p, "f16", 2, 8), ok, p=p)
    refused("one pitch", be.policy_loss, wide, ok, ip, p, grad=p)
    refused("2147483647", be.draw, policy.dense_rows(p, "f32", 2 ** 31, 1), ok, index=ip)
    be.draw(wide, ok, index=ip, p=p, p_pitch=10)
    be.synchronize()
