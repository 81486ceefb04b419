"""Turns over cached banks: against a 64-bit restatement that quantises what the
cache holds, against themselves however the records are spread over turns, and
beside the uncached forward."""
import copy

import numpy as np
import pytest

from krystal_b200 import SessionBanks, abi, synth
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.frame import QUERY_BAND, pack_host_frame
from krystal_b200.policy import Sampling
from tests import cache_cases as ref
from tests import numpy_forward as NF

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

WL = synth.WORKLOADS["ragged_4096"]
CFG = synth.workload_config(WL)
W = synth.workload_weights(CFG, WL.vocab)


@pytest.fixture(scope="module")
def be():
    b = CudaBrainBackend(CFG, W, 0)
    yield b
    b.destroy()


def frame_records(seed, frames):
    """Record lists of a drawn batch: (bank records, questions) of each frame."""
    batch = synth.make_batch(WL, seed=seed, frames=frames)
    out = []
    for f in range(frames):
        g = batch.frame(f)
        recs = [dict(schemaId=int(g.schema_ids[s]), band=int(g.band_ids[s]),
                     tokens=[int(t) for t in g.token_ids[s * 8:(s + 1) * 8] if t]) for s in range(g.schema_ids.size)]
        out.append(([r for r in recs if r["band"] != QUERY_BAND], [r for r in recs if r["band"] == QUERY_BAND]))
    return out


def cached_p(bank, asks, fmt, mask=None):
    """The distributions in 64 bits, over projections rounded as the cache rounds them."""
    frame = pack_host_frame(bank + asks)
    h, hd = CFG.hidden_size, CFG.head_dim
    bare = copy.copy(W)
    bare.mixer = []  # without mixer blocks the query is the pooled one
    enc = NF.forward(CFG, bare, frame)
    bk, bv = enc["bank_keys"].reshape(-1, h), enc["bank_values"].reshape(-1, h)
    q = enc["query_output"].reshape(-1, h).astype(np.float64)
    heads = lambda x: ref.quantised(x.reshape(-1, CFG.head_count, hd), fmt)  # noqa: E731
    for blk in W.mixer:
        mk, mv = heads(NF.mm(bk, blk.wk, h, h)), heads(NF.mm(bv, blk.wv, h, h))
        mq = NF.mm(q, blk.wq, h, h).reshape(-1, CFG.head_count, hd)
        q = q + np.stack([ref.attend(x, mk, mv, hd ** -0.5)[0].reshape(-1) for x in mq])
        hid = np.maximum(q @ blk.w1.astype(np.float64).reshape(-1, h).T, 0)
        q = q + hid @ blk.w2.astype(np.float64).reshape(h, -1).T
    sk = ref.quantised(NF.mm(bk, W.selector.wk, h, h), fmt).astype(np.float64)
    s = (q @ W.selector.wq.astype(np.float64).reshape(h, h).T) @ sk.T / np.sqrt(h)
    if mask is not None:
        s = s + mask
    e = np.exp(s - s.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_a_turn_is_the_forward_over_quantised_banks(be, fmt):
    """Tolerance: the device's projections differ by 1e-6 of themselves, which may
    move a few of a frame's 60 000 codes by one step each. A step is 1 / 127 (i8)
    or 1 / 16 (e4m3) of a row's largest entry, about 3 of its standard deviations;
    it moves one of a score's 32 or 128 terms by that, a score by less than
    3 / 127 / sqrt(32) = 0.004 (0.033) of its spread and p by a quarter of it times
    the spread, about 1: 0.002 (0.02) for two codes in one row."""
    turns = frame_records(3, 3)
    banks = SessionBanks(be, 40, 600, fmt)
    got = banks.turn([(i, bank + asks) for i, (bank, asks) in enumerate(turns)])
    for (bank, asks), g, i in zip(turns, got, range(3)):
        want = cached_p(bank, asks, fmt)
        assert g.p.shape == want.shape
        assert np.abs(g.p - want).max() <= (0.002 if fmt == "i8" else 0.02)
        assert np.allclose(g.p.sum(1), 1, atol=1e-5)
        assert (g.index == g.p.argmax(1)).all()
        assert np.allclose(g.logp, np.log(g.p.max(1)), atol=1e-5)
        assert banks.length(i) == len(bank)


def test_turns_however_the_records_come(be):
    """All at once, or over several turns with questions between: the last
    answers are the same to the bit, and so for sessions in another order."""
    turns = frame_records(5, 4)
    asks = [a for _, a in turns]
    one = SessionBanks(be, 60, 600)
    for i, (bank, _) in enumerate(turns):
        one.turn([(i, bank)])
    want = one.turn([(i, a) for i, a in enumerate(asks)])
    many = SessionBanks(be, 60, 600)
    rng = np.random.default_rng(1)
    at = [0] * 4
    while any(a < len(b) for a, (b, _) in zip(at, turns)):
        some = []
        for i, (bank, a) in enumerate(turns):
            n = int(rng.choice([1, 5, 70]))
            new = bank[at[i]:at[i] + n]
            at[i] += len(new)
            if new:
                some.append((i, a[:1] + new if rng.random() < 0.5 else new))
        many.turn(some[::-1])
    got = many.turn([(i, a) for i, a in enumerate(asks)])
    for g, w in zip(got, want):
        assert np.array_equal(g.p, w.p) and np.array_equal(g.index, w.index)


def test_beside_the_uncached_forward(be):
    """The answers of an 8-bit bank: within a few percent of the forward's
    distributions, and the same where the forward's first has a clear lead."""
    turns = frame_records(7, 8)
    banks = SessionBanks(be, 80, 600)
    got = banks.turn([(i, bank + asks) for i, (bank, asks) in enumerate(turns)])
    from krystal_b200.frame import pack_frame_batch
    batch = pack_frame_batch([bank + asks for bank, asks in turns])
    res = be.forward_batch(batch)
    for f, g in enumerate(got):
        q, r = g.p.shape
        want = res["p"][int(res["p_off"][f]):][:q * r].reshape(q, r)
        assert np.abs(g.p - want).max() < 0.05
        top = np.sort(want, 1)
        clear = top[:, -1] - top[:, -2] > 0.1 if r > 1 else np.ones(q, bool)
        assert (g.index[clear] == want.argmax(1)[clear]).all()


def test_masks_draws_and_empty_banks(be):
    (bank, asks), (other, _) = frame_records(9, 2)
    banks = SessionBanks(be, 40, 600)
    q, r = len(asks), len(bank)
    rng = np.random.default_rng(2)
    mask = np.where(rng.random((q, r)) < 0.5, -1e30, rng.normal(0, 1, (q, r))).astype(np.float32)
    mask[:, 0] = 0
    mask[0] = -1e30
    u = rng.random(2 * q)
    got, empty = banks.turn([("a", bank + asks), ("b", asks)], [mask, np.zeros((q, 0))], u, Sampling(0.7, top_k=5))
    want = cached_p(bank, asks, "i8", mask.astype(np.float64))
    for i in range(q):
        if i == 0:
            assert got.index[0] == abi.KC_NO_SELECTION and (got.p[0] == 0).all() and got.logp[0] == -np.inf
            continue
        kept = np.flatnonzero(got.p[i])
        assert len(kept) == min(5, (mask[i] > -1e29).sum()) and (mask[i][kept] > -1e29).all()
        pi = want[i][kept] ** (1 / 0.7)
        assert np.abs(got.p[i][kept] - pi / pi.sum()).max() <= 0.005  # at 1 / 0.7 of the scores, over part of the mass
        assert got.index[i] == kept[min(int((np.cumsum(got.p[i][kept].astype(np.float64)) <= u[i]).sum()), len(kept) - 1)]
    assert empty.p.shape == (q, 0) and (empty.index == abi.KC_NO_SELECTION).all()
    # row limits, and a turn without questions
    banks.turn([("b", other)])
    t = np.linspace(0.5, 2.0, q).astype(np.float32)
    a = banks.turn([("b", asks)], sampling=Sampling(row_temperature=t))[0]
    w = cached_p(other, asks, "i8") ** (1 / t[:, None].astype(np.float64))
    assert np.abs(a.p - w / w.sum(1, keepdims=True)).max() <= 0.005


def test_sessions_come_and_go(be):
    turns = frame_records(11, 3)
    (bank, asks), (other, _), _ = turns
    banks = SessionBanks(be, 8, 300)
    first = banks.turn([("a", bank + asks)])[0]
    banks.turn([("a", other[:20])])
    assert banks.length("a") == len(bank) + 20
    banks.cut("a", len(bank))
    again = banks.turn([("a", asks)])[0]
    assert np.array_equal(again.p, first.p)
    free = len(banks.free)
    with pytest.raises(ValueError, match="more pages"):
        banks.turn([("b", (other * 9)[:300]), ("c", (other * 9)[:300])])
    with pytest.raises(ValueError, match="more than 300"):
        banks.turn([("a", (other * 9)[:300])])
    with pytest.raises(ValueError, match="one turn at a time"):
        banks.turn([("a", asks), ("a", asks)])
    with pytest.raises(ValueError, match="mask must be"):
        banks.turn([("a", asks)], [np.zeros(3)])
    with pytest.raises(ValueError, match="a mask per turn"):
        banks.turn([("a", asks)], [])
    with pytest.raises(ValueError, match="one entry per question"):
        banks.turn([("a", asks)], uniforms=[0.5] * 99)
    with pytest.raises(abi.KrystalCudaError, match="tokenRows"):  # refused on the device: nothing is kept of the turn
        banks.turn([("z", [dict(schemaId=1, band=0, tokens=[WL.vocab + 7])])])
    assert len(banks.free) == free and banks.length("z") == 0 and banks.length("a") == len(bank)
    assert np.array_equal(banks.turn([("a", asks)])[0].p, first.p)
    banks.drop("a")
    assert len(banks.free) == 8
    assert banks.turn([]) == []


def test_refusals(be):
    banks = SessionBanks(be, 4, 64)
    t = torch.zeros(64, dtype=torch.int64, device="cuda")
    p = t.data_ptr()
    from krystal_b200.cache import BankCache, page_table
    table = page_table(p, p, 1, 1, 64)
    call = lambda mixer=banks.mixer, selector=banks.selector, table=table, **kw: be.bank_turn(  # noqa: E731
        1, 1, p, p, p, p, p, mixer, selector, table, p, 1, **kw)
    with pytest.raises(ValueError, match="per mixer block"):
        call(mixer=banks.mixer[:1])
    wrong = BankCache(4, 2, 64)
    with pytest.raises(abi.KrystalCudaError, match="brain's heads"):
        call(mixer=[wrong] * len(banks.mixer))
    with pytest.raises(abi.KrystalCudaError, match="one head"):
        call(selector=wrong)
    with pytest.raises(abi.KrystalCudaError, match="a sequence a frame"):
        call(table=page_table(p, p, 2, 1, 64))
    with pytest.raises(abi.KrystalCudaError, match="KC_MAX_ROW"):
        call(table=page_table(p, p, 1, 5000))
    with pytest.raises(abi.KrystalCudaError, match="temperature"):
        call(sampling=Sampling(temperature=-1.0))
    for bad in (dict(max_length=0), dict(max_length=abi.KC_MAX_ROW + 1)):
        with pytest.raises(ValueError, match="records"):
            SessionBanks(be, 4, **bad)


def test_an_expired_wait_is_reported_and_the_turn_repeats(be):
    (bank, asks), = frame_records(13, 1)
    banks = SessionBanks(be, 10, 600)
    want = banks.turn([("a", bank + asks)])[0]
    banks.drop("a")
    be.inject_wait_expiry("gemm")
    with pytest.raises(abi.KrystalCudaError, match="wait expired"):
        banks.turn([("a", bank + asks)])
    assert banks.length("a") == 0
    assert np.array_equal(banks.turn([("a", bank + asks)])[0].p, want.p)


def test_activations_out_of_the_split_run_again():
    """Token rows 3000 times as large: the turn finds a scale at which they split."""
    big = synth.workload_weights(CFG, WL.vocab)
    big.embeddings *= np.float32(3000)
    b = CudaBrainBackend(CFG, big, 0)
    try:
        (bank, asks), = frame_records(15, 1)
        got = SessionBanks(b, 10, 600).turn([("a", bank + asks)])[0]
        assert np.isfinite(got.p).all() and np.allclose(got.p.sum(1), 1, atol=1e-5)
    finally:
        b.destroy()
