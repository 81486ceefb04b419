"""Drawing from a tempered and cut policy, and the drawn policy's loss and
gradient, against plain 64-bit forms.

Tolerances. The kernels' weights are 64-bit and a result is rounded once, so
an f32 result lies within half a step, 2^-24 of its value; what the 64-bit
arithmetic adds (below 1e-12 of the value for the row lengths here) is
covered by a factor of 1.001, values below f32's normal range by 2^-149. A
log probability is a difference of numbers up to 700, exact to about 1e-12.
Gradients: half a step of their type of the value; the terms that cancel in
it are 64-bit, below 1e-12 of the largest.

Where nothing is cut, the loss works in f32 (whole_tolerances). A weight 2^u
is off by ex2's 2^-22 and by one rounding of u, |u| ln 2 2^-24, of itself; a
partial sum has at most 16 terms, 2^-20. The mean of |u| under pi is at most
L = log2 n (H <= ln n), so Z is within 2^-20 + 2^-22 + 0.7 2^-24 L < 2^-19 of
itself for L <= 18, and log Z within 2^-18. log pi(a) adds its own u's
rounding, 2^-24 of it; H = ln 2 (log2 Z - S / Z) has S / Z within 2^-18 of
at most L + 2, and 0.7 2^-24 E[u^2] <= 2^-24 (L + 2)^2 < 2^-19 (L + 2) on top.
A gradient is pi's error of its terms, and H's.
"""
import numpy as np
import pytest

from krystal_b200 import abi, policy, synth
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from tests import policy_cases as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CUTS = [dict(), dict(temperature=0.7, top_p=0.9), dict(temperature=1.6, top_k=5),
        dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.02), dict(min_p=0.1), dict(top_p=0.3), dict(top_k=1),
        dict(temperature=0.0), dict(temperature=2.0, top_k=1000, top_p=0.999), dict(top_p=0.0), dict(min_p=1.0)]
LENGTHS = [1, 2, 31, 33, 129, 249, 256, 257, 1020, 1024, 1025, 4096, 8185, 8193, 20001, 32768, 40003, 262128]


@pytest.fixture(scope="module")
def be():
    cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
    b = CudaBrainBackend(cfg, create_brain_forward_weights(cfg, 1337), 0)
    yield b
    b.destroy()


def on_gpu(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t.to(dtype) if dtype is not None else t


def scores(rng, rows, n, dtype, masked=0.1):
    """Rows of scores in their type: masked entries of every sort, one row in
    five with everything masked."""
    v = rng.normal(0, 2.5, (rows, n)).astype(np.float32)
    odd = np.array([-np.inf, np.nan, -1e30, np.finfo(np.float32).min], np.float32)
    hit = rng.random((rows, n)) < masked
    v[hit] = odd[rng.integers(0, odd.size, int(hit.sum()))]
    if rows > 4:
        v[4::5] = odd[rng.integers(0, odd.size, v[4::5].shape)]
    t = torch.from_numpy(v).to(TYPES[dtype])
    if dtype == "f16":  # the lowest value as a mask
        t[torch.from_numpy(hit) & torch.isinf(t)] = -65504.0
    return t


def wide(t):
    return t.double().numpy()


def sampling(cut):
    return policy.Sampling(**cut)


def limits(cut):
    """A cut's limits as the library holds them: f32."""
    f = lambda x: float(np.float32(x))  # noqa: E731
    return (f(cut.get("temperature", 1.0)), int(cut.get("top_k", 0)), f(cut.get("top_p", 1.0)), f(cut.get("min_p", 0.0)))


def near(got, want, half, tiny=0.0):
    """Within `half` of the value, or both infinite the same way."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    got, want, tiny = got[~inf], want[~inf], np.broadcast_to(tiny, want.shape)[~inf]
    bad = ~(np.abs(got - want) <= half * 1.001 * np.abs(want) + tiny)
    assert not bad.any(), (got[bad][:4], want[bad][:4])


class Place:
    """A device matrix at an offset and a pitch inside a buffer whose other
    elements must stay as they are."""

    def __init__(self, rows, n, pitch, offset, dtype, fill):
        self.buf = torch.full((offset + rows * pitch + 9,), fill, dtype=dtype, device="cuda")
        self.fill, self.shape, self.pitch, self.offset = fill, (rows, n), pitch, offset

    def view(self):
        rows, n = self.shape
        return self.buf[self.offset:self.offset + rows * self.pitch].view(rows, self.pitch)[:, :n]

    def ptr(self):
        return self.buf.data_ptr() + self.offset * self.buf.element_size()

    def rest_untouched(self):
        b = self.buf.clone()
        rows, n = self.shape
        b[self.offset:self.offset + rows * self.pitch].view(rows, self.pitch)[:, :n] = self.fill
        return bool((b == self.fill).all())


def check_draw(be, v, dtype, cut, u, kind="scores", pitch=0, offset=0):
    rows, n = v.shape
    t, k, p, mp = limits(cut)
    place = Place(rows, n, pitch or n, offset, v.dtype, 7.0)
    place.view().copy_(v)
    out = Place(rows, n, (pitch or n) + 3, offset, torch.float32, 9.0)
    idx = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    kept, logp = idx.clone(), torch.full((rows,), 3.0, device="cuda")
    du = on_gpu(u) if u is not None else None
    torch.cuda.synchronize()
    be.draw(policy.dense_rows(place.ptr(), dtype, rows, n, place.pitch, kind), sampling(cut),
            du.data_ptr() if du is not None else None, index=idx.data_ptr(), kept=kept.data_ptr(),
            logp=logp.data_ptr(), p=out.ptr(), p_pitch=out.pitch)
    be.synchronize()
    got_p = out.view().cpu().numpy()
    assert out.rest_untouched()
    for i in range(rows):
        row = ref.policy(wide(v[i]), t, k, p, mp, kind, dtype == "f16")
        want = np.zeros(n)
        want[row[0]] = row[1]
        at, lp = ref.draw(row, None if u is None else u[i])
        assert int(kept[i]) == row[0].size, (i, cut)
        assert int(idx[i]) == at, (i, cut)
        near(got_p[i], want, HALF["f32"], TINY["f32"])
        near([float(logp[i])], [lp], HALF["f32"], 2e-12)
    return idx, got_p


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_draw_every_length_and_type(be, n, dtype):
    rng = np.random.default_rng(n)
    rows = 6 if n <= 4096 else 2
    for c, cut in enumerate(CUTS if n <= 4096 else CUTS[:5]):
        u = rng.random(rows) if c % 4 else None
        check_draw(be, scores(rng, rows, n, dtype), dtype, cut, u, pitch=n + (c % 3), offset=c % 5)


@pytest.mark.parametrize("n", [1, 7, 130, 700, 4096])
@pytest.mark.parametrize("cut", CUTS)
def test_draw_from_probabilities(be, n, cut):
    rng = np.random.default_rng(n)
    x = rng.normal(0, 3, (5, n))
    p = np.exp(x - x.max(1, keepdims=True))
    p[rng.random((5, n)) < 0.3] = 0
    p[3] = 0
    p[4, :1] = np.nan
    p = (p / np.maximum(np.nansum(p, 1, keepdims=True), 1e-20)).astype(np.float32)
    check_draw(be, torch.from_numpy(p), "f32", cut, rng.random(5), kind="p")


def test_borders_and_ties(be):
    flat = torch.zeros(4, 10)
    for cut, want in ((dict(top_p=0.5), 5), (dict(top_k=3), 3), (dict(top_k=10), 10), (dict(top_k=11), 10),
                      (dict(min_p=1.0), 10), (dict(top_k=4, top_p=0.5), 2), (dict(top_p=0.51), 6)):
        idx, p = check_draw(be, flat, "f32", cut, np.array([0.0, 0.3, 0.999999, 1.0 - 2.0 ** -53]))
        assert (p[0] > 0).sum() == want and p[0, want - 1] > 0  # ties stay with the lowest index
    # the border of min_p and of top_p in exact values
    half = torch.tensor([[0.5, 0.25, 0.125, 0.125]])
    assert check_draw(be, half, "f32", dict(min_p=0.25), np.array([0.9]), kind="p")[1].astype(bool).sum() == 4
    assert check_draw(be, half, "f32", dict(min_p=0.26), np.array([0.9]), kind="p")[1].astype(bool).sum() == 2
    assert check_draw(be, half, "f32", dict(top_p=0.75), np.array([0.9]), kind="p")[1].astype(bool).sum() == 2
    # a uniform on an edge belongs to the entry behind it; u outside [0, 1) is clamped
    for u, want in ((0.0, 0), (0.5, 1), (0.75, 2), (0.875, 3), (1.0, 3), (-1.0, 0), (2.0, 3)):
        assert int(check_draw(be, half, "f32", dict(), np.array([u]), kind="p")[0][0]) == want
    # +-0 are one value; signed extremes, and values far below the largest
    odd = torch.tensor([[0.0, -0.0, 0.0, -1e28, 3e38, float("inf")], [-0.0, 0.0, -5.0, -300.0, -699.0, -701.0]])
    for cut in (dict(top_k=2), dict(), dict(top_p=0.4), dict(temperature=0.0)):
        check_draw(be, odd, "f32", cut, np.array([0.1, 0.7]))


def test_values_over_the_whole_range(be):
    """Rows whose values span the type: the halving ends for any of them."""
    rng = np.random.default_rng(5)
    bits = rng.integers(0, 2 ** 32, (6, 500), dtype=np.uint64).astype(np.uint32)
    v = torch.from_numpy(bits.view(np.float32).copy())
    for cut in (dict(top_k=37), dict(top_p=0.5), dict(temperature=1e30, top_p=0.5), dict(temperature=1e30, top_k=99)):
        check_draw(be, v, "f32", cut, rng.random(6))
    p = torch.from_numpy(np.abs(bits.view(np.float32)).copy())
    check_draw(be, torch.nan_to_num(p, 0, 0, 0), "f32", dict(top_p=0.9), rng.random(6), kind="p")
    check_draw(be, torch.nan_to_num(p, 0, 0, 0), "f32", dict(temperature=1.5, top_k=50), rng.random(6), kind="p")


def ragged(rng, frames, q_hi, r_hi, dtype):
    """A packed batch with frames without questions and frames without a bank."""
    q, r = rng.integers(0, q_hi + 1, frames), rng.integers(0, r_hi + 1, frames)
    q[0], r[0], q[-1], r[-1] = 0, 5, q_hi, r_hi
    if frames > 3:
        r[2], q[2] = 0, 3
    q_off = np.concatenate([[0], np.cumsum(q)]).astype(np.uint64)
    p_off = np.concatenate([[0], np.cumsum(q * r)]).astype(np.uint64)
    v = scores(rng, 1, max(1, int(p_off[-1])), dtype)[0][:int(p_off[-1])]
    where = [(int(p_off[f]) + i * int(r[f]), int(r[f])) for f in range(frames) for i in range(int(q[f]))]
    return q_off, p_off, v, where


@pytest.mark.parametrize("frames,q_hi,r_hi", [(1, 4, 9), (5, 3, 40), (40, 16, 240), (33, 2, 900), (3, 5, 4096),
                                              (1100, 2, 11)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_packed_batches(be, frames, q_hi, r_hi, dtype):
    rng = np.random.default_rng(frames + r_hi)
    if frames == 1:
        q_off, p_off = np.array([0, q_hi], np.uint64), np.array([0, q_hi * r_hi], np.uint64)
        v = scores(rng, 1, q_hi * r_hi, dtype)[0]
        where = [(i * r_hi, r_hi) for i in range(q_hi)]
    else:
        q_off, p_off, v, where = ragged(rng, frames, q_hi, r_hi, dtype)
    rows, spare, total = len(where), 5, v.numel()
    cut = dict(temperature=0.8, top_k=60, top_p=0.92)
    t, k, p, mp = limits(cut)
    u = rng.random(rows + spare)
    dv, dq, dp, du = v.cuda(), on_gpu(q_off.view(np.int64)), on_gpu(p_off.view(np.int64)), on_gpu(u)
    act = np.array([rng.integers(0, n) if n and rng.random() < 0.9 else -1 for _, n in where] + [0] * spare, np.int32)
    adv = rng.normal(size=rows + spare).astype(np.float32)
    da, dadv = on_gpu(act), on_gpu(adv)
    new = lambda dt, m, fill: torch.full((m,), fill, dtype=dt, device="cuda")  # noqa: E731
    idx, kept, logp = new(torch.int32, rows + spare, -9), new(torch.int32, rows + spare, -9), new(torch.float32, rows + spare, 9)
    out, grad = new(torch.float32, total + 4, 9), new(v.dtype, total + 4, 9)
    lo, lp2, ent = (new(torch.float32, rows + spare, 9) for _ in range(3))
    torch.cuda.synchronize()
    view = policy.ragged_rows(dv.data_ptr(), dtype, rows + spare, frames, dq.data_ptr(), dp.data_ptr(), r_hi)
    be.draw(view, sampling(cut), du.data_ptr(), index=idx.data_ptr(), kept=kept.data_ptr(), logp=logp.data_ptr(),
            p=out.data_ptr())
    be.policy_loss(view, sampling(cut), da.data_ptr(), dadv.data_ptr(), 0.02, loss=lo.data_ptr(), logp=lp2.data_ptr(),
                   entropy=ent.data_ptr(), grad=grad.data_ptr())
    be.synchronize()
    # what lies behind the last question and the last entry stays as it was
    for a in (idx, kept, logp, lo, lp2, ent):
        assert bool((a[rows:] == a[-1]).all()) and abs(float(a[-1])) == 9
    assert bool((out[total:] == 9).all()) and bool((grad[total:] == 9).all())
    got_p, got_g = out.cpu().numpy(), grad.double().cpu().numpy()
    for i, (at, n) in enumerate(where):
        row = ref.policy(wide(v[at:at + n]), t, k, p, mp, f16=dtype == "f16")
        want = np.zeros(n)
        want[row[0]] = row[1]
        j, lp = ref.draw(row, u[i])
        assert (int(idx[i]), int(kept[i])) == (j, row[0].size), i
        near(got_p[at:at + n], want, HALF["f32"], TINY["f32"])
        near([float(logp[i])], [lp], HALF["f32"], 2e-12)
        L, lp, h, g = ref.loss(row, n, int(act[i]), float(adv[i]), float(np.float32(0.02)), t)
        near([float(lo[i]), float(lp2[i]), float(ent[i])], [L, lp, h], HALF["f32"], 4e-12)
        near(got_g[at:at + n], g, HALF[dtype], TINY[dtype] + 4e-12 * abs(adv[i]))


def test_one_row_a_frame_and_the_row_bound(be):
    """q_off NULL: one row a frame. A row over the stated bound is refused by itself."""
    rng = np.random.default_rng(8)
    n = np.array([3, 0, 200, 17])
    off = np.concatenate([[0], np.cumsum(n)]).astype(np.int64)
    v = scores(rng, 1, int(off[-1]), "f32", 0)[0]
    dv, dp, du = v.cuda(), on_gpu(off), on_gpu(np.full(6, 0.5))
    idx = torch.full((6,), -9, dtype=torch.int32, device="cuda")
    p = torch.full((int(off[-1]),), 9.0, device="cuda")
    torch.cuda.synchronize()
    for bound in (200, 100):
        p.fill_(9.0)
        idx.fill_(-9)
        torch.cuda.synchronize()
        be.draw(policy.ragged_rows(dv.data_ptr(), "f32", 6, 4, None, dp.data_ptr(), bound), policy.Sampling(),
                du.data_ptr(), index=idx.data_ptr(), p=p.data_ptr())
        be.synchronize()
        for i in range(4):
            want = ref.draw(ref.policy(wide(v[off[i]:off[i + 1]])), 0.5)[0]
            assert int(idx[i]) == (want if n[i] <= bound else -1)
        assert idx[4:].tolist() == [-9, -9]
        assert bool((p[3:203] == 9).all()) == (bound == 100) and not bool((p[203:] == 9).any())


def test_limits_row_by_row(be):
    rng = np.random.default_rng(12)
    rows, n = 40, 300
    v = scores(rng, rows, n, "f32")
    t = rng.uniform(0.3, 2, rows).astype(np.float32)
    t[:3] = [0.0, np.nan, -1.0]  # one answer each
    k = rng.integers(0, 50, rows).astype(np.int32)
    p = rng.uniform(0.1, 1.2, rows).astype(np.float32)
    p[5] = np.nan
    m = rng.uniform(0, 0.2, rows).astype(np.float32)
    m[6] = np.nan
    u = rng.random(rows)
    dev = [on_gpu(x) for x in (t, k, p, m, u)]
    dv = v.cuda()
    idx, kept = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    s = policy.Sampling(1.0, 0, 1.0, 0.0, *(x.data_ptr() for x in dev[:4]))
    be.draw(policy.dense_rows(dv.data_ptr(), "f32", rows, n), s, dev[4].data_ptr(), index=idx.data_ptr(),
            kept=kept.data_ptr())
    be.synchronize()
    for i in range(rows):
        row = ref.policy(wide(v[i]), float(t[i]) if t[i] > 0 else 0.0, int(k[i]), float(p[i]) if p[i] == p[i] else 1.0,
                         float(m[i]) if m[i] == m[i] else 0.0)
        assert (int(idx[i]), int(kept[i])) == (ref.draw(row, u[i])[0], row[0].size), i


@pytest.mark.parametrize("bound", [200, 1000, 4096, 30000, 200000])
def test_a_row_does_not_depend_on_how_it_is_split(be, bound):
    """The same short rows under every group size: the same answers, and pi to
    a last bit."""
    rng = np.random.default_rng(3)
    rows, n = 24, 190
    v, u = scores(rng, rows, n, "f32").cuda(), on_gpu(rng.random(rows))
    off = torch.arange(rows + 1, dtype=torch.int64, device="cuda") * n
    res = []
    for b in (n, bound):
        idx = torch.zeros(rows, dtype=torch.int32, device="cuda")
        p = torch.zeros(rows * n, device="cuda")
        torch.cuda.synchronize()
        be.draw(policy.ragged_rows(v.data_ptr(), "f32", rows, rows, None, off.data_ptr(), b),
                policy.Sampling(0.8, 30, 0.9), u.data_ptr(), index=idx.data_ptr(), p=p.data_ptr())
        be.synchronize()
        res.append((idx.cpu().numpy(), p.cpu().numpy()))
    assert np.array_equal(res[0][0], res[1][0])
    near(res[0][1], res[1][1], 2 * HALF["f32"])


@pytest.mark.parametrize("n", [1, 5, 60, 250, 999, 4096, 9000, 32001, 50001])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_policy_loss(be, n, dtype):
    rng = np.random.default_rng(n + 1)
    rows = 7 if n <= 4096 else 3
    for c, cut in enumerate([dict(), dict(temperature=0.7, top_p=0.9), dict(temperature=1.5, top_k=20, min_p=0.01),
                             dict(temperature=0.5)]):
        v = scores(rng, rows, n, dtype)
        if c % 2:  # likely answers, so that a cut policy holds them
            act = np.array([int(np.argmax(np.nan_to_num(wide(r), nan=-1e300, neginf=-1e300))) for r in v], np.int32)
        else:
            act = rng.integers(0, n, rows).astype(np.int32)
        act[0], act[-1] = -1, n + 3 if c == 2 else act[-1]
        adv, w = rng.normal(size=rows).astype(np.float32), rng.uniform(0.5, 2, rows).astype(np.float32)
        beta = [0.0, 0.05, 0.3, 0.01][c]
        t, k, p, mp = limits(cut)
        src = Place(rows, n, n + c, c, TYPES[dtype], 5.0)
        src.view().copy_(v)
        grad = Place(rows, n, n + 2, 3 * c, TYPES[dtype], 9.0)
        lo, lp, h = (torch.full((rows,), 9.0, device="cuda") for _ in range(3))
        da, dadv, dw = on_gpu(act), on_gpu(adv), on_gpu(w)
        torch.cuda.synchronize()
        view = policy.dense_rows(src.ptr(), dtype, rows, n, src.pitch)
        be.policy_loss(view, sampling(cut), da.data_ptr(), dadv.data_ptr(), beta, dw.data_ptr(), loss=lo.data_ptr(),
                       logp=lp.data_ptr(), entropy=h.data_ptr(), grad=grad.ptr(), grad_pitch=grad.pitch)
        be.synchronize()
        assert grad.rest_untouched()
        got = grad.view().double().cpu().numpy()
        for i in range(rows):
            row = ref.policy(wide(v[i]), t, k, p, mp, f16=dtype == "f16")
            L, l, e, g = ref.loss(row, n, int(act[i]), float(adv[i]), float(np.float32(beta)), t, float(w[i]))
            if c in (0, 3):
                stat, part = whole_tolerances(row, n, float(adv[i]), beta, float(w[i]) / t, l)
                near([float(lo[i]), float(lp[i]), float(h[i])], [L, l, e], HALF["f32"], stat)
                near(got[i], g, HALF[dtype], TINY[dtype] + part)
                continue
            near([float(lo[i]), float(lp[i]), float(h[i])], [L, l, e], HALF["f32"], 1e-11 * (1 + abs(float(adv[i]))))
            size = (abs(float(adv[i])) + beta * (np.log(n) + 1)) * float(w[i]) / t  # of the terms that cancel
            near(got[i], g, HALF[dtype], TINY[dtype] + 1e-11 * size)
        # in place: the gradient over the scores
        be.policy_loss(view, sampling(cut), da.data_ptr(), dadv.data_ptr(), beta, dw.data_ptr(), grad=src.ptr(),
                       grad_pitch=src.pitch)
        be.synchronize()
        assert bool((src.view() == grad.view()).all()) and src.rest_untouched()


def whole_tolerances(row, n, adv, beta, scale, logp):
    """What f32 weights add to half a step: of (loss, logp, entropy), and of each gradient."""
    j, pi, logpi = row
    h = -float((pi * logpi).sum()) if j.size else 0.0
    logp = logp if np.isfinite(logp) else 0.0
    e_logp, e_h = 2.0 ** -18 + 2.0 ** -22 * abs(logp), 2.0 ** -17 * (np.log2(n) + 2)
    part = np.zeros(n)
    part[j] = scale * pi * ((abs(adv) + beta * (np.abs(logpi) + h)) * (2.0 ** -17 + 2.0 ** -22 * np.abs(logpi))
                            + beta * e_h)
    # A weight below 2^-126 is 0: such a pi is off by at most 2^-126 (Z is 1 or
    # more), and pi |log pi|, which grows with pi there, by 126 ln 2 times that.
    part[j] += scale * 2.0 ** -126 * (abs(adv) + beta * (88 + h))
    return np.array([abs(adv) * e_logp + beta * e_h, e_logp, e_h]), part


def whole_loss(be, v, dtype, act, adv, beta, temps):
    """The uncut loss of v with a temperature a row, against the plain form."""
    rows, n = v.shape
    dv, dt = v.cuda(), on_gpu(np.asarray(temps, np.float32))
    da, dadv = on_gpu(np.asarray(act, np.int32)), on_gpu(np.asarray(adv, np.float32))
    lo, lp, h = (torch.zeros(rows, device="cuda") for _ in range(3))
    grad = torch.zeros_like(dv)
    torch.cuda.synchronize()
    be.policy_loss(policy.dense_rows(dv.data_ptr(), dtype, rows, n), policy.Sampling(row_temperature=dt.data_ptr()),
                   da.data_ptr(), dadv.data_ptr(), beta, loss=lo.data_ptr(), logp=lp.data_ptr(), entropy=h.data_ptr(),
                   grad=grad.data_ptr())
    be.synchronize()
    got = grad.double().cpu().numpy()
    for i in range(rows):
        t = float(np.float32(temps[i]))
        t = t if t > 0 else 0.0
        row = ref.policy(wide(v[i]), t, f16=dtype == "f16")
        L, l, e, g = ref.loss(row, n, int(act[i]), float(np.float32(adv[i])), float(np.float32(beta)), t)
        if dtype == "f16":  # half a step above 65504 and beyond, f16 rounds to infinity
            g = np.where(np.abs(g) >= 65520.0, np.copysign(np.inf, g), g)
        stat, part = whole_tolerances(row, n, float(adv[i]), beta, 1.0 / t if t else 0.0, l)
        near([float(lo[i]), float(lp[i]), float(h[i])], [L, l, e], HALF["f32"], stat)
        near(got[i], g, HALF[dtype], TINY[dtype] + part)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [40, 900, 5000])
def test_whole_softmax_where_masks_do_not_vanish_by_themselves(be, dtype, n):
    """Rows whose masked entries a plain exponential would let through: hot
    temperatures, largest scores next to the mask's floor, infinities, and
    temperatures of 0 and infinity."""
    rng = np.random.default_rng(n)
    v = scores(rng, 9, n, dtype, 0.3)
    v[1, :n // 2] = float("inf")
    if dtype == "f16":
        v[2] = torch.where(torch.from_numpy(rng.random(n) < 0.5), torch.tensor(-65504.0), torch.tensor(-65472.0)).half()
    else:
        v[2] = torch.where(torch.from_numpy(rng.random(n) < 0.5), torch.tensor(-1e30), torch.tensor(-9.5e28)).to(v.dtype)
    v[3] = torch.from_numpy(np.where(rng.random(n) < 0.5, np.nan, 1.0)).to(v.dtype)
    v[5, 7], v[5, 9] = 50.0, 50.0
    act = [int(ref.support(wide(r), f16=dtype == "f16")[:1].sum()) for r in v]
    act[5] = 9  # a later one of two largest
    temps = [700.0, 1.0, 1.0, 0.5, 1.0, 0.0, 1e25, np.inf, np.nan]
    whole_loss(be, v, dtype, act, rng.normal(size=9), 0.1, temps)
    act[5] = 7
    whole_loss(be, v, dtype, act, rng.normal(size=9), 0.0, temps)


def test_loss_gradient_against_differences(be):
    """Central differences of the reported f32 loss: a step of 2^-6 leaves a
    truncation below s^2/6 |L'''| <= 4e-5 (|A| <= 1, T = 0.8: |L'''| < 1 / T^3)
    and a rounding of 2^-24 |L| / s <= 2.4e-5 for |L| <= 6. The loss jumps
    where a step changes what top-k keeps: -0.31055 and -0.32520, the 7th and
    8th largest, lie 0.01465 < 2^-6 apart, so a step of either exchanges them
    and their differences say nothing of the gradient (the 64-bit form's are
    6e-4 off there too). Only steps that keep the set are compared."""
    rng = np.random.default_rng(2)
    n, s = 12, 2.0 ** -6
    base = rng.normal(0, 1, n).astype(np.float32)
    base = np.round(base * 1024) / 1024
    rows = np.repeat(base[None], 2 * n + 1, 0).astype(np.float32)
    for j in range(n):
        rows[1 + 2 * j, j] += s
        rows[2 + 2 * j, j] -= s
    v, m = on_gpu(rows), 2 * n + 1
    act = torch.full((m,), int(np.argsort(base)[-2]), dtype=torch.int32, device="cuda")
    adv = torch.full((m,), 0.9, device="cuda")
    lo, grad = torch.zeros(m, device="cuda"), torch.zeros(m * n, device="cuda")
    torch.cuda.synchronize()
    be.policy_loss(policy.dense_rows(v.data_ptr(), "f32", m, n), policy.Sampling(0.8, 7), act.data_ptr(),
                   adv.data_ptr(), 0.2, loss=lo.data_ptr(), grad=grad.data_ptr())
    be.synchronize()
    L, g = lo.double().cpu().numpy(), grad.double().cpu().numpy()[:n]
    held = [set(np.argsort(-r, kind="stable")[:7]) for r in rows]
    same = np.array([held[1 + 2 * j] == held[2 + 2 * j] == held[0] for j in range(n)])
    assert same.sum() == n - 2
    assert np.abs((L[1::2] - L[2::2]) / (2 * s) - g)[same].max() < 7e-5 + 7e-5
    assert (g != 0).sum() == 7  # what top-k leaves out has no gradient


def test_captured_draw_replays_on_new_inputs(be):
    rng = np.random.default_rng(4)
    rows, n = 9, 500
    v = torch.zeros(rows, n, device="cuda")
    u = torch.zeros(rows, dtype=torch.float64, device="cuda")
    idx = torch.zeros(rows, dtype=torch.int32, device="cuda")
    act, adv = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.ones(rows, device="cuda")
    grad = torch.zeros(rows, n, device="cuda")
    view = policy.dense_rows(v.data_ptr(), "f32", rows, n)
    s = policy.Sampling(0.9, 50, 0.9)
    prev = be.stream_ptr()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    be.set_stream(side.cuda_stream)  # before the capture begins: it orders the new stream after the old
    try:
        with torch.cuda.graph(g, stream=side):
            be.draw(view, s, u.data_ptr(), index=idx.data_ptr())
            be.policy_loss(view, s, idx.data_ptr(), adv.data_ptr(), 0.1, grad=grad.data_ptr())
    finally:
        be.set_stream(prev)
    for rep in range(3):
        hv, hu = scores(rng, rows, n, "f32"), rng.random(rows)
        v.copy_(hv)
        u.copy_(torch.from_numpy(hu))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for i in range(rows):
            row = ref.policy(wide(hv[i]), limits(dict(temperature=0.9))[0], 50, limits(dict(top_p=0.9))[2])
            j, _ = ref.draw(row, hu[i])
            assert int(idx[i]) == j
            want = ref.loss(row, n, j, 1.0, float(np.float32(0.1)), limits(dict(temperature=0.9))[0])[3]
            near(grad[i].cpu().numpy(), want, HALF["f32"], 1e-11)
    g.reset()


def check_ragged(be, v, dtype, where, view, cut, u, total, spare=0, kind="scores"):
    """A packed batch's draws against the plain form; `spare` rows behind the last question."""
    t, k, p, mp = limits(cut)
    rows = len(where)
    du = on_gpu(u)
    idx, kept = (torch.full((rows + spare,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    logp, out = torch.full((rows + spare,), 9.0, device="cuda"), torch.full((total + 3,), 9.0, device="cuda")
    torch.cuda.synchronize()
    be.draw(view, sampling(cut), du.data_ptr(), index=idx.data_ptr(), kept=kept.data_ptr(), logp=logp.data_ptr(),
            p=out.data_ptr())
    be.synchronize()
    idx, kept, logp, out = (x.cpu().numpy() for x in (idx, kept, logp, out))
    assert (idx[rows:] == -9).all() and (kept[rows:] == -9).all() and (logp[rows:] == 9).all() and (out[total:] == 9).all()
    for i, (at, n) in enumerate(where):
        row = ref.policy(wide(v[at:at + n]), t, k, p, mp, kind, dtype == "f16")
        want = np.zeros(n)
        want[row[0]] = row[1]
        j, lp = ref.draw(row, u[i])
        assert (int(idx[i]), int(kept[i])) == (j, row[0].size), i
        near(out[at:at + n], want, HALF["f32"], TINY["f32"])
        near([logp[i]], [lp], HALF["f32"], 2e-12)


@pytest.mark.parametrize("rows", [30, 3000, 45000])
def test_runs_of_short_rows(be, rows):
    """Many short rows: a warp walks through a run of them, over frames without
    questions and without a bank, and stops behind the last."""
    rng = np.random.default_rng(rows)
    frames = rows // 3
    q, r = rng.integers(0, 7, frames), rng.integers(0, 20, frames)
    q[rng.random(frames) < 0.2] = 0
    q_off = np.concatenate([[0], np.cumsum(q)]).astype(np.uint64)
    p_off = np.concatenate([[0], np.cumsum(q * r)]).astype(np.uint64)
    v = scores(rng, 1, int(p_off[-1]), "f32")[0]
    where = [(int(p_off[f]) + i * int(r[f]), int(r[f])) for f in range(frames) for i in range(int(q[f]))]
    dv, dq, dp = v.cuda(), on_gpu(q_off.view(np.int64)), on_gpu(p_off.view(np.int64))
    spare = rows // 4 + 1
    view = policy.ragged_rows(dv.data_ptr(), "f32", len(where) + spare, frames, dq.data_ptr(), dp.data_ptr(), 20)
    check_ragged(be, v, "f32", where, view, dict(temperature=0.8, top_k=7, top_p=0.8), rng.random(len(where) + spare),
                 int(p_off[-1]), spare)


@pytest.mark.parametrize("open_", [1, 32, 33, 64, 65, 128, 129, 250])
def test_lists_of_every_length(be, open_):
    """What the mask leaves of a row is gathered: every size of list, each cut, with ties."""
    rng = np.random.default_rng(open_)
    for n, dtype in ((250, "f32"), (900, "bf16"), (5000, "f16"), (40000, "bf16")):
        v = np.full((4, n), -np.inf, np.float32)
        for i in range(4):
            at = np.sort(rng.choice(n, open_, replace=False))
            v[i, at] = rng.normal(0, 2, open_) if i % 2 else np.round(rng.normal(0, 1, open_))
        t = torch.from_numpy(v).to(TYPES[dtype])
        for cut in (dict(), dict(top_k=open_ // 2 + 1), dict(top_p=0.8, temperature=1.3),
                    dict(top_k=open_ // 3 + 1, top_p=0.7, min_p=0.05), dict(temperature=0.0)):
            check_draw(be, t, dtype, cut, rng.random(4), offset=3, pitch=n + 2)


@pytest.mark.parametrize("n,dtype", [(1000, "f32"), (4096, "bf16"), (12000, "f32"), (30000, "f16"), (100000, "bf16"),
                                     (200000, "f32")])
def test_top_k_bounds_that_hold_too_much(be, n, dtype):
    """Rows of few values: the lower bound of the k-th largest admits more than
    a list, and the row stays spread over its group; and k beyond any list."""
    rng = np.random.default_rng(n)
    few = np.round(rng.normal(0, 0.6, (3, n))).astype(np.float32)
    few[1] = 1.0
    few[2, 5] = 9.0
    t = torch.from_numpy(few).to(TYPES[dtype])
    for cut in (dict(top_k=50), dict(top_k=2), dict(top_k=200, top_p=0.6), dict(top_k=n // 2, top_p=0.9),
                dict(top_k=n - 1)):
        check_draw(be, t, dtype, cut, rng.random(3))
    u = torch.from_numpy(rng.normal(0, 2, (3, n)).astype(np.float32)).to(TYPES[dtype])
    for cut in (dict(top_k=207), dict(top_k=209), dict(top_k=208, top_p=0.5), dict(top_k=1, top_p=0.5)):
        check_draw(be, u, dtype, cut, rng.random(3))


@pytest.mark.parametrize("rows,n", [(3000, 700), (1500, 1500)])
def test_batches_of_long_rows(be, rows, n):
    """Enough long rows that a CTA takes several: lists, rows that stay spread,
    empty rows and the rows behind the last question side by side."""
    rng = np.random.default_rng(rows)
    lens = rng.integers(0, n + 1, rows)
    off = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    v = scores(rng, 1, int(off[-1]), "bf16", 0.5)[0]
    v[off[7]:off[40]] = v[off[7]:off[40]].round()  # many ties
    where = [(int(off[i]), int(lens[i])) for i in range(rows)]
    dv, dp = v.cuda(), on_gpu(off)
    spare = 9
    view = policy.ragged_rows(dv.data_ptr(), "bf16", rows + spare, rows, None, dp.data_ptr(), n)
    for cut in (dict(top_k=60, top_p=0.9), dict(temperature=0.7, top_p=0.8)):
        check_ragged(be, v, "bf16", where, view, cut, rng.random(rows + spare), int(off[-1]), spare)


@pytest.mark.parametrize("n", [4096, 60000])
def test_uniforms_at_the_borders_of_the_warps(be, n):
    """Nothing is cut, so the row stays spread over its group, and uniforms step
    by last bits over every border a split into 32 could have. A last bit of
    the sums may move the answer to the border's other entry, no further."""
    rng = np.random.default_rng(n)
    p = (rng.random(n) ** 3 + 1e-6).astype(np.float32)
    p[rng.random(n) < 0.02] = 0.0
    cum = np.cumsum(p.astype(np.longdouble))
    borders = np.unique(np.concatenate([np.arange(1, 32) * n // 32, np.arange(512, n, 512), np.arange(1024, n, 1024)]))
    if n > 4096:
        borders = borders[rng.permutation(borders.size)[:24]]
    u, where = [], []
    for b in borders:
        mid = float(cum[b - 1] / cum[-1])
        for k in range(-20, 21):
            u.append(mid + k * np.spacing(mid))
            where.append(b)
    rows = len(u)
    v = on_gpu(p).expand(rows, n).contiguous()
    du, idx = on_gpu(np.array(u)), torch.zeros(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.draw(policy.dense_rows(v.data_ptr(), "f32", rows, n, kind="p"), policy.Sampling(), du.data_ptr(),
            index=idx.data_ptr())
    be.synchronize()
    open_ = np.flatnonzero(p > 0)
    for got, b in zip(idx.tolist(), where):
        at = int(np.searchsorted(open_, b))  # the first open entry at or behind the border
        assert got in open_[max(at - 1, 0):at + 1], (got, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [249, 301, 505, 1017, 2001, 3501, 7001, 8185, 13001, 16377, 30001])
def test_whole_softmax_at_every_group(be, dtype, n):
    """Odd rows, each at an alignment of its own, on both sides of the group
    sizes' borders; the large advantage takes the gradient's 64-bit form."""
    rng = np.random.default_rng(n)
    v = scores(rng, 7, n, dtype, 0.2)
    act = [int(ref.support(wide(r), f16=dtype == "f16")[-1:].sum()) for r in v]
    adv, temps = rng.normal(size=7), np.array([1.0, 0.6, 0.05, 1.0, 1.0, 2.5, 0.3])
    adv[2] = 1e4
    whole_loss(be, v, dtype, act, adv, 0.1, temps)
    if dtype != "f16":  # f16 gradients end at 65504
        whole_loss(be, v, dtype, act, adv, 300.0, temps)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [40, 900, 5000])
def test_whole_softmax_at_the_smallest_temperatures(be, dtype, n):
    """1 / T beyond f32: one entry has all of the mass, no gradient is left."""
    v = scores(np.random.default_rng(n), 4, n, dtype, 0.3)
    v[:, 5] = 40.0
    temps = [1e-38, 1e-40, 2.0 ** -149, 3e-39]
    whole_loss(be, v, dtype, [5, 5, 5, 6], [1.0, -2.0, 0.5, 1.0], 0.1, temps)


def test_draws_over_the_values_themselves(be):
    """p may be the f32 values: short rows, lists of long ones, and spread rows."""
    rng = np.random.default_rng(6)
    for rows, n, cut in ((40, 200, dict(top_p=0.9)), (700, 1500, dict(top_k=20)), (5, 9000, dict(top_p=0.95)),
                         (3, 50000, dict(top_k=30)), (2, 50000, dict(top_p=0.9))):
        v = scores(rng, rows, n, "f32").cuda()
        u = on_gpu(rng.random(rows))
        want = torch.zeros(rows, n, device="cuda")
        idx = [torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        view = policy.dense_rows(v.data_ptr(), "f32", rows, n)
        be.draw(view, sampling(cut), u.data_ptr(), index=idx[0].data_ptr(), p=want.data_ptr())
        be.draw(view, sampling(cut), u.data_ptr(), index=idx[1].data_ptr(), p=v.data_ptr())
        be.synchronize()
        assert torch.equal(v, want) and torch.equal(idx[0], idx[1])


@pytest.mark.parametrize("n", [50, 700, 5000])
def test_loss_limits_row_by_row(be, n):
    """Cut losses with a temperature a row: 0, NaN and negative have one answer,
    infinity weighs every kept entry alike."""
    rng = np.random.default_rng(n)
    rows = 8
    v = scores(rng, rows, n, "f32")
    temps = np.array([0.5, 0.0, np.nan, -1.0, 0.9, np.inf, 2.0, 1.0], np.float32)
    ks = rng.integers(1, n, rows).astype(np.int32)
    act = np.array([int(np.argmax(np.nan_to_num(wide(r), nan=-1e300, neginf=-1e300))) for r in v], np.int32)
    adv = rng.normal(size=rows).astype(np.float32)
    dev = [on_gpu(x) for x in (temps, ks, act, adv)]
    dv, grad = v.cuda(), torch.full((rows, n), 9.0, device="cuda")
    lo, lp, h = (torch.full((rows,), 9.0, device="cuda") for _ in range(3))
    torch.cuda.synchronize()
    s = policy.Sampling(row_temperature=dev[0].data_ptr(), row_top_k=dev[1].data_ptr())
    be.policy_loss(policy.dense_rows(dv.data_ptr(), "f32", rows, n), s, dev[2].data_ptr(), dev[3].data_ptr(), 0.1,
                   loss=lo.data_ptr(), logp=lp.data_ptr(), entropy=h.data_ptr(), grad=grad.data_ptr())
    be.synchronize()
    for i in range(rows):
        t = float(temps[i]) if temps[i] > 0 else 0.0
        row = ref.policy(wide(v[i]), t, int(ks[i]))
        L, l, e, g = ref.loss(row, n, int(act[i]), float(adv[i]), float(np.float32(0.1)), t)
        near([float(lo[i]), float(lp[i]), float(h[i])], [L, l, e], HALF["f32"], 4e-11)
        near(grad[i].cpu().numpy(), g, HALF["f32"], 4e-11)


def test_offsets_past_32_bits(be):
    """Rows, packed blocks and outputs that start behind 2^32 elements."""
    rng = np.random.default_rng(1)
    n, far = 300, (1 << 32) + 5
    buf = torch.empty(far + 4 * n, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(far + 4 * n, dtype=torch.float32, device="cuda")
    grad = torch.empty(far + 4 * n, dtype=torch.bfloat16, device="cuda")
    v = scores(rng, 2, n, "bf16")
    u = rng.random(2)
    idx = torch.zeros(2, dtype=torch.int32, device="cuda")
    act, adv = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda")
    du, s = on_gpu(u), policy.Sampling(0.9, 40, 0.9)
    views = [(policy.dense_rows(buf.data_ptr(), "bf16", 2, n, far), [0, far], far),
             (policy.ragged_rows(buf.data_ptr(), "bf16", 2, 1, None, 0, n), [far, far + n], 0)]
    q, p = torch.tensor([0, 2], device="cuda"), torch.tensor([far, far + 2 * n], device="cuda")
    views[1][0].q_off, views[1][0].p_off = q.data_ptr(), p.data_ptr()
    for view, starts, pitch in views:
        for i, at in enumerate(starts):
            buf[at:at + n] = v[i].cuda()
            out[at:at + n] = 9.0
            grad[at:at + n] = 9.0
        torch.cuda.synchronize()
        be.draw(view, s, du.data_ptr(), index=idx.data_ptr(), p=out.data_ptr(), p_pitch=pitch)
        act.copy_(idx)
        torch.cuda.synchronize()
        be.policy_loss(view, s, idx.data_ptr(), adv.data_ptr(), 0.0, grad=grad.data_ptr(), grad_pitch=pitch)
        be.synchronize()
        for i, at in enumerate(starts):
            t, k, tp, _ = limits(dict(temperature=0.9, top_k=40, top_p=0.9))
            row = ref.policy(wide(v[i]), t, k, tp)
            want = np.zeros(n)
            want[row[0]] = row[1]
            assert int(idx[i]) == ref.draw(row, u[i])[0]
            near(out[at:at + n].cpu().numpy(), want, HALF["f32"], TINY["f32"])
            g = ref.loss(row, n, int(idx[i]), 1.0, 0.0, t)[3]
            near(grad[at:at + n].double().cpu().numpy(), g, HALF["bf16"], TINY["bf16"] + 1e-11)


FIRST_CALL = """
import numpy as np, torch
from krystal_b200 import BRAIN_FORWARD_CONFIG, GradList, Sampling, create_brain_forward_weights, cuda_backend, policy
cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
be = cuda_backend(0)(cfg, create_brain_forward_weights(cfg, 1))
v = {n: torch.randn(3, n, device="cuda") for n in (40, 900, 5000, 60000)}
u = torch.rand(3, dtype=torch.float64, device="cuda")
adv = torch.ones(3, device="cuda")
idx = {n: torch.zeros(3, dtype=torch.int32, device="cuda") for n in v}
grad = {n: [torch.zeros_like(x) for _ in range(2)] for n, x in v.items()}
res = torch.zeros(2, dtype=torch.float64, device="cuda")
lst = GradList([g[0] for g in grad.values()])
side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
be.set_stream(side.cuda_stream)
cut = Sampling(0.9, 20, 0.9)
with torch.cuda.graph(graph, stream=side):
    for n, x in v.items():
        rows = policy.dense_rows(x.data_ptr(), "f32", 3, n)
        be.draw(rows, cut, u.data_ptr(), index=idx[n].data_ptr())
        for s, g in zip((cut, Sampling()), grad[n]):
            be.policy_loss(rows, s, idx[n].data_ptr(), adv.data_ptr(), 0.1, grad=g.data_ptr())
    be.clip_grads(lst, 0.5, res.data_ptr())
graph.replay()
torch.cuda.synchronize()
captured = [t.clone() for n in v for t in (idx[n], *grad[n])] + [res.clone()]
for n, x in v.items():
    rows = policy.dense_rows(x.data_ptr(), "f32", 3, n)
    be.draw(rows, cut, u.data_ptr(), index=idx[n].data_ptr())
    for s, g in zip((cut, Sampling()), grad[n]):
        be.policy_loss(rows, s, idx[n].data_ptr(), adv.data_ptr(), 0.1, grad=g.data_ptr())
be.clip_grads(lst, 0.5, res.data_ptr())
torch.cuda.synchronize()
now = [t for n in v for t in (idx[n], *grad[n])] + [res]
assert all(torch.equal(a, b) for a, b in zip(captured, now))
assert float(res[0]) > 0 and all(bool((i >= 0).all()) for i in idx.values())
graph.reset()
be.destroy()
print("captured first calls agree")
"""


def test_the_first_calls_of_a_process_can_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first calls agree" in r.stdout, r.stderr[-2000:]
