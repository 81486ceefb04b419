"""The policy loss where factors are not finite or leave f32: rows that must
have no gradient, masked entries, and gradients whose factors overflow; and
confident rows, where pi - 1 and log pi are small."""
import numpy as np
import pytest

from krystal_b200 import policy
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from tests.test_gpu_policy import scores, whole_loss

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# a row a warp, a row in a CTA's shared memory, a row over a cluster (f32)
LENGTHS = [40, 300, 900, 5000, 20001]
CUTS = [dict(), dict(top_k=7), dict(top_p=0.9)]


@pytest.fixture(scope="module")
def be():
    cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
    b = CudaBrainBackend(cfg, create_brain_forward_weights(cfg, 1337), 0)
    yield b
    b.destroy()


def on_gpu(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype))).cuda()


def policy_loss(be, v, dtype, act, adv, weight, temps=None, beta=0.1, cut=None):
    """(loss, logp, entropy, grad in its type) of the rows of v."""
    rows, n = v.shape
    dv, da, dadv, dw = v.cuda(), on_gpu(act, np.int32), on_gpu(adv, np.float32), on_gpu(weight, np.float32)
    dt = on_gpu(temps, np.float32) if temps is not None else None
    lo, lp, h = (torch.full((rows,), 9.0, device="cuda") for _ in range(3))
    grad = torch.full_like(dv, 9.0)
    s = policy.Sampling(**(cut or {}), row_temperature=dt.data_ptr() if dt is not None else None)
    torch.cuda.synchronize()
    be.policy_loss(policy.dense_rows(dv.data_ptr(), dtype, rows, n), s, da.data_ptr(), dadv.data_ptr(), beta,
                   dw.data_ptr(), loss=lo.data_ptr(), logp=lp.data_ptr(), entropy=h.data_ptr(), grad=grad.data_ptr())
    be.synchronize()
    return lo.cpu().numpy(), lp.cpu().numpy(), h.cpu().numpy(), grad.cpu()


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
def test_a_row_without_an_answer_has_no_gradient_whatever_its_factors(be, n, dtype, cut):
    """No target, a target outside the row, a masked one and a temperature of 0,
    each with advantages and weights that are not finite, between rows that
    learn."""
    rng = np.random.default_rng(n)
    nan, inf = np.nan, np.inf
    factors = [(nan, 1.0), (inf, 1.0), (-inf, 2.0), (1.0, nan), (0.5, inf), (nan, nan)]
    kinds = [-1, n + 3, 0, 1]  # of the row's action; entry 0 is masked, entry 1 the largest, at temperature 0
    rows = [(k, a, w) for k in kinds for a, w in factors]
    v = torch.from_numpy(rng.normal(0, 1.5, (len(rows) + 2, n)).astype(np.float32))
    v[:, 1] = v.amax(1) + 0.5
    v[:, 0] = -inf
    act = [1] + [r[0] for r in rows] + [1]
    adv, weight = [0.7] + [r[1] for r in rows] + [-0.4], [1.0] + [r[2] for r in rows] + [1.5]
    temps = [0.8] + [0.0 if r[0] == 1 else 0.8 for r in rows] + [0.8]
    lo, lp, h, g = policy_loss(be, v.to(TYPES[dtype]), dtype, act, adv, weight, temps, cut=cut)
    quiet = slice(1, len(rows) + 1)
    assert (lo[quiet] == 0).all()
    assert bool((g[quiet] == 0).all())
    assert [x for x in lp[quiet]] == [0.0 if r[0] == -1 or r[0] == 1 else -inf for r in rows]
    assert np.isfinite(h).all()
    for i in (0, len(rows) + 1):  # the rows beside them learn
        assert np.isfinite(lo[i]) and lo[i] != 0 and bool(torch.isfinite(g[i]).all()) and float(g[i, 1]) != 0


def plain_gradient(v, act, adv, beta, t, weight, f16):
    """The uncut gradient of one row in 64 bits, and the size of the terms that
    cancel in it; 0 for masked entries whatever the factors, and everywhere
    where the action's weight is below e^-700, which cannot be drawn."""
    v = v.double().numpy()
    j = np.flatnonzero(v > (-65504.0 if f16 else -1e29))
    j = j[(v[j] - v[j].max()) / t >= -700.0]
    x = (v[j] - v[j].max()) / t
    w = np.exp(x)
    pi, logpi = w / w.sum(), x - np.log(w.sum())
    h = -(pi * logpi).sum()
    d = adv * pi + beta * pi * (logpi + h)
    d[j == act] -= adv
    g, size = np.zeros(v.size), np.zeros(v.size)
    if act not in j:
        return j, pi, g, size
    g[j] = weight * d / t
    size[j] = abs(weight) / t * (abs(adv) * (pi + (j == act)) + abs(beta) * pi * (np.abs(logpi) + h))
    return j, pi, g, size


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("beta", [0.0, 0.1])
def test_gradients_whose_factors_leave_f32(be, n, dtype, beta):
    """weight * advantage / T beyond f32: masked entries stay 0, and so do those
    whose weight is 0 in 64 bits; the others are rounded from 64-bit products,
    to infinity where they leave their type. A weight is off by 2^-17 of itself
    (f32 sums and ex2, as for every uncut row) and below 2^-126 it is 0; half a
    step of the type on top."""
    rng = np.random.default_rng(n)
    v = torch.from_numpy(rng.normal(0, 1.5, (6, n)).astype(np.float32))
    v[:, ::5] = -np.inf
    v[:, 1::5] -= 2000.0  # e^-2000 is 0 in 64 bits
    v[:, 2::10] -= 60.0   # pi about 1e-27: finite gradients
    v = v.to(TYPES[dtype])
    likely = v.float()[:, 3::5]
    act = (likely.argmin(1) * 5 + 3).tolist()  # not the largest: a gradient is left at T = 1e-3
    temps = [1.0, 0.7, 1.0, 2.0, 1e-3, 0.5]
    adv, weight = [1e30, -1e25, 3e38, 1e20, -2e36, 1e38], [1e25, 1e30, 4.0, 1e33, 1.0, -1e38]
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    tiny = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[dtype]
    most = float(torch.finfo(TYPES[dtype]).max)
    f = lambda x: float(np.float32(x))  # noqa: E731
    beta = f(beta)
    g = policy_loss(be, v, dtype, act, adv, weight, temps, beta)[3].double().numpy()
    for i in range(6):
        t = f(temps[i])
        j, pi, want, size = plain_gradient(v[i], act[i], f(adv[i]), beta, t, f(weight[i]), dtype == "f16")
        assert not np.isnan(g[i]).any()
        off = np.ones(n, bool)
        off[j] = False
        assert (g[i][off] == 0).all() and (g[i][want == 0] == 0).all()
        # pi's error: 2^-17 of itself, more by the rounding of x where |x| is large; all of it where the weight is 0
        x = np.zeros(n)
        x[j] = np.abs(np.log(np.maximum(pi, 1e-320)))
        slack = size * (2.0 ** -17 + 2.0 ** -22 * x) + half * 1.001 * np.abs(want)
        gone = np.zeros(n, bool)
        gone[j] = pi < 2.0 ** -125
        sure = (np.abs(want) + slack < most) & ~gone
        assert (np.abs(g[i] - want)[sure] <= slack[sure] + tiny).all()
        over = (np.abs(want) - slack > 2 * most) & ~gone
        assert (g[i][over] == np.copysign(np.inf, want[over])).all()
        assert over.any() or act[i] not in j


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
def test_masked_entries_have_no_gradient_whatever_the_factors(be, n, dtype, cut):
    rng = np.random.default_rng(n)
    v = torch.from_numpy(rng.normal(0, 1.5, (4, n)).astype(np.float32))
    v[:, 1] = v.amax(1) + 0.5
    v[:, ::3] = torch.tensor([-np.inf, np.nan, -1e30, np.nan], dtype=torch.float32)[:, None]
    inf = np.inf
    g = policy_loss(be, v.to(TYPES[dtype]), dtype, [1] * 4, [np.nan, inf, -inf, 1.0], [1.0, 1.0, 2.0, inf],
                    cut=cut)[3]
    assert bool((g[:, ::3] == 0).all())
    assert not bool(torch.isfinite(g[:, 1]).any())


@pytest.mark.parametrize("dtype,at", [("f32", 0.0), ("f16", 0.0), ("bf16", 0.0), ("f32", 1e3), ("f32", 1e6)])
@pytest.mark.parametrize("n", LENGTHS)
def test_confident_rows_keep_their_small_gradient(be, n, dtype, at):
    """The action holds all but 1e-3 to 1e-12 of the mass. Its gradient, the loss
    and the entropy are as exact as the others' weights: an f32 exponent x is
    off by 2^-23 |x| (log2(e) / T in f32) and its own rounding, |x| <= 35, the
    weight by ex2's 2^-22 and the sum's 18 terms: below 2^-16 of each, which
    makes 2^-15 of what is made of them; half a step of the type on top. At 1e3
    (f32) every exponent holds one rounding of m log2(e) / T, which cancels; at
    1e6 the largest score is subtracted first."""
    rng = np.random.default_rng(n)
    gap = np.array([8.0, 14.0, 20.0, 30.0]) + np.log(n)
    v = np.round(rng.uniform(-2, 0, (4, n)) - gap[:, None], 0 if at else 3)  # (f32 steps of 1e6 are 2^-4)
    act = [n - 1, 0, n // 2, n // 3]
    v[np.arange(4), act] = 0.0
    v[:, 7 % n] = -np.inf if 7 not in act else v[:, 7]
    v = torch.from_numpy((v + at).astype(np.float32)).to(TYPES[dtype])
    adv, weight = [1.0, -0.7, 2.0, 1.5], [1.0, 1.0, 3.0, 0.25]
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    tiny = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[dtype]
    for beta in (0.0, 0.125):
        lo, lp, h, g = policy_loss(be, v, dtype, act, adv, weight, beta=beta)
        g = g.double().numpy()
        for i in range(4):
            x = v[i].double().numpy() - float(v[i, act[i]])
            keep = np.isfinite(x)
            w = np.where(keep, np.exp(np.where(keep, x, 0.0)), 0.0)
            others = w.sum() - 1.0 if w.sum() > 1.1 else np.delete(w, act[i]).sum()
            z = 1.0 + others
            logp = -np.log1p(others)
            ent = -logp / z - (np.where(keep, w * (np.where(keep, x, 0.0) + logp), 0.0).sum() - logp) / z
            a = act[i]
            want = weight[i] * (-adv[i] * others / z + beta / z * (logp + ent))
            size = weight[i] * (abs(adv[i]) * others / z + beta / z * (abs(logp) + ent))
            assert 0 < others < 1e-3
            assert abs(g[i, a] - want) <= 2.0 ** -15 * size + 1.001 * half * abs(want) + tiny
            assert abs(lp[i] - logp) <= 2.0 ** -15 * abs(logp)
            assert abs(h[i] - ent) <= 2.0 ** -15 * ent
            assert abs(lo[i] - (-adv[i] * logp - beta * ent)) <= 2.0 ** -15 * (abs(adv[i] * logp) + beta * ent)
            if dtype == "f32" and not beta:  # pi - 1 and the other pi sum to nothing
                assert abs(g[i].sum()) <= 2.0 ** -14 * abs(want)


@pytest.mark.parametrize("dtype,n", [("f32", 17000), ("f32", 18400), ("bf16", 34000), ("bf16", 36800), ("f16", 36801)])
def test_rows_whose_threads_add_eighteen_terms(be, dtype, n):
    """The longest partial sums: 17 and 18 terms a thread, off by 18 2^-24. With
    ex2's 2^-22 and 0.7 2^-24 log2 n of the exponents' rounding (log2 n <= 15.2)
    Z is within 2^-18.9 of itself, below the 2^-18 that whole_loss allows of
    log Z."""
    rng = np.random.default_rng(n)
    v = scores(rng, 4, n, dtype, 0.05)
    act = [int(np.argmax(np.nan_to_num(r.double().numpy(), nan=-1e300, neginf=-1e300))) for r in v]
    act[1] = int(np.flatnonzero(v[1].double().numpy() > -1e4)[n // 2])
    whole_loss(be, v, dtype, act, rng.normal(size=4), 0.1, [1.0, 0.8, 5.0, 30.0])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
def test_the_entropy_of_rows_whose_action_is_masked(be, n, dtype):
    """Every sort of mask under the action, and an action outside the row: H is
    the row's, within 2^-17 (log2 n + 2) as for every uncut row."""
    rng = np.random.default_rng(n)
    masks = [np.nan, -np.inf, -1e30, float(np.finfo(np.float32).min), np.nan, np.nan]
    v = torch.from_numpy(rng.normal(0, 1.5, (6, n)).astype(np.float32))
    act = [1, 5, n - 2, n // 2, n + 3, -1]
    for i, a in enumerate(act):
        if 0 <= a < n:
            v[i, a] = masks[i]
    v = v.to(TYPES[dtype])
    temps = [1.0, 0.5, 2.0, 1.0, 1.0, 1e-3]
    lo, lp, h, g = policy_loss(be, v, dtype, act, [1.0] * 6, [1.0] * 6, temps)
    assert (lo == 0).all() and bool((g == 0).all()) and (lp == [-np.inf] * 5 + [0.0]).all()
    for i in range(6):
        x = v[i].double().numpy()
        x = x[x > (-65504.0 if dtype == "f16" else -1e29)]
        x = (x - x.max()) / float(np.float32(temps[i]))
        pi = np.exp(x) / np.exp(x).sum()
        want = float(np.log(np.exp(x).sum()) - (pi * x).sum())
        assert abs(h[i] - want) <= 2.0 ** -17 * (np.log2(n) + 2)
