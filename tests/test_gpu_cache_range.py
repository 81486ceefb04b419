"""The bank cache's attention and scores over the whole range that its cache and
its questions take: open rows whose values lie many orders apart."""
import numpy as np
import pytest

from krystal_b200 import cache as kc
from tests import cache_cases as ref
from tests.test_gpu_cache import TYPES, Asked, Bank, be, cuda, offsets  # noqa: F401 (be: the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -23


def filled(be, lengths, keys, values, fmt="i8", dtype="f32"):
    """A bank that holds these rows [all, kv, dim]."""
    kv, dim = keys.shape[1:]
    b = Bank(be, lengths, kv, dim, fmt, dtype=dtype)
    most = float(np.finfo(np.float32).max)
    x = cuda(np.clip([keys, values], -most, most).astype(np.float32), TYPES[dtype])
    host = x.float().cpu().numpy()
    torch.cuda.synchronize()
    be.cache_write(b.cache, b.table, kc.cache_rows(x[0].data_ptr(), x[1].data_ptr(), dtype, sum(lengths),
                                                   b.d["off"].data_ptr()))
    be.synchronize()
    off = offsets(lengths)
    k, v = ref.quantised(host[0], fmt), ref.quantised(host[1], fmt)
    b.keys = [k[off[s]:off[s + 1]] for s in range(b.n)]
    b.values = [v[off[s]:off[s + 1]] for s in range(b.n)]
    return b


def close(a, got, scale=0.0, mask=False, least=1e-37):
    """As Asked.check, but the output's room follows what each row adds to it, not
    the largest value: with p the weights' shares,
      a share is off by 4 ds (its own score, the maximum's, and the sum's), by the
      weight's rounding and by the sums' n / 8 + 64 steps, so that the output is by
      that of sum p |v|; a weight's rounding does not go below 2^-33 of the largest
      product of a weight and its row's scale, a step of which is at most the row's
      largest |v|: n / 2^33 of the largest p max|v|. least: f16's own smallest numbers."""
    out, lse = got
    b = a.bank
    sc = scale or float(np.float32(1 / np.sqrt(b.dim)))
    half = float(torch.finfo(TYPES[a.dtype]).eps) / 2
    weight = 2.0 ** -11 if a.dtype == "bf16" else 2.0 ** -22
    g = a.heads // b.kv
    for i in range(a.total):
        s = a.seq[i]
        m = a.mask[s][i - a.off[s]] if mask else np.zeros(b.lengths[s])
        for h in range(a.heads):
            k, v = (x[s][:, h // g].astype(np.float64) for x in (b.keys, b.values))
            q, n = a.q[i, h].astype(np.float64), len(k)
            x, ok = ref.masked(k @ q * sc, m)
            if not ok.any():
                assert (out[i, h] == 0).all() and lse[i, h] == -np.inf, (i, h)
                continue
            x = np.where(ok, x, -np.inf)
            p = np.exp(x - x.max())
            wl = x.max() + np.log(p.sum())
            p /= p.sum()
            want, size = p @ v, p @ np.abs(v)
            terms = (np.abs(k) @ np.abs(q)).max() * abs(sc)
            ds = terms * (b.dim * U + 2.0 ** -22) + 4 * U * (abs(wl) + terms + 128 + (16 if mask else 0))
            assert abs(lse[i, h] - wl) <= 2 * ds + (n / 8 + 64) * U, (i, h, lse[i, h], wl)
            room = size * (4 * ds + weight + (n / 8 + 64) * U) + half * np.abs(want)
            room += n * 2.0 ** -33 * (p * np.abs(v).max(1)).max()
            assert (np.abs(out[i, h] - want) <= room + least).all(), (i, h, np.abs(out[i, h] - want).max(), room.min())


# --- value scales ----------------------------------------------------------------

SIZES = {"side by side": [0.0, 1e-20, 1.0, 1e30], "a zero row beside 1e20": [0.0, 1e20], "1e-20 beside 1e25": [1e-20, 1e25],
         "in runs of 40": [x for x in (1e-25, 1.0, 0.0, 1e15, 1e30) for _ in range(40)], "all near the floor": [1e-29, 3e-30],
         "all large": [1e35, 1e38, 1e36], "zeros": [0.0], "falling": list(10.0 ** np.linspace(38, -29, 200))}


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("lengths,kv,heads,dim,fmt", [([2, 5, 31], 1, 1, 32, "i8"), ([300, 1000], 2, 4, 64, "e4m3"),
                                                      ([20000], 1, 4, 32, "e4m3"), ([40000, 130], 1, 2, 128, "i8"),
                                                      ([(7 * i) % 150 for i in range(700)], 4, 4, 32, "i8")])
def test_open_rows_of_any_value_scale(be, lengths, kv, heads, dim, fmt, sizes, dtype):
    """Within a warp's cells, over the teams of a CTA, over parts, and a team a
    sequence: every row has its share of the sum, whatever the size of its values."""
    rng = np.random.default_rng(1)
    n = sum(lengths)
    size = np.resize(np.array(SIZES[sizes]), n)[:, None, None]
    values = np.clip(rng.normal(0, 1, (n, kv, dim)), -2, 2) * size
    b = filled(be, lengths, rng.normal(0, 1, (n, kv, dim)) * 0.5, values, fmt, dtype)
    few = range(0, 700, 23) if len(lengths) == 700 else range(len(lengths))
    a = Asked(b, [3 if s in few else 1 for s in range(len(lengths))], heads, dtype)
    close(a, a.attend())
    a.masks()
    close(a, a.attend(mask=True), mask=True)


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("sizes", [[1.0, 0.0], [1e-25, 1.0, 0.0], [0.0] * 70 + [1e-25] * 70, [1.0] * 70 + [1e3] + [1e-15] * 70])
def test_half_precision_over_rows_of_any_scale(be, sizes, mask):
    """f16 questions over banks that were written from f32."""
    rng = np.random.default_rng(4)
    n = 1300
    values = rng.normal(0, 1, (n, 2, 64)) * np.resize(np.array(sizes), n)[:, None, None]
    b = filled(be, [1000, 300], rng.normal(0, 1, (n, 2, 64)) * 0.5, values)
    a = Asked(b, [2, 9], 4, "f16")
    a.masks()
    got = a.attend(mask=mask)
    close(a, (np.where(np.abs(got[0]) < 2.0 ** -14, 0, got[0]), got[1]), mask=mask, least=2.0 ** -13)


@pytest.mark.parametrize("lengths", [[40], [4000], [30000]])
def test_shares_that_large_values_leave(be, lengths):
    """Rows that the mask's bias puts 2^-16 to 2^-60 below others, the large
    values among them: what they add counts beside what the others do."""
    rng = np.random.default_rng(2)
    n = lengths[0]
    size = np.resize(np.array([0.0, 1.0, 1e14, 1e28]), n)
    bias = np.resize(np.array([0.0, -3.0, -11.0, -41.0]), n)
    values = rng.normal(0, 1, (n, 1, 32)) * size[:, None, None]
    b = filled(be, lengths, rng.normal(0, 1, (n, 1, 32)) * 0.5, values)
    a = Asked(b, [6], 1)
    a.masks()
    a.mask = [np.tile(bias.astype(np.float32), (6, 1))]
    a.mask[0][3] = bias[::-1]
    a.mask[0][4, rng.random(n) < 0.8] = -1e30
    a.d_mask = cuda(a.mask[0].reshape(-1))
    close(a, a.attend(mask=True), mask=True)


# --- products ---------------------------------------------------------------------

FACTORS = [(2e37, 1e-36, 0.0), (1e38, 3e-38, 0.0), (3e37, 1e-44, 1e6), (1e-28, 1e36, 1e-8), (1e-20, 3e37, 1e-18), (1.0, 1e-30, 1e30),
           (1.0, 1e30, -1e-30), (1e20, 1e-25, 3e4), (1e-26, 1e-12, 1e38), (1e37, 1e2, 3e-39), (1.0, 1e-38, 1e38), (1e10, 1.0, 1e-10),
           (1e-28, 3e37, 0.0), (6e37, 8e-38, 0.0), (6e37, 4e-38, 0.0), (6e37, 2e-38, 0.0), (1e-3, 3e32, 1e-30)]


@pytest.mark.parametrize("dtype,size,ask,scale", [(t, *f) for f in FACTORS for t in ("f32", "bf16")
                                                  if t == "f32" or f[1] > 1e-40])  # below bf16's smallest
def test_scores_whose_factors_are_far_from_one(be, dtype, size, ask, scale):
    """Keys, questions and a scale that leave f32 two at a time, and whose product
    does not: attention and pointer scores. Beside what Asked.check counts, factors
    below 2^-126 are rounded to steps of 2^-149 (a question's) or of the least key
    scale's codes (in the cached keys already)."""
    rng = np.random.default_rng(6)
    lengths, dim = [3, 70, 400], 32
    n = sum(lengths)
    b = filled(be, lengths, rng.normal(0, 1, (n, 1, dim)) * size, rng.normal(0, 1, (n, 1, dim)))
    a = Asked(b, [2, 9, 3], 1, dtype, size=ask)
    a.masks()
    assert np.isfinite(a.q).all()
    for mask in (False, True):
        out, lse = a.attend(mask=mask, scale=scale)
        assert np.isfinite(out).all()
        close(a, (out, lse), scale=scale, mask=mask)
    scores = torch.full((int(a.mask_off[-1]),), 7.0, device="cuda")
    for mask in (False, True):
        torch.cuda.synchronize()
        be.cache_scores(b.cache, b.table, a.view, scores.data_ptr(), a.d_mask_off.data_ptr(),
                        a.d_mask.data_ptr() if mask else None, scale)
        be.synchronize()
        s = scores.cpu().numpy()
        sc = scale or float(np.float32(1 / np.sqrt(dim)))
        for i in range(a.total):
            q = a.seq[i]
            at = a.mask_off[q] + (i - a.off[q]) * lengths[q]
            k, x = b.keys[q][:, 0].astype(np.float64), a.q[i, 0].astype(np.float64)
            want, ok = ref.masked(k @ x * sc, a.mask[q][i - a.off[q]] if mask else np.zeros(lengths[q]))
            room = (np.abs(k) @ np.abs(x)) * abs(sc) * (dim * U + 2.0 ** -22) + 4 * U * (np.abs(want) + 16)
            assert (np.abs(s[at:at + lengths[q]] - want)[ok] <= room[ok]).all(), i
            assert (s[at:at + lengths[q]][~ok] == np.float32(-1e30)).all()


# --- small weights ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gap,mask", [(14.0, False), (22.0, True), (28.0, False), (45.0, True), (60.0, False)])
def test_the_tail_behind_one_leading_row(be, gap, mask, dtype):
    """One row whose score lies `gap` above 20000 others', its values zeros and then
    ones, under questions enough that each warp has every row. The tail's share is
    20000 e^-gap: beside zeros it is the output. Room is the header's: a weight is
    rounded to 22 bits (11) or to 2^-33 of the largest product of a weight and its value
    scale, a row of zeros counting with 2^-40."""
    n, dim, nq, heads = 20000, 32, 300, 128
    rng = np.random.default_rng(8)
    keys = np.zeros((n, 1, dim))
    values = rng.normal(1, 0.1, (n, 1, dim))
    lead = 777
    for value in (0.0, 1.0):
        keys[lead], values[lead] = 1.0, value
        b = filled(be, [n], keys, values)
        a = Asked(b, [nq], heads, dtype)
        q = torch.full_like(a.flat, gap / 32 * 32 ** 0.5)
        q.view(nq * heads, dim)[::7] *= 0.5  # rows of half the gap between
        a.flat.copy_(q)
        a.q = q.float().cpu().numpy().reshape(nq, heads, dim)
        some = [0, 1, 6, 150, 299]
        if mask:
            m = rng.normal(0, 0.5, (nq, n)).astype(np.float32)
            m[:, lead] = 0
            m[:, 1::3] = -1e30
            a.mask, a.mask_off = [m], offsets([nq * n])
            a.d_mask, a.d_mask_off = cuda(m.reshape(-1)), cuda(a.mask_off)
        out, lse = a.attend(mask=mask)
        k, v = (x[0][:, 0].astype(np.float64) for x in (b.keys, b.values))
        half = float(torch.finfo(TYPES[dtype]).eps) / 2
        weight = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -22
        sc = float(np.float32(1 / np.sqrt(dim)))
        for i in some:
            for h in (0, 1, 7, 64, 127):
                x = k @ a.q[i, h].astype(np.float64) * sc
                if mask:
                    x, ok = ref.masked(x, a.mask[0][i].astype(np.float64))
                    x = np.where(ok, x, -np.inf)
                p = np.exp(x - x.max())
                wl = x.max() + np.log(p.sum())
                p /= p.sum()
                want = p @ v
                # the scores, sums of 32 equal terms, and masks of up to 4 beside them; sums of n terms
                ds = gap * (dim * U + 2.0 ** -22) + 4 * U * (2 * gap + 16)
                rel = 4 * ds + weight + (n / 8 + 64) * U
                least = (p * np.maximum(np.abs(v).max(1), 127 * 2.0 ** -40)).max() * n * 2.0 ** -33
                assert abs(lse[i, h] - wl) <= 2 * ds + (n / 8 + 64) * U
                room = (p @ np.abs(v)) * rel + half * np.abs(want) + least
                if dtype == "f16":
                    room = room + 2.0 ** -25  # half its smallest step
                assert (np.abs(out[i, h] - want) <= room).all(), (value, i, h, out[i, h][:3], want[:3])
