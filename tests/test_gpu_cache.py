"""The bank cache against plain 64-bit forms: rows written and read back, block
bounds and their selection, attention and pointer scores, at lengths that end
inside a cell, a page and a part, under masks that leave a row nothing, at every
type, head layout and alignment."""
import numpy as np
import pytest

from krystal_b200 import BankCache, abi, policy
from krystal_b200 import cache as kc
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from tests import cache_cases as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LENGTHS = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 130, 200, 257]


@pytest.fixture(scope="module")
def be():
    cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
    b = CudaBrainBackend(cfg, create_brain_forward_weights(cfg, 1337), 0)
    yield b
    b.destroy()


def cuda(a, dtype=None):
    a = np.ascontiguousarray(a)
    a = a.astype({np.dtype(np.uint32): np.int32, np.dtype(np.uint64): np.int64}.get(a.dtype, a.dtype), copy=False)
    t = torch.from_numpy(a).cuda()
    return t if dtype is None else t.to(dtype)


def offsets(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int64)


class Bank:
    """A cache of sequences of given lengths, in shuffled pages, and what it holds."""

    def __init__(self, be, lengths, kv=4, dim=32, fmt="i8", seed=0, dtype="f32", spread=1.0, spare=3,
                 fill=0xA5):
        rng = np.random.default_rng(seed)
        self.be, self.lengths, self.kv, self.dim, self.fmt = be, list(lengths), kv, dim, fmt
        self.n = len(self.lengths)
        self.pitch = max(1, max(-(-n // 64) for n in self.lengths))
        count = self.n * self.pitch + spare
        self.pages = rng.permutation(count)[:self.n * self.pitch].reshape(self.n, self.pitch).astype(np.uint32)
        self.cache = BankCache(count, kv, dim, fmt, storage=torch.full(
            (BankCache.bytes_for(count, kv, dim),), fill, dtype=torch.uint8, device="cuda"))
        total = sum(self.lengths)
        x = rng.normal(0, 1, (2, total, kv, dim)) * np.exp(rng.normal(0, spread, (2, total, kv, 1)))
        x[:, ::29] = 0
        x = cuda(x.astype(np.float32), TYPES[dtype])
        host = x.float().cpu().numpy()
        off = offsets(self.lengths)
        k, v = ref.quantised(host[0], fmt), ref.quantised(host[1], fmt)
        self.keys = [k[off[s]:off[s + 1]] for s in range(self.n)]
        self.values = [v[off[s]:off[s + 1]] for s in range(self.n)]
        self.d = {"pages": cuda(self.pages), "lengths": cuda(np.array(self.lengths, np.uint32)), "off": cuda(off),
                  "x": x}
        self.table = kc.page_table(self.d["pages"].data_ptr(), self.d["lengths"].data_ptr(), self.n, self.pitch)
        torch.cuda.synchronize()
        if total:
            be.cache_write(self.cache, self.table, kc.cache_rows(x[0].data_ptr(), x[1].data_ptr(), dtype, total,
                                                                 self.d["off"].data_ptr()))
        be.synchronize()


class Asked:
    """Questions over a bank, and what the calls wrote."""

    def __init__(self, bank, counts, heads=None, dtype="f32", seed=1, pitch=0, shift=0, max_q=0, size=1.0):
        rng = np.random.default_rng(seed)
        self.bank, self.heads, self.dtype = bank, heads or bank.kv, dtype
        self.counts, self.total = list(counts), int(sum(counts))
        width = self.heads * bank.dim
        self.pitch = pitch or width
        flat = cuda((rng.normal(0, size, self.total * self.pitch + shift)).astype(np.float32), TYPES[dtype])
        self.flat, self.shift = flat, shift
        at = np.arange(self.total)[:, None] * self.pitch + np.arange(width)
        self.q = flat.float().cpu().numpy()[shift:][at].reshape(self.total, self.heads, bank.dim)
        self.off = offsets(self.counts)
        self.d_off = cuda(self.off)
        self.view = kc.questions(flat.data_ptr() + shift * flat.element_size(), dtype, self.total, self.heads,
                                 self.d_off.data_ptr(), max_q, pitch)
        self.seq = np.repeat(np.arange(bank.n), self.counts)

    def masks(self, seed=3, kind="mixed"):
        """A mask block a sequence: open entries with a bias, shut ones of every kind, some rows with nothing."""
        rng = np.random.default_rng(seed)
        rows, at = [], []
        for s, n in enumerate(self.counts):
            r = self.bank.lengths[s]
            m = rng.normal(0, 2, (n, r)).astype(np.float32)
            shut = rng.choice(np.array([-1e30, -np.inf, np.nan, -3.4028235e38, -1e29], np.float32), (n, r))
            m = np.where(rng.random((n, r)) < 0.6, shut, m)
            for i in range(n):
                if (i + s) % 4 == 1:
                    m[i] = rng.choice(np.array([-1e30, -np.inf, np.nan], np.float32), r)
            rows.append(m)
            at.append(n * r)
        self.mask = rows
        self.mask_off = offsets(at)
        flat = np.concatenate([m.reshape(-1) for m in rows]) if sum(at) else np.zeros(1, np.float32)
        self.d_mask, self.d_mask_off = cuda(flat), cuda(self.mask_off)

    def attend(self, mask=False, blocks=None, block_count=0, scale=0.0, out_pitch=0, lse=True, repeat=1):
        b, width = self.bank, self.heads * self.bank.dim
        op = out_pitch or width
        out = torch.full((max(1, self.total * op) + self.shift,), 7.0, dtype=TYPES[self.dtype], device="cuda")
        ls = torch.full((max(1, self.total), self.heads), 7.0, device="cuda")
        size = b.be.attend_workspace(b.cache, b.table, self.view, block_count)
        work = torch.full((max(16, size),), 0xFF, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for _ in range(repeat):
            b.be.cache_attend(b.cache, b.table, self.view, out.data_ptr() + self.shift * out.element_size(), out_pitch,
                              ls.data_ptr() if lse else None, self.d_mask.data_ptr() if mask else None,
                              self.d_mask_off.data_ptr() if mask else None,
                              blocks.data_ptr() if blocks is not None else None, block_count, scale, work.data_ptr(),
                              work.numel())
        b.be.synchronize()
        self.raw = out
        at = np.arange(self.total)[:, None] * op + np.arange(width)
        return out.float().cpu().numpy()[self.shift:][at].reshape(self.total, self.heads, b.dim), ls.cpu().numpy()

    def check(self, got, mask=False, lists=None, scale=0.0, seqs=None):
        """Every question against the 64-bit form. With u = 2^-23 the unit of an
        f32 sum that may truncate:
          a score is off by d u sum |q k| scale (its sum) plus 2^-22 of the same
          (22 bits of an f32 q; 16-bit types are exact) and 4 u of itself, of the
          mask's and of the value scale's logarithm (up to 2^7) it is added to;
          a weight by twice that (its own score and the maximum's) and by its
          rounding, 2^-22 or, for 16-bit questions, 2^-11; the sums of n weights
          by n / 8 + 64 steps of u; the output by half a step of its type."""
        out, lse = got
        b, u = self.bank, 2.0 ** -23
        sc = scale or float(np.float32(1 / np.sqrt(b.dim)))
        half = float(torch.finfo(TYPES[self.dtype]).eps) / 2
        weight = 2.0 ** -22 if self.dtype == "f32" else 2.0 ** -11
        for i in range(self.total):
            s = self.seq[i]
            if seqs is not None and s not in seqs:
                continue
            keys, values = b.keys[s], b.values[s]
            m = self.mask[s][i - self.off[s]] if mask else None
            rows = None
            if lists is not None:
                rows = [np.concatenate([np.arange(x * 64, min(len(keys), x * 64 + 64)) for x in li
                                        if x * 64 < len(keys)] + [np.zeros(0, int)]) for li in lists[i]]
            want, wl = ref.attend(self.q[i], keys, values, sc, m, rows)
            g = self.heads // b.kv
            for h in range(self.heads):
                if not np.isfinite(wl[h]):
                    assert (out[i, h] == 0).all() and lse[i, h] == -np.inf, (i, h)
                    continue
                k, v = keys[:, h // g].astype(np.float64), values[:, h // g].astype(np.float64)
                terms = (np.abs(k) @ np.abs(self.q[i, h]).astype(np.float64)).max() * abs(sc)
                big = abs(wl[h]) + terms + 128 + (0 if m is None else 16)
                ds = terms * (b.dim * u + 2.0 ** -22) + 4 * u * big
                n = len(keys) if rows is None else len(rows[h // g])
                assert abs(lse[i, h] - wl[h]) <= 2 * ds + (n / 8 + 64) * u, (i, h)
                room = np.abs(v).max() * (4 * ds + weight + (n / 8 + 64) * u) + half * np.abs(want[h])
                assert (np.abs(out[i, h] - want[h]) <= room + 1e-37).all(), (i, h, np.abs(out[i, h] - want[h]).max())


# --- write and read ------------------------------------------------------------

def read_all(bank, dtype="f32", starts=None, counts=None, shift=0, pitch=0):
    counts = bank.lengths if counts is None else counts
    total, width = int(sum(counts)), bank.kv * bank.dim
    p = pitch or width
    k = torch.full((total * p + shift + 1,), 7.0, dtype=TYPES[dtype], device="cuda")
    v = torch.full_like(k, 7.0)
    off = cuda(offsets(counts))
    st = cuda(np.array(starts, np.uint32)) if starts is not None else None
    step = k.element_size() * shift
    torch.cuda.synchronize()
    bank.be.cache_read(bank.cache, bank.table, kc.cache_rows(k.data_ptr() + step, v.data_ptr() + step, dtype, total,
                                                             off.data_ptr(), pitch), st.data_ptr() if starts else None)
    bank.be.synchronize()
    at = shift + np.arange(total)[:, None] * p + np.arange(width)
    return [x.float().cpu().numpy()[at].reshape(total, bank.kv, bank.dim) for x in (k, v)] + [k]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("kv,dim", [(4, 32), (1, 128), (3, 64), (8, 128)])
def test_rows_come_back_as_the_values_they_stand_for(be, kv, dim, fmt, dtype):
    b = Bank(be, LENGTHS, kv, dim, fmt, dtype=dtype)
    k, v, _ = read_all(b)
    assert np.array_equal(k, np.concatenate(b.keys)) and np.array_equal(v, np.concatenate(b.values))
    k16, v16, _ = read_all(b, dtype)
    assert np.array_equal(k16, torch.from_numpy(k).to(TYPES[dtype]).float().numpy())
    assert np.array_equal(v16, torch.from_numpy(v).to(TYPES[dtype]).float().numpy())
    got = b.cache.bounds().cpu().numpy()
    for s in range(b.n):
        for p, (lo, hi) in zip(b.pages[s], ref.bounds(b.keys[s])):
            assert np.array_equal(got[p, :, 0], lo) and np.array_equal(got[p, :, 1], hi), s


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kv,dim,fmt", [(4, 32, "i8"), (2, 64, "e4m3"), (1, 128, "i8")])
def test_a_bank_grows_turn_by_turn(be, kv, dim, fmt, dtype):
    """A record at a time and in runs that end anywhere: the cache is what one
    write of all the rows leaves, bounds too; then sequences are cut back and
    written on."""
    rng = np.random.default_rng(5)
    whole = Bank(be, [70, 200, 5], kv, dim, fmt, dtype=dtype)
    b = Bank(be, [70, 200, 5], kv, dim, fmt, dtype=dtype)
    b.cache.storage.fill_(0x5A)
    off, at = offsets(b.lengths), [0, 0, 0]
    x = b.d["x"]
    while at != b.lengths:
        n = [min(int(rng.choice([0, 1, 1, 3, 40, 64])), r - a) for r, a in zip(b.lengths, at)]
        rows = np.concatenate([np.arange(off[s] + at[s], off[s] + at[s] + n[s]) for s in range(3)]).astype(np.int64)
        at = [a + k for a, k in zip(at, n)]
        part = x[:, torch.from_numpy(rows).cuda()].contiguous()
        lengths, o = cuda(np.array(at, np.uint32)), cuda(offsets(n))
        torch.cuda.synchronize()
        be.cache_write(b.cache, kc.page_table(b.d["pages"].data_ptr(), lengths.data_ptr(), 3, b.pitch),
                       kc.cache_rows(part[0].data_ptr(), part[1].data_ptr(), dtype, len(rows), o.data_ptr()))
        be.synchronize()
    for s in range(3):
        for p in b.pages[s][:-(-b.lengths[s] // 64)]:
            assert torch.equal(b.cache.bounds()[p], whole.cache.bounds()[p])
    for one, other in zip(read_all(b)[:2], read_all(whole)[:2]):
        assert np.array_equal(one, other)
    # back to 66 rows and 4 other ones behind them: the bounds forget what was cut off
    lengths, o = cuda(np.array([70], np.uint32)), cuda(np.array([0, 4]))
    part = x[:, 100:104].contiguous()
    torch.cuda.synchronize()
    be.cache_write(b.cache, kc.page_table(b.d["pages"].data_ptr(), lengths.data_ptr(), 1, b.pitch),
                   kc.cache_rows(part[0].data_ptr(), part[1].data_ptr(), dtype, 4, o.data_ptr()))
    be.synchronize()
    keys = np.concatenate([b.keys[0][64:66], ref.quantised(part[0].float().cpu().numpy(), fmt)])
    got = b.cache.bounds()[int(b.pages[0][1])].cpu().numpy()
    assert np.array_equal(got[:, 0], keys.min(0)) and np.array_equal(got[:, 1], keys.max(0))


def test_one_row_a_sequence_needs_no_offsets(be):
    b = Bank(be, [1, 1, 1], 2, 64)
    x = b.d["x"] * 3
    torch.cuda.synchronize()
    be.cache_write(b.cache, b.table, kc.cache_rows(x[0].data_ptr(), x[1].data_ptr(), "f32", 3))
    out = torch.zeros_like(x)
    be.cache_read(b.cache, b.table, kc.cache_rows(out[0].data_ptr(), None, "f32", 3))
    be.synchronize()
    assert np.array_equal(out[0].cpu().numpy(), ref.quantised(x[0].cpu().numpy(), "i8"))
    assert bool((out[1] == 0).all())


@pytest.mark.parametrize("dtype,shift,more", [("f32", 1, 3), ("bf16", 1, 5), ("f16", 0, 8), ("f16", 3, 0)])
def test_rows_at_any_alignment_and_pitch(be, dtype, shift, more):
    lengths, kv, dim = [3, 0, 90, 64], 2, 64
    b = Bank(be, lengths, kv, dim, dtype=dtype)
    total, width = sum(lengths), kv * dim
    pitch = width + more
    flat = torch.full((2, total * pitch + shift), 3.0, dtype=TYPES[dtype], device="cuda")
    at = torch.from_numpy(shift + np.arange(total)[:, None] * pitch + np.arange(width)).cuda()
    flat[0, at], flat[1, at] = b.d["x"][0].flatten(1), b.d["x"][1].flatten(1)
    b.cache.storage.fill_(0x11)
    step = shift * flat.element_size()
    torch.cuda.synchronize()
    be.cache_write(b.cache, b.table, kc.cache_rows(flat[0].data_ptr() + step, flat[1].data_ptr() + step, dtype, total,
                                                   b.d["off"].data_ptr(), pitch))
    be.synchronize()
    k, v, raw = read_all(b, "f32", shift=shift, pitch=width + more)
    assert np.array_equal(k, np.concatenate(b.keys)) and np.array_equal(v, np.concatenate(b.values))
    untouched = np.ones(raw.numel(), bool)
    untouched[(shift + np.arange(total)[:, None] * (width + more) + np.arange(width)).reshape(-1)] = False
    assert (raw.cpu().numpy()[untouched] == 7.0).all()


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_extreme_rows(be, fmt):
    """Zeros, denormals, the floor of the scale, the largest f32, infinities and
    NaN, and values that lie half-way between two codes."""
    top = ref.TOP[fmt]
    rows = np.zeros((10, 1, 32), np.float32)
    rows[1, 0, :3] = [1e-45, -1e-40, 1e-38]
    rows[2, 0, :3] = [2.0 ** -100, -(2.0 ** -101), 3 * 2.0 ** -101]
    rows[3, 0, :3] = [3.4028235e38, -1e38, 1.0]
    rows[4, 0, :4] = [np.inf, -np.inf, np.nan, 1.0]
    rows[5, 0, :2] = [np.nan, np.nan]
    rows[6, 0] = np.concatenate([np.arange(31) + 0.5, [top]])
    rows[7, 0] = np.concatenate([-(np.arange(31) + 0.5) * 2.0 ** -9, [-top]])
    rows[8, 0] = np.nextafter(np.float32(1), np.float32(2)) * np.linspace(-top, top, 32)
    rows[9, 0, :2] = [-0.0, 5.0]
    b = Bank(be, [10], 1, 32, fmt)
    x = cuda(np.stack([rows, -rows]))
    torch.cuda.synchronize()
    be.cache_write(b.cache, b.table, kc.cache_rows(x[0].data_ptr(), x[1].data_ptr(), "f32", 10, b.d["off"].data_ptr()))
    be.synchronize()
    k, v, _ = read_all(b)
    assert np.array_equal(k, ref.quantised(rows, fmt)) and np.array_equal(v, ref.quantised(-rows, fmt))
    assert np.isfinite(k).all() and np.isfinite(b.cache.bounds()[int(b.pages[0][0])].cpu().numpy()).all()


def test_reads_from_anywhere_and_of_what_is_not_there(be):
    b = Bank(be, [100, 64, 0, 7], 2, 32)
    k, v, _ = read_all(b, starts=[60, 0, 0, 3], counts=[30, 64, 2, 9])
    pad = lambda x, n: np.concatenate([x, np.zeros((n - len(x), 2, 32), np.float32)])  # noqa: E731
    want = [b.keys[0][60:90], b.keys[1], pad(b.keys[2], 2), pad(b.keys[3][3:], 9)]
    assert np.array_equal(k, np.concatenate(want))


def test_pages_outside_the_cache_are_shut_out(be):
    """Bad page numbers: nothing is written outside, reads are 0, attention and
    scores pass the rows over."""
    b = Bank(be, [200, 130], 1, 64)
    before = b.cache.storage.clone()
    pages = b.pages.copy()
    pages[0, 1], pages[1, 0] = b.cache.pages, 0xFFFFFFFF
    bad = cuda(pages)
    table = kc.page_table(bad.data_ptr(), b.d["lengths"].data_ptr(), 2, b.pitch)
    torch.cuda.synchronize()
    be.cache_write(b.cache, table, kc.cache_rows(b.d["x"][0].data_ptr(), b.d["x"][1].data_ptr(), "f32", 330,
                                                 b.d["off"].data_ptr()))
    be.synchronize()
    assert torch.equal(b.cache.storage, before)
    good, b.table = b.table, table
    k = read_all(b)[0]
    want = np.concatenate(b.keys)
    want[64:128], want[200:264] = 0, 0
    assert np.array_equal(k, want)
    a = Asked(b, [2, 1])
    lists = [[[0, 2, 3]], [[0, 2, 3]], [[1, 2]]]
    a.check(a.attend(), lists=lists)
    off = offsets([2 * 200, 130])
    d_off, scores = cuda(off), torch.full((530,), 7.0, device="cuda")
    torch.cuda.synchronize()
    be.cache_scores(b.cache, table, a.view, scores.data_ptr(), d_off.data_ptr())
    blocks = torch.full((3, 1, 3), 9, dtype=torch.int32, device="cuda")
    be.cache_blocks(b.cache, table, a.view, 3, 0, blocks.data_ptr())
    be.synchronize()
    s = scores.cpu().numpy()
    assert (s[64:128] == np.float32(-1e30)).all() and (s[400:464] == np.float32(-1e30)).all()
    assert (s[:64] > -1e29).all() and (s[464:] > -1e29).all()
    assert 1 not in blocks[0].tolist()[0] and blocks[2].tolist()[0] == [0, 1, 2]
    b.table = good


# --- attention -------------------------------------------------------------------

@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,heads,dim,fmt", [(4, 4, 32, "i8"), (4, 4, 32, "e4m3"), (2, 8, 64, "i8"), (1, 7, 64, "e4m3"),
                                              (1, 1, 128, "i8"), (2, 6, 128, "e4m3")])
def test_attention_over_ragged_banks(be, kv, heads, dim, fmt, dtype, mask):
    b = Bank(be, LENGTHS, kv, dim, fmt, dtype=dtype)
    a = Asked(b, [1, 3, 0, 17, 1, 2, 33, 1, 0, 5, 16, 70, 2], heads, dtype)
    a.masks()
    a.check(a.attend(mask=mask), mask=mask)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kv,heads,dim,lengths", [(4, 4, 32, [5000, 1, 2049, 0]), (1, 8, 128, [9000]), (2, 2, 64, [20011, 64])])
def test_long_sequences_are_cut_and_joined(be, kv, heads, dim, lengths, dtype):
    b = Bank(be, lengths, kv, dim, "i8", dtype=dtype, spread=0.3)
    a = Asked(b, [2] * len(lengths), heads, dtype)
    a.masks()
    first = a.attend(mask=True)
    a.check(first, mask=True)
    a.check(a.attend())
    again = a.attend(mask=True, repeat=3)
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


@pytest.mark.parametrize("dtype,shift,more", [("f32", 1, 1), ("f16", 1, 3), ("bf16", 5, 8)])
def test_questions_at_any_alignment_and_pitch(be, dtype, shift, more):
    b = Bank(be, [50, 0, 300], 2, 64, dtype=dtype)
    width = 4 * 64
    a = Asked(b, [3, 1, 20], 4, dtype, pitch=width + more, shift=shift)
    a.check(a.attend(out_pitch=width + 2 * more))
    raw = a.raw.float().cpu().numpy()
    used = np.zeros(raw.size, bool)
    used[(shift + np.arange(24)[:, None] * (width + 2 * more) + np.arange(width)).reshape(-1)] = True
    assert (raw[~used] == 7.0).all()


@pytest.mark.parametrize("size", [1e-20, 30.0, 1e15])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_questions_of_any_size(be, size, dtype):
    """Scores that are all but equal, and scores of which one takes all: the
    tolerance follows their size."""
    b = Bank(be, [100, 400], 2, 64, dtype=dtype)
    a = Asked(b, [4, 4], 2, dtype, size=size)
    out, lse = a.attend()
    assert np.isfinite(out).all()
    if size < 1e3:
        a.check((out, lse))
    else:  # one row takes all, where no other is near
        for i in range(a.total):
            for h in range(2):
                k = b.keys[a.seq[i]][:, h].astype(np.float64) @ a.q[i, h].astype(np.float64)
                top = np.sort(k)[-2:]
                if top[1] - top[0] > 1e-4 * np.abs(k).max():
                    want = b.values[a.seq[i]][np.argmax(k), h]
                    half = float(torch.finfo(TYPES[dtype]).eps) / 2 + 2.0 ** -11
                    assert (np.abs(out[i, h] - want) <= half * np.abs(want)).all()


def test_value_scales_of_any_size(be):
    """Rows whose values differ by a factor of 1e60, and a large one that the
    mask shuts out: the small ones keep their digits."""
    for big in (1e30, 1e-28, 1.0):
        b = Bank(be, [130], 1, 32)
        x = torch.randn(2, 130, 1, 32, device="cuda")
        x[1] *= big
        x[1, 7] = 1e30
        torch.cuda.synchronize()
        be.cache_write(b.cache, b.table, kc.cache_rows(x[0].data_ptr(), x[1].data_ptr(), "f32", 130,
                                                       b.d["off"].data_ptr()))
        be.synchronize()
        b.keys, b.values = ([ref.quantised(y.cpu().numpy(), "i8")] for y in x)
        a = Asked(b, [5], 1)
        a.masks()
        for m in a.mask:
            m[:, 7] = -1e30
            m[:, 8] = 0.5
        a.d_mask = cuda(np.concatenate([m.reshape(-1) for m in a.mask]))
        got = a.attend(mask=True)
        b.values[0][7] = 0  # shut out: its size is not the tolerance's
        a.check(got, mask=True)


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("kv,heads,dim", [(4, 4, 32), (2, 8, 64), (1, 40, 128)])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_what_lies_behind_the_last_row_does_not_matter(be, kv, heads, dim, fmt, mask):
    """Storage that was never cleared: NaN codes (0x7f, 0xff), NaN and infinite
    scales behind a sequence's end and in its other rows' neighbours."""
    got = []
    for fill in (0x00, 0x7F, 0xFF):
        b = Bank(be, [0, 1, 37, 64, 100, 300], kv, dim, fmt, fill=fill)
        a = Asked(b, [2, 1, 9, 1, 20, 3], heads)
        a.masks()
        got.append(a.attend(mask=mask))
        one = Asked(b, [1] * 6, heads)
        lists = select(b, one, 3, 1)
        got[-1] += one.attend(blocks=lists, block_count=3) + (lists.cpu().numpy(),)
    a.check(got[0][:2], mask=mask)
    for other in got[1:]:
        for x, y in zip(got[0], other):
            assert np.array_equal(x, y)


def test_masks_beyond_1e29_and_short_masks(be):
    b = Bank(be, [70], 2, 32)
    a = Asked(b, [3])
    a.masks()
    m = np.zeros((3, 70), np.float32)
    m[0, [3, 60]] = [np.inf, 3e38]     # both count as 1e29: nothing beside them, their scores share
    m[1, 5] = -9.9e28                  # open, and nothing beside the others
    m[2] = -1e30
    m[2, 69] = -9.9e28                 # the only one that is open takes all
    a.mask = [m]
    a.d_mask = cuda(m.reshape(-1))
    out, lse = a.attend(mask=True)
    # exp(s + 1e29) / sum exp(s' + 1e29) = exp(s) / sum exp(s'): what is added to all of them cancels
    want = np.stack([ref.attend(a.q[0], b.keys[0][[3, 60]], b.values[0][[3, 60]], float(np.float32(32 ** -0.5)))[0]])[0]
    assert np.allclose(out[0], want, atol=2.0 ** -16 * np.abs(b.values[0]).max())
    assert np.allclose(out[2], b.values[0][69], atol=2.0 ** -20 * np.abs(b.values[0]).max())
    # a mask of 40 entries a question: rows behind its end are shut out
    short = np.zeros((3, 40), np.float32)
    short[0, 3] = np.nan
    a.mask = [short]
    a.d_mask, a.d_mask_off = cuda(short.reshape(-1)), cuda(np.array([0, 120]))
    got = a.attend(mask=True)
    b.keys[0], b.values[0] = b.keys[0][:40], b.values[0][:40]
    a.check(got, mask=True)


def test_questions_beyond_the_bound_and_behind_the_last_are_left(be):
    b = Bank(be, [90, 20], 2, 32)
    a = Asked(b, [40, 40], 2, max_q=20)
    got = a.attend()
    left = np.concatenate([np.arange(20, 40), np.arange(60, 80)])
    assert (got[0][left] == 7.0).all() and (got[1][left] == 7.0).all()
    full = Asked(b, [40, 40], 2).attend()
    for x, y in zip(got, full):
        x[left] = y[left]
    a.check(got)
    # more questions than the offsets name
    a = Asked(b, [3, 2], 2)
    a.view.questions = 5
    a.d_off.copy_(cuda(np.array([0, 3, 4])))
    out, lse = a.attend()
    assert (out[4] == 7.0).all() and (lse[4] == 7.0).all() and (out[:4] != 7.0).any()


def test_lengths_beyond_the_bound(be):
    """max_length bounds a sequence: rows behind it are not attended."""
    b = Bank(be, [150, 40], 2, 32)
    b.table.max_length = 100
    a = Asked(b, [2, 2], 2)
    got = a.attend()
    b.keys[0], b.values[0] = b.keys[0][:100], b.values[0][:100]
    a.check(got)


# --- blocks ------------------------------------------------------------------------

def select(bank, a, count, recent):
    out = torch.full((max(1, a.total), bank.kv, count), 77, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    bank.be.cache_blocks(bank.cache, bank.table, a.view, count, recent, out.data_ptr())
    bank.be.synchronize()
    return out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("count,recent", [(1, 0), (1, 1), (3, 1), (8, 2), (40, 40), (100, 0)])
@pytest.mark.parametrize("kv,heads,dim,fmt", [(4, 4, 32, "i8"), (2, 8, 64, "e4m3"), (1, 3, 128, "i8")])
def test_blocks_are_those_of_the_highest_bounds(be, kv, heads, dim, fmt, count, recent, dtype):
    b = Bank(be, [0, 1, 64, 65, 700, 2500], kv, dim, fmt, dtype=dtype)
    a = Asked(b, [2, 1, 0, 3, 2, 19], heads, dtype)
    got = select(b, a, count, recent)
    lists = got.cpu().numpy().astype(np.uint32)
    for i in range(a.total):
        score = ref.block_scores(a.q[i], ref.bounds(b.keys[a.seq[i]]) or [np.zeros((2, kv, dim))] * 0) \
            if b.lengths[a.seq[i]] else np.zeros((kv, 0))
        for h in range(kv):
            assert lists[i, h].tolist() == ref.chosen(score[h], count, recent), (i, h)
    a.masks()
    for mask in (False, True):
        a.check(a.attend(mask=mask, blocks=got, block_count=count), mask=mask,
                lists=[[[int(x) for x in row if x != ref.NONE] for row in lists[i]] for i in range(a.total)])


def test_equal_bounds_go_to_the_lowest_block(be):
    b = Bank(be, [64 * 40], 1, 32)
    x = torch.randn(1, 64, 1, 32, device="cuda").expand(40, 64, 1, 32).reshape(2560, 1, 32).contiguous()
    torch.cuda.synchronize()
    be.cache_write(b.cache, b.table, kc.cache_rows(x.data_ptr(), x.data_ptr(), "f32", 2560, b.d["off"].data_ptr()))
    got = select(b, Asked(b, [3]), 5, 2)
    assert got.cpu().tolist() == [[[0, 1, 2, 38, 39]]] * 3
    # a question of zeros, of either sign, is a tie of all
    a = Asked(b, [2])
    a.flat[:32], a.flat[32:64] = 0.0, -0.0
    assert select(b, a, 3, 0).cpu().tolist() == [[[0, 1, 2]]] * 2


def test_lists_with_repeats_and_numbers_outside(be):
    b = Bank(be, [300, 64, 0], 2, 32)
    a = Asked(b, [2, 1, 1], 4)
    lists = np.array([[[4, 1, 1, 9], [ref.NONE, 0, 0, 0]], [[5, 6, 7, ref.NONE], [2, 3, 1, 0]],
                      [[0, 0, 1, 1], [1, 1, 1, 1]], [[0, 1, 2, 3], [0, 0, 0, 0]]], np.uint32)
    got = a.attend(blocks=cuda(lists), block_count=4)
    a.check(got, lists=[[[int(x) for x in row] for row in lists[i]] for i in range(4)])


@pytest.mark.parametrize("dtype,heads,count,mask", [("f32", 4, 20, False), ("bf16", 8, 40, False), ("f16", 4, 32, True)])
def test_lists_of_many_short_sequences(be, dtype, heads, count, mask):
    """Lists longer than their sequences: holes, repeats and numbers outside at any place, or nothing at all."""
    b = Bank(be, [(37 * i) % 131 for i in range(210)], 4, 32, dtype=dtype)
    a = Asked(b, [3 + i % 2 for i in range(210)], heads, dtype)
    a.masks()
    rng = np.random.default_rng(count)
    lists = rng.integers(0, 4, (a.total, 4, count)).astype(np.uint32)
    lists[rng.random(lists.shape) < 0.8] = ref.NONE
    lists[:, 1, 5:] = ref.NONE
    lists[:, 2, :-1] = ref.NONE
    lists[::7, 3] = ref.NONE
    a.check(a.attend(mask=mask, blocks=cuda(lists), block_count=count), mask=mask, lists=lists.tolist())


def test_long_lists_are_cut_and_joined(be):
    b = Bank(be, [64 * 700 + 3], 1, 64, spread=0.3)
    a = Asked(b, [1], 4, "f16")
    rng = np.random.default_rng(2)
    lists = np.sort(rng.permutation(701)[:600]).reshape(1, 1, 600).astype(np.uint32)
    a.check(a.attend(blocks=cuda(lists), block_count=600), lists=lists.tolist())


# --- scores ------------------------------------------------------------------------

@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,fmt", [(32, "i8"), (64, "e4m3"), (128, "i8"), (128, "e4m3")])
def test_pointer_scores(be, dim, fmt, dtype, mask):
    b = Bank(be, LENGTHS + [1000], 1, dim, fmt, dtype=dtype)
    a = Asked(b, [1, 3, 0, 17, 1, 2, 33, 1, 0, 5, 16, 70, 2, 9], 1, dtype)
    a.masks()
    scores = torch.full((int(a.mask_off[-1]) + 5,), 7.0, device="cuda")
    torch.cuda.synchronize()
    be.cache_scores(b.cache, b.table, a.view, scores.data_ptr(), a.d_mask_off.data_ptr(),
                    a.d_mask.data_ptr() if mask else None)
    be.synchronize()
    s = scores.cpu().numpy()
    assert (s[-5:] == 7.0).all()
    sc, u = float(np.float32(1 / np.sqrt(dim))), 2.0 ** -23
    for i in range(a.total):
        q = a.seq[i]
        n, at = b.lengths[q], a.mask_off[q] + (i - a.off[q]) * b.lengths[q]
        k = b.keys[q][:, 0].astype(np.float64)
        x = k @ a.q[i, 0].astype(np.float64) * sc
        m = a.mask[q][i - a.off[q]].astype(np.float64) if mask else np.zeros(n)
        x, ok = ref.masked(x, m)
        got = s[at:at + n]
        assert (got[~ok] == np.float32(-1e30)).all()
        # a sum of d terms that may truncate, 22 bits of an f32 q, and the mask added
        room = (np.abs(k) @ np.abs(a.q[i, 0]).astype(np.float64)) * sc * (dim * u + 2.0 ** -22)
        room += 4 * u * (np.abs(x) + np.abs(np.where(ok, m, 0)))
        assert (np.abs(got - x)[ok] <= room[ok]).all(), i


def test_score_rows_longer_or_shorter_than_the_bank(be):
    """Rows of 100 over banks of 70 and 130: -1e30 behind the bank's end, no more
    than 100 of the longer one."""
    b = Bank(be, [70, 130], 1, 128)
    a = Asked(b, [2, 1], 1)
    full = torch.zeros(270, device="cuda")
    off = cuda(np.array([0, 140, 270]))
    rows, off2 = torch.full((300,), 7.0, device="cuda"), cuda(np.array([0, 200, 300]))
    torch.cuda.synchronize()
    be.cache_scores(b.cache, b.table, a.view, full.data_ptr(), off.data_ptr())
    be.cache_scores(b.cache, b.table, a.view, rows.data_ptr(), off2.data_ptr())
    be.synchronize()
    f, r = full.cpu().numpy(), rows.cpu().numpy()
    assert np.array_equal(r[:70], f[:70]) and np.array_equal(r[100:170], f[70:140])
    assert (r[70:100] == np.float32(-1e30)).all() and (r[170:200] == np.float32(-1e30)).all()
    assert np.array_equal(r[200:300], f[140:240])


# --- together ------------------------------------------------------------------------

def test_a_turn_over_a_cached_bank(be):
    """Write, score, draw, select, attend: captured once, replayed on another
    turn's rows, questions and lengths, beside a second graph of its own buffers;
    each replay is what the calls give one by one."""
    rng = np.random.default_rng(11)

    class Turn:
        def __init__(self, seed):
            self.n, self.kv, self.dim, self.pitch = 3, 1, 128, 5
            self.cache = BankCache(20, 1, 128, storage=torch.zeros(BankCache.bytes_for(20, 1, 128), dtype=torch.uint8,
                                                                  device="cuda"))
            z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
            self.pages = cuda(rng.permutation(20)[:15].reshape(3, 5).astype(np.uint32))
            self.lengths, self.row_off, self.q_off, self.off = (z(3, t=torch.int32), *(z(4, t=torch.int64) for _ in range(3)))
            self.x, self.q, self.u = z(2, 400, 1, 128), z(12, 1, 128), z(12, t=torch.float64)
            self.scores, self.index, self.logp = z(12 * 320), z(12, t=torch.int32), z(12)
            self.blocks, self.out, self.lse, self.back = z(12, 1, 2, t=torch.int32), z(12, 1, 128), z(12, 1), z(400, 1, 128)
            self.table = kc.page_table(self.pages.data_ptr(), self.lengths.data_ptr(), 3, 5)
            self.ask = kc.questions(self.q.data_ptr(), "f32", 12, 1, self.q_off.data_ptr(), 6)
            self.work = z(max(16, be.attend_workspace(self.cache, self.table, self.ask, 2)), t=torch.uint8)
            self.fill(seed)

        def fill(self, seed):
            g = np.random.default_rng(seed)
            lengths, q = g.integers(0, 321, 3), g.integers(0, 5, 3)
            new = np.minimum(lengths, g.integers(1, 130, 3))
            self.lengths.copy_(cuda(lengths.astype(np.uint32)))
            self.row_off.copy_(cuda(offsets(new)))
            self.q_off.copy_(cuda(offsets(q)))
            self.off.copy_(cuda(offsets(q * lengths)))
            self.x.copy_(cuda(g.normal(0, 1, (2, 400, 1, 128)).astype(np.float32)))
            self.q.copy_(cuda(g.normal(0, 1, (12, 1, 128)).astype(np.float32)))
            self.u.copy_(cuda(g.random(12)))

        def calls(self):
            be.cache_write(self.cache, self.table, kc.cache_rows(self.x[0].data_ptr(), self.x[1].data_ptr(), "f32", 400,
                                                                 self.row_off.data_ptr()))
            be.cache_read(self.cache, self.table, kc.cache_rows(None, self.back.data_ptr(), "f32", 400,
                                                                self.row_off.data_ptr()))
            be.cache_scores(self.cache, self.table, self.ask, self.scores.data_ptr(), self.off.data_ptr())
            be.draw(policy.ragged_rows(self.scores.data_ptr(), "f32", 12, 3, self.q_off.data_ptr(), self.off.data_ptr(),
                                       320), policy.Sampling(0.8, top_k=20), self.u.data_ptr(),
                    index=self.index.data_ptr(), logp=self.logp.data_ptr())
            be.cache_blocks(self.cache, self.table, self.ask, 2, 1, self.blocks.data_ptr())
            be.cache_attend(self.cache, self.table, self.ask, self.out.data_ptr(), lse=self.lse.data_ptr(),
                            blocks=self.blocks.data_ptr(), block_count=2, workspace=self.work.data_ptr(),
                            workspace_bytes=self.work.numel())

        def results(self):
            return [t.clone() for t in (self.cache.storage, self.back, self.scores, self.index, self.logp, self.blocks,
                                        self.out, self.lse)]

    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    try:
        turns = [Turn(1), Turn(2)]
        torch.cuda.synchronize()
        graphs = []
        for t in turns:
            with torch.cuda.stream(stream):
                t.calls()  # before the capture
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                t.calls()
            graphs.append(g)
        for seed in (3, 4, 5):
            starts = [t.cache.storage.clone() for t in turns]
            for k, t in enumerate(turns):
                t.fill(seed * 10 + k)
            torch.cuda.synchronize()
            other = torch.cuda.Stream()
            graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()  # both at once, on two streams
            torch.cuda.synchronize()
            got = [t.results() for t in turns]
            for t, st in zip(turns, starts):
                t.cache.storage.copy_(st)
            torch.cuda.synchronize()
            for t, g in zip(turns, got):
                t.calls()
                torch.cuda.synchronize()
                for x, y in zip(t.results(), g):
                    assert torch.equal(x, y) or torch.equal(x.nan_to_num(0, 0, 0), y.nan_to_num(0, 0, 0))
        del graphs
    finally:
        be.set_stream(None)


def test_a_cut_sequence_in_a_graph(be):
    """The join follows the parts it was launched behind, in a graph too, and the
    workspace is the graph's."""
    stream = torch.cuda.Stream()
    b = Bank(be, [9000, 40], 1, 64, spread=0.3)
    a = Asked(b, [1, 1], 4)
    out, lse = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 4, device="cuda")
    size = be.attend_workspace(b.cache, b.table, a.view)
    assert size > 0
    work = torch.zeros(size, dtype=torch.uint8, device="cuda")
    after = torch.zeros_like(out)
    torch.cuda.synchronize()
    be.set_stream(stream.cuda_stream)
    try:
        def call():
            be.cache_attend(b.cache, b.table, a.view, out.data_ptr(), lse=lse.data_ptr(), workspace=work.data_ptr(),
                            workspace_bytes=size)
        with torch.cuda.stream(stream):
            call()
            after.copy_(out)  # what follows the call follows its join
        torch.cuda.synchronize()
        assert torch.equal(after, out)
        a.check((out.cpu().numpy(), lse.cpu().numpy()))
        first = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            call()
            after.copy_(out)
        for _ in range(5):
            out.zero_()
            after.zero_()
            work.fill_(0xFF)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(after, first)
        with pytest.raises(abi.KrystalCudaError, match="workspace"):
            be.cache_attend(b.cache, b.table, a.view, out.data_ptr(), workspace=work.data_ptr(), workspace_bytes=size - 16)
        del g
    finally:
        be.set_stream(None)


def test_offsets_past_32_bits(be):
    """A cache of 5 GB whose last pages hold the rows, and a mask and scores
    behind 2^32 bytes."""
    kv, dim = 8, 128
    count = 5 * (1 << 30) // BankCache.bytes_for(1, kv, dim)
    b = Bank(be, [100, 70], kv, dim)
    big = BankCache(count, kv, dim)
    pages = cuda((count - 1 - np.arange(b.n * b.pitch)).reshape(b.n, b.pitch).astype(np.uint32))
    b.cache, b.d["pages"] = big, pages
    b.table = kc.page_table(pages.data_ptr(), b.d["lengths"].data_ptr(), b.n, b.pitch)
    torch.cuda.synchronize()
    be.cache_write(big, b.table, kc.cache_rows(b.d["x"][0].data_ptr(), b.d["x"][1].data_ptr(), "f32", 170,
                                               b.d["off"].data_ptr()))
    be.synchronize()
    k, v, _ = read_all(b)
    assert np.array_equal(k, np.concatenate(b.keys)) and np.array_equal(v, np.concatenate(b.values))
    a = Asked(b, [3, 2], 16)
    a.masks()
    far = (1 << 30) + 12345
    room = torch.empty(far + int(a.mask_off[-1]), device="cuda")
    room[far:] = a.d_mask
    a.d_mask, a.d_mask_off = room, cuda(a.mask_off + far)
    a.check(a.attend(mask=True), mask=True)
    got = select(b, a, 1, 0).cpu().numpy()
    for i in range(a.total):
        score = ref.block_scores(a.q[i], ref.bounds(b.keys[a.seq[i]]))
        assert [got[i, h].tolist() for h in range(kv)] == [ref.chosen(score[h], 1, 0) for h in range(kv)]
    one = Bank(be, [300], 1, 128)
    q = Asked(one, [2], 1)
    off = cuda(np.array([far, far + 600]))
    room.fill_(7.0)
    torch.cuda.synchronize()
    be.cache_scores(one.cache, one.table, q.view, room.data_ptr(), off.data_ptr())
    be.synchronize()
    assert bool((room[:far] == 7.0).all()) and bool((room[far:far + 600] != 7.0).all())


def test_refusals(be):
    b = Bank(be, [70, 5], 2, 64)
    a = Asked(b, [2, 1], 4)
    x, p = b.d["x"], lambda t: t.data_ptr()
    out = torch.zeros(3, 4, 64, device="cuda")
    good = dict(cache=b.cache, table=b.table, questions=a.view, out=p(out))

    def refused(match, call, *args, **kw):
        with pytest.raises(abi.KrystalCudaError, match=match):
            call(*args, **kw)

    rows = lambda **kw: kc.cache_rows(**{"keys": p(x), "values": p(x), "dtype": "f32", "rows": 75,  # noqa: E731
                                         "row_off": p(b.d["off"]), **kw})
    for write in (lambda r: be.cache_write(b.cache, b.table, r), lambda r: be.cache_read(b.cache, b.table, r)):
        refused("pitch is smaller", write, rows(pitch=127))
        refused("one row a sequence", write, rows(row_off=None))
        refused("aligned", write, rows(keys=p(x) + 1))
        refused("aligned", write, rows(row_off=p(b.d["off"]) + 4))
        refused("f32, f16 or bf16", write, rows(dtype="f64"))
    refused("keys and values", be.cache_write, b.cache, b.table, rows(values=None))
    refused("keys or values", be.cache_read, b.cache, b.table, rows(values=None, keys=None))
    refused("2147483647", be.cache_write, b.cache, b.table, rows(rows=1 << 31))
    for field, value, match in [("format", 5, "i8 or e4m3"), ("head_dim", 48, "32, 64 or 128"), ("kv_heads", 0, "1 to 128"),
                                ("pages", 0, "without pages"), ("bytes", 100, "smaller than"), ("storage", None, "16-byte"),
                                ("storage", p(b.cache.storage) + 8, "16-byte")]:
        old = getattr(b.cache.view, field)
        setattr(b.cache.view, field, value)
        refused(match, be.cache_attend, **good)
        assert be.attend_workspace(b.cache, b.table, a.view) == 0
        setattr(b.cache.view, field, old)
    for bad, match in [(kc.page_table(None, p(b.d["lengths"]), 2, 2), "needs its pages"),
                       (kc.page_table(p(b.d["pages"]), None, 2, 2), "needs its pages"),
                       (kc.page_table(p(b.d["pages"]) + 2, p(b.d["lengths"]), 2, 2), "4-byte"),
                       (kc.page_table(p(b.d["pages"]), p(b.d["lengths"]), 2, 2, 129), "longer than the table")]:
        refused(match, be.cache_attend, **{**good, "table": bad})
    ask = lambda **kw: kc.questions(**{"q": p(a.flat), "dtype": "f32", "questions": 3, "heads": 4,  # noqa: E731
                                       "q_off": p(a.d_off), **kw})
    for kw, match in [(dict(heads=3), "multiple of kv_heads"), (dict(heads=0), "multiple"), (dict(heads=2048), "multiple"),
                      (dict(pitch=255), "pitch is smaller"), (dict(q_off=None), "one question a sequence"),
                      (dict(q=None), "no values"), (dict(q=p(a.flat) + 2), "aligned"), (dict(dtype="f64"), "f32, f16 or bf16"),
                      (dict(questions=0x7fffffff), "2147483647")]:
        refused(match, be.cache_attend, **{**good, "questions": ask(**kw)})
    for kw, match in [(dict(out=None), "an output"), (dict(out_pitch=255), "pitch is smaller"), (dict(mask=p(out)), "offsets"),
                      (dict(block_count=2), "list of blocks"), (dict(blocks=p(out)), "list of blocks"),
                      (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(out=p(out) + 1), "aligned"),
                      (dict(out=p(a.flat)), "over its questions"), (dict(lse=p(out) + 2), "aligned"),
                      (dict(workspace=p(out) + 4), "16 bytes")]:
        refused(match, be.cache_attend, **{**good, **kw})
    blocks = torch.zeros(3, 2, 2, dtype=torch.int32, device="cuda")
    refused("at least one block", be.cache_blocks, b.cache, b.table, a.view, 0, 0, p(blocks))
    refused("at most count", be.cache_blocks, b.cache, b.table, a.view, 2, 3, p(blocks))
    refused("must be there", be.cache_blocks, b.cache, b.table, a.view, 2, 1, None)
    wide = kc.page_table(p(b.d["pages"]), p(b.d["lengths"]), 2, 30000)
    refused("KC_CACHE_MAX_SELECT", be.cache_blocks, b.cache, wide, a.view, 2, 1, p(blocks))
    refused("one head", be.cache_scores, b.cache, b.table, a.view, p(out), p(a.d_off))
    one = Bank(be, [70, 5], 1, 128)
    q = Asked(one, [2, 1], 1)
    refused("their offsets", be.cache_scores, one.cache, one.table, q.view, p(out), None)
    refused("their offsets", be.cache_scores, one.cache, one.table, q.view, None, p(a.d_off))
    refused("aligned", be.cache_scores, one.cache, one.table, q.view, p(out) + 2, p(a.d_off))
    # nothing to do is no error, and the handle goes on
    empty = kc.page_table(None, None, 0, 0)
    be.cache_write(b.cache, empty, kc.cache_rows(None, None, "f32", 0))
    be.cache_attend(b.cache, empty, kc.questions(None, "f32", 0, 2), out=None)
    a.check(a.attend())


def test_a_dropped_cache_stays_until_the_stream_has_passed(be):
    """A cache that is dropped while its write is queued: another tensor that
    takes memory at once does not get the storage."""
    x = torch.randn(2, 6400, 4, 32, device="cuda")
    lengths, pages = cuda(np.array([6400], np.uint32)), cuda(np.arange(100, dtype=np.uint32))
    off = cuda(np.array([0, 6400]))
    table = kc.page_table(pages.data_ptr(), lengths.data_ptr(), 1, 100)
    back = torch.zeros_like(x[0])
    cache = BankCache(100)
    torch.cuda.synchronize()
    for _ in range(20):
        be.cache_write(cache, table, kc.cache_rows(x[0].data_ptr(), x[1].data_ptr(), "f32", 6400, off.data_ptr()))
    be.cache_read(cache, table, kc.cache_rows(back.data_ptr(), None, "f32", 6400, off.data_ptr()))
    size, at = cache.storage.numel(), cache.storage.data_ptr()
    del cache
    taken = [torch.full((size,), 1, dtype=torch.uint8, device="cuda") for _ in range(3)]
    assert all(t.data_ptr() != at for t in taken)
    be.synchronize()
    assert np.array_equal(back.cpu().numpy(), ref.quantised(x[0].cpu().numpy(), "i8"))
