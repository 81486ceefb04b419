"""The forms that the bank cache's launches take at the sizes they are made for:
batches of many short sequences, selection by clusters and over the longest
sequences, writes behind gaps, sequences of hundreds of parts."""
import numpy as np
import pytest

from krystal_b200 import cache as kc
from tests import cache_cases as ref
from tests.test_gpu_cache import Asked, Bank, be, cuda, offsets, read_all, select  # noqa: F401 (be: the fixture)
from tests.test_gpu_cache_range import close, filled

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# --- attention: a team of warps a unit -----------------------------------------------

@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("kv,heads,dim,dtype,most", [(4, 4, 32, "f32", 8), (4, 4, 32, "f32", 16), (4, 4, 32, "bf16", 32),
                                                     (4, 8, 32, "f32", 30), (2, 8, 64, "f16", 5), (2, 2, 64, "f32", 9),
                                                     (1, 4, 128, "bf16", 13), (4, 4, 32, "f16", 100)])
def test_a_team_a_unit(be, kv, heads, dim, dtype, most, mask):
    """Enough sequences of at most 512 rows that each has a team of 1 to 8 warps to
    itself, of one tile and of two; some have no rows, some no questions."""
    n = 2400 // kv + 7
    b = Bank(be, [(53 * i) % 513 for i in range(n)], kv, dim, dtype=dtype, spare=0)
    a = Asked(b, [(7 * i) % (most + 1) for i in range(n)], heads, dtype, max_q=most)
    a.masks()
    got = a.attend(mask=mask)
    some = set(range(3, n, max(1, n * most // 250)))
    a.check(got, mask=mask, seqs=some)
    again = a.attend(mask=mask)
    assert np.array_equal(got[0], again[0]) and np.array_equal(got[1], again[1])
    assert np.isfinite(got[0]).all() and ((got[1] > -50) | (got[1] == -np.inf)).all()


def test_a_team_a_unit_over_rows_of_any_scale(be):
    """Teams of two warps whose cells go over to the general form at different places."""
    n = 620
    lengths = [(31 * i) % 400 for i in range(n)]
    rng = np.random.default_rng(3)
    total = sum(lengths)
    size = np.where(rng.random(total) < 0.01, 10.0 ** rng.uniform(-28, 30, total), np.where(rng.random(total) < 0.1, 0.0, 1.0))
    b = filled(be, lengths, rng.normal(0, 1, (total, 4, 32)), rng.normal(0, 1, (total, 4, 32)) * size[:, None, None])
    a = Asked(b, [1 + (5 * i) % 24 if i % 20 == 7 else 1 for i in range(n)], 4, max_q=24)
    close(a, a.attend())
    a.masks()
    close(a, a.attend(mask=True), mask=True)


# --- attention: hundreds of parts ------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("sizes", [[1.0], [0.0, 1.0, 1e-15, 1.0, 3e4], [1.0] * 100000 + [1e-20] * 100000 + [0.0] * 90000])
def test_hundreds_of_parts(be, sizes, dtype):
    """300003 rows: more parts than the joining warps take in one go."""
    rng = np.random.default_rng(5)
    n = 300003
    values = rng.normal(0, 1, (n, 1, 32)) * np.resize(np.array(sizes), n)[:, None, None]
    b = filled(be, [n], rng.normal(0, 1, (n, 1, 32)), values)
    a = Asked(b, [1], 3, dtype)
    got = a.attend()
    close(a, got, least=1e-37 if dtype == "f32" else 2.0 ** -25)
    again = a.attend()
    assert np.array_equal(got[0], again[0]) and np.array_equal(got[1], again[1])


# --- blocks ------------------------------------------------------------------------------

@pytest.mark.parametrize("pages,kv,heads,dim,dtype,count,recent,asks",
                         [(256, 1, 1, 32, "f32", 16, 1, 5), (300, 2, 8, 64, "bf16", 40, 0, 9), (600, 1, 4, 128, "f16", 64, 2, 3),
                          (1100, 1, 1, 32, "f32", 7, 7, 11), (1100, 1, 2, 32, "bf16", 300, 2, 16), (3201, 1, 1, 32, "f32", 50, 1, 9),
                          (6007, 2, 2, 32, "f16", 33, 3, 8), (25600, 1, 1, 32, "f32", 100, 1, 2), (25600, 1, 1, 128, "f32", 3, 0, 1),
                          (13000, 1, 1, 64, "bf16", 2000, 5, 3)])
def test_blocks_of_long_sequences(be, pages, kv, heads, dim, dtype, count, recent, asks):
    """Scores by clusters of 2, 4 and 8 CTAs, up to KC_CACHE_MAX_SELECT rows. A few
    hundred pages are named again and again, so that most scores have equals: they go to the
    lowest block. Beside it a short sequence."""
    held = 250
    b = Bank(be, [held * 64], kv, dim, dtype=dtype)
    rng = np.random.default_rng(pages)
    names = np.stack([rng.integers(0, held, pages), np.zeros(pages, np.int64)])
    names[1, :3] = [5, 9, 2]
    lengths = np.array([pages * 64 - 13, 130], np.uint32)
    d = [cuda(b.pages[0][names].astype(np.uint32)), cuda(lengths)]
    table = kc.page_table(d[0].data_ptr(), d[1].data_ptr(), 2, pages)
    a = Asked(b, [asks], heads, dtype)
    both, off = kc.questions(a.flat.data_ptr(), dtype, asks, heads, None, 0), cuda(np.array([0, asks - 1, asks]))
    both.q_off = off.data_ptr()
    out = torch.full((asks, kv, count), 77, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.cache_blocks(b.cache, table, both, count, recent, out.data_ptr())
    be.synchronize()
    got = out.cpu().numpy().astype(np.uint32)
    bounds = ref.bounds(b.keys[0])
    for i in range(asks):
        score = ref.block_scores(a.q[i], bounds)
        for h in range(kv):
            row = score[h][names[0]] if i < asks - 1 else score[h][names[1, :3]]
            assert got[i, h].tolist() == ref.chosen(row, count, recent), (i, h)


# --- writes ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,kv,dim", [("f32", 4, 32), ("bf16", 1, 128)])
@pytest.mark.parametrize("lengths", [[3] + [0] * 40 + [5] + [0] * 70 + [130] + [0] * 33 + [1], [0] * 100 + [1] * 3 + [0] * 200 + [2],
                                     [1, 0] * 40 + [0] * 31 + [1] + [0] * 32 + [64] + [0] * 33 + [7], [0] * 700 + [900] + [0] * 50])
def test_rows_behind_gaps_of_empty_sequences(be, lengths, dtype, kv, dim):
    b = Bank(be, lengths, kv, dim, dtype=dtype)
    k, v, _ = read_all(b)
    assert np.array_equal(k, np.concatenate(b.keys)) and np.array_equal(v, np.concatenate(b.values))
    got = b.cache.bounds().cpu().numpy()
    for s in range(b.n):
        for p, (lo, hi) in zip(b.pages[s], ref.bounds(b.keys[s])):
            assert np.array_equal(got[p, :, 0], lo) and np.array_equal(got[p, :, 1], hi), s
    # each of the sequences' last rows again, behind the same gaps
    counts = [min(n, 2) for n in lengths]
    k, v, _ = read_all(b, counts=counts)
    assert np.array_equal(k, np.concatenate([x[len(x) - c:] for x, c in zip(b.keys, counts)]))
    assert np.array_equal(v, np.concatenate([x[len(x) - c:] for x, c in zip(b.values, counts)]))


def test_a_cut_sequence_is_selected_by_the_bounds_of_its_last_write(be):
    """Cut back and not written to: the last page's bounds still hold the rows that
    are gone; a row written to it takes them out."""
    b = Bank(be, [64 * 4 + 40], 1, 32)
    a = Asked(b, [6])
    held = b.keys[0]
    lengths = cuda(np.array([64 * 4 + 3], np.uint32))
    b.table = kc.page_table(b.d["pages"].data_ptr(), lengths.data_ptr(), 1, b.pitch)

    def check(bounds):
        got = select(b, a, 2, 0).cpu().numpy().astype(np.uint32)
        for i in range(6):
            assert got[i, 0].tolist() == ref.chosen(ref.block_scores(a.q[i], bounds)[0], 2, 0)

    check(ref.bounds(held))
    x = torch.randn(2, 1, 1, 32, device="cuda")
    off = cuda(np.array([0, 1]))
    torch.cuda.synchronize()
    be.cache_write(b.cache, b.table, kc.cache_rows(x[0].data_ptr(), x[1].data_ptr(), "f32", 1, off.data_ptr()))
    be.synchronize()
    check(ref.bounds(np.concatenate([held[:64 * 4 + 2], ref.quantised(x[0].cpu().numpy(), "i8")])))
