"""Plain 64-bit forms of the bank cache's operators, for the tests."""
import numpy as np

PAGE, CELL = 64, 32
TOP = {"i8": 127.0, "e4m3": 448.0}
LEAST, MOST = 2.0 ** -100, 2.0 ** 127
NONE = 0xFFFFFFFF


def meaning(fmt):
    """The value of each of the 256 codes."""
    c = np.arange(256)
    if fmt == "i8":
        return c - 128.0
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m / 8 * 2.0 ** -6)
    return np.where(c & 128, -v, v)


def quantised(x, fmt):
    """The stored values of rows x [..., dim], f32: the scale and the quotient
    rounded to f32, then the nearest code, halves to the even."""
    x = np.asarray(x, np.float64)
    x = np.clip(np.where(np.isnan(x), 0.0, x), -MOST, MOST)
    scale = np.maximum((np.abs(x).max(-1, keepdims=True) / TOP[fmt]).astype(np.float32).astype(np.float64), LEAST)
    y = (x / scale).astype(np.float32).astype(np.float64)
    if fmt == "i8":
        code = np.rint(y)
    else:
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
        code = np.clip(np.rint(y / step) * step, -448.0, 448.0)
    return (code * scale).astype(np.float32)


def bounds(keys):
    """[pages, 2, kv, dim] smallest and largest of each page of keys [n, kv, dim]."""
    return [np.stack([keys[i:i + PAGE].min(0), keys[i:i + PAGE].max(0)]) for i in range(0, len(keys), PAGE)]


def masked(x, m):
    """Scores x [..., n] under a mask row m [n], and which are open."""
    with np.errstate(invalid="ignore"):
        ok = m > -1e29
    return x + np.where(ok, np.minimum(np.where(ok, m, 0.0), 1e29), 0.0), ok


def attend(q, keys, values, scale, mask=None, rows=None):
    """(out [heads, dim], lse [heads]) of one question q [heads, dim] over cached
    rows [n, kv, dim]; rows: the rows it sees, with repeats."""
    heads, dim = q.shape
    g = heads // keys.shape[1]
    out, lse = np.zeros((heads, dim)), np.full(heads, -np.inf)
    for h in range(heads):
        at = np.arange(len(keys)) if rows is None else np.asarray(rows[h // g], np.int64)
        k, v = keys[at, h // g].astype(np.float64), values[at, h // g].astype(np.float64)
        s, ok = masked(k @ q[h].astype(np.float64) * scale, np.zeros(len(at)) if mask is None else mask[at])
        s, v = s[ok], v[ok]
        if s.size:
            m = s.max()
            e = np.exp(s - m)
            out[h], lse[h] = e @ v / e.sum(), m + np.log(e.sum())
    return out, lse


def block_scores(q, lo_hi):
    """[kv, blocks] of one question q [heads, dim] over bounds [blocks, 2, kv, dim]."""
    kv = lo_hi[0].shape[1]
    g = q.shape[0] // kv
    q = q.astype(np.float64).reshape(kv, g, -1)
    out = np.zeros((kv, len(lo_hi)))
    for b, (lo, hi) in enumerate(lo_hi):
        for h in range(kv):
            out[h, b] = np.maximum(q[h] * lo[h].astype(np.float64), q[h] * hi[h].astype(np.float64)).sum()
    return out


def chosen(scores, count, recent):
    """The blocks taken of one row of scores: ascending, NONE behind the last."""
    n = len(scores)
    s = np.where(np.arange(n) + recent >= n, np.inf, scores)
    took = sorted(np.lexsort((np.arange(n), -s))[:count].tolist())
    return took + [NONE] * (count - len(took))
