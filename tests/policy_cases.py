"""Plain 64-bit forms of the policy operators, row by row, for the tests."""
import numpy as np

F32_MAX = float(np.finfo(np.float32).max)


def support(v, kind="scores", f16=False):
    """Open entries of one row of float64 values."""
    with np.errstate(invalid="ignore"):
        return np.flatnonzero(v > 0 if kind == "p" else v > (-65504.0 if f16 else -1e29))


def policy(v, t=1.0, k=0, p=1.0, mp=0.0, kind="scores", f16=False):
    """(kept entries in bank order, their pi, their log pi) of one row."""
    v = np.asarray(v, np.float64)
    j = support(v, kind, f16)
    none = np.zeros(0)
    if not j.size:
        return j, none, none
    u = np.minimum(v[j], F32_MAX)
    if not t > 0:
        top = j[u == u.max()][:1]
        return top, np.ones(1), np.zeros(1)
    x = (np.log(u) - np.log(u.max())) / t if kind == "p" else (u - u.max()) / t
    w = u.copy() if kind == "p" and t == 1 else np.exp(x)
    order = np.lexsort((j, -u))
    if 0 < k:
        order = order[:k]
    if p < 1:
        ws = w[order]
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        order = order[:max(1, int((before < max(p, 0.0) * ws.sum()).sum()))]
    at = np.sort(order)
    at = at[x[at] >= -700.0]
    if mp > 0:
        at = at[w[at] >= min(mp, 1.0) * w.max()]
    z = w[at].sum()
    return j[at], w[at] / z, (np.log(w[at] / z) if kind == "p" and t == 1 else x[at] - np.log(z))


def draw(row, u):
    """The entry a uniform hits (None: the first largest), or -1; its log pi."""
    j, pi, logpi = row
    if not j.size:
        return -1, -np.inf
    if u is None:
        i = int(np.argmax(pi))
    else:
        i = min(int(np.searchsorted(np.cumsum(pi), min(max(u, 0.0), 1.0), side="right")), j.size - 1)
    return int(j[i]), float(logpi[i])


def loss(row, n, action, advantage, beta, t, weight=1.0):
    """(loss, logp, entropy, gradient over the row's n entries)."""
    j, pi, logpi = row
    h = -float((pi * logpi).sum()) if j.size else 0.0
    g = np.zeros(n)
    at = np.flatnonzero(j == action)
    if action < 0:
        return 0.0, 0.0, h, g
    if not at.size or not t > 0:
        return 0.0, (float(logpi[at[0]]) if at.size else -np.inf), h, g
    logp = float(logpi[at[0]])
    d = advantage * pi + beta * pi * (logpi + h)
    d[at[0]] -= advantage
    g[j] = weight * d / t
    return -advantage * logp - beta * h, logp, h, g
