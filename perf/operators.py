"""What the policy operators are measured on: drawing an answer from a tempered
and cut distribution (``draw``), the loss of drawn answers with its gradient
(``loss``), and the global gradient norm with clipping (``clip``).

Rows are laid out as the framework lays out its distributions: a packed batch
of frames, frame f's [Q_f, R_f] block at p_off[f] and its first question at
q_off[f]; or a dense [rows, row_len] matrix with a pitch. ``run`` computes the
plain form with elementary torch operations, or (``own``) calls the backend.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
BLOCKED = -1e29      # a score at or below it is masked out
DROPPED = -700.0     # a tempered log weight below it cannot be drawn
LIMITS = ("temperature", "top_k", "top_p", "min_p")


# --- the cases ---------------------------------------------------------------

def _cut(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    return {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}


def listed():
    return [
        # one interactive turn: a 64-record frame with 8 questions, drawn from its distribution
        {"name": "draw one frame", "op": "draw", "dtype": "f32", "kind": "p", "frames": 1, "q_lo": 8, "q_hi": 8,
         "r_lo": 56, "r_hi": 56, "rule": False, "rows_apart": False, "want_p": True, **_cut(0.8, 0, 0.9, 0.0)},
        # a packed batch under a schema x band grammar, as forward_batch returns it (ragged_4096's geometry)
        {"name": "draw ragged batch", "op": "draw", "dtype": "f32", "kind": "p", "frames": 4096, "q_lo": 1,
         "q_hi": 16, "r_lo": 8, "r_hi": 240, "rule": True, "rows_apart": False, "want_p": True,
         **_cut(0.7, 0, 0.92, 0.0)},
        # long banks: 64 questions over 4096 records a frame, every cut in force
        {"name": "draw long banks", "op": "draw", "dtype": "f32", "kind": "scores", "frames": 64, "q_lo": 64,
         "q_hi": 64, "r_lo": 4096, "r_hi": 4096, "rule": False, "rows_apart": False, "want_p": True,
         **_cut(1.3, 200, 0.95, 0.002)},
        # few rows of a vocabulary's length, each with its own limits; only the drawn entry is asked for
        {"name": "draw wide rows bf16", "op": "draw", "dtype": "bf16", "kind": "scores", "frames": 0, "rows": 32,
         "row_len": 131071, "pitch": 131072, "rows_apart": True, "want_p": False, **_cut(0.9, 50, 0.95, 0.01)},
        # one remembered turn: 4 questions over 60 records
        {"name": "loss one frame", "op": "loss", "dtype": "f32", "kind": "scores", "frames": 1, "q_lo": 4, "q_hi": 4,
         "r_lo": 60, "r_hi": 60, "rule": False, "rows_apart": False, "entropy": 0.01, **_cut(0.8, 0, 0.9, 0.0)},
        # the learn step's batch: 1024 frames of 4 questions, learned under the policy that drew
        {"name": "loss learn batch", "op": "loss", "dtype": "f32", "kind": "scores", "frames": 1024, "q_lo": 4,
         "q_hi": 4, "r_lo": 12, "r_hi": 252, "rule": True, "rows_apart": False, "entropy": 0.01,
         **_cut(0.7, 0, 0.92, 0.0)},
        # the whole softmax over long rows of 16-bit scores, no cut
        {"name": "loss long rows bf16", "op": "loss", "dtype": "bf16", "kind": "scores", "frames": 0, "rows": 4096,
         "row_len": 32001, "pitch": 32008, "rows_apart": False, "entropy": 0.003, **_cut(1.2)},
        # a learn step's f64 sums: both selector matrices, the pool and the token and field rows
        {"name": "clip learn sums", "op": "clip", "set": "sums", "dtype": "f64", "max_norm": 0.5},
        # a gradient for every matrix of the default brain
        {"name": "clip brain", "op": "clip", "set": "brain", "dtype": "f32", "max_norm": 1.0},
        # many tensors of many sizes and of three types
        {"name": "clip many tensors", "op": "clip", "set": "many", "dtype": "mixed", "tensors": 301,
         "elements": 200000000, "max_norm": 2.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["draw", "draw", "loss", "loss", "clip"])
    if op == "clip":
        kind = rng.choice(["f32", "bf16", "f16", "f64", "mixed"])
        return {"op": "clip", "set": "many", "dtype": kind, "tensors": _log_int(rng, 1, 400),
                "elements": _log_int(rng, 5000, 60000000), "max_norm": round(math.exp(rng.uniform(-2, 8)), 3)}
    case = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "kind": "scores",
            "rows_apart": rng.random() < 0.4}
    if rng.random() < 0.6:  # a packed batch of frames
        r_hi = _log_int(rng, 1, 4096)
        r_lo = max(0, _log_int(rng, 1, r_hi) - (1 if rng.random() < 0.2 else 0))
        q_hi = _log_int(rng, 1, 64)
        most = max(1, 3000000 // (r_hi * q_hi))
        case.update(frames=_log_int(rng, 1, min(4096, most)), q_lo=rng.randint(0, q_hi), q_hi=q_hi, r_lo=r_lo,
                    r_hi=r_hi, rule=rng.random() < 0.5)
        if op == "draw" and rng.random() < 0.5:
            case.update(kind="p", dtype="f32")
    else:  # a dense matrix
        row_len = _log_int(rng, 1, 200000)
        case.update(frames=0, rows=_log_int(rng, 1, max(1, min(2000, 6000000 // row_len))), row_len=row_len,
                    pitch=row_len + rng.choice([0, 0, 1, 5, 64]))
    cut = _cut(round(rng.uniform(0.3, 2.0), 3))
    if rng.random() < 0.5:
        cut["top_k"] = _log_int(rng, 1, 500)
    if rng.random() < 0.6:
        cut["top_p"] = round(rng.uniform(0.05, 0.999), 4)
    if rng.random() < 0.4:
        cut["min_p"] = round(math.exp(rng.uniform(-8, -1)), 5)
    case.update(cut)
    if op == "draw":
        case["want_p"] = rng.random() < 0.7
    else:
        case["entropy"] = rng.choice([0.0, 0.01, 0.1])
    return case


# --- geometry ----------------------------------------------------------------

def _geometry(case):
    """Rows of a case: (rows, q_off, p_off, longest row) with the offsets of a
    packed batch, or (rows, None, None, row_len) of a dense matrix."""
    if not case["frames"]:
        return case["rows"], None, None, case["row_len"]
    g = np.random.RandomState((case["frames"] * 7919 + case["q_hi"] * 131 + case["r_hi"]) % (1 << 31))
    q = g.randint(case["q_lo"], case["q_hi"] + 1, case["frames"]).astype(np.int64)
    r = g.randint(case["r_lo"], case["r_hi"] + 1, case["frames"]).astype(np.int64)
    q[-1], r[-1] = case["q_hi"], case["r_hi"]
    off = lambda n: np.concatenate([[0], np.cumsum(n)]).astype(np.int64)  # noqa: E731
    return int(q.sum()), off(q), off(q * r), int(r.max())


def _brain_sizes():
    h, f = 128, 384
    block = [h * h] * 3 + [f * h] * 2
    return [8728 * h] + block * 4 + [2 * h, h * h, h * h, 4 * 3 * h, 3 * h]


def _tensors(case):
    """(elements, type, weight in the norm) of each tensor of a clip case."""
    if case["set"] == "sums":
        h = 128
        return [(h * h, "f64", 1.0), (h * h, "f64", 1.0), (2 * h, "f64", 1.0), (8704 * h, "f64", 0.1)]
    if case["set"] == "brain":
        return [(n, "f32", 1.0) for n in _brain_sizes()]
    g = np.random.RandomState((case["tensors"] * 7919 + case["elements"]) % (1 << 31))
    share = np.exp(g.uniform(-4, 4, case["tensors"]))
    sizes = np.maximum(1, (share / share.sum() * case["elements"]).astype(np.int64))
    kinds = ["f32", "bf16", "f16"]
    return [(int(n), kinds[i % 3] if case["dtype"] == "mixed" else case["dtype"], 1.0) for i, n in enumerate(sizes)]


def work(case):
    if case["op"] == "clip":
        size = {"f32": 4, "bf16": 2, "f16": 2, "f64": 8}
        t = _tensors(case)
        return {"bytes": sum(2 * n * size[d] for n, d, _ in t), "flops": sum(3 * n for n, _, _ in t)}
    rows, _, p_off, row_len = _geometry(case)
    n = int(p_off[-1]) if p_off is not None else rows * row_len
    size = 4 if case["dtype"] == "f32" else 2
    limits = 16 if case["rows_apart"] else 0
    if case["op"] == "draw":
        return {"bytes": n * size + (n * 4 if case["want_p"] else 0) + rows * (8 + limits + 12), "flops": 12 * n}
    return {"bytes": 2 * n * size + rows * (8 + limits + 12), "flops": 16 * n}


# --- inputs ------------------------------------------------------------------

def _flat_outputs(grads):
    """One flat buffer a type for the clipped gradients, as an optimizer or an
    all-reduce keeps them: the buffers, and each tensor's place (16-byte steps)."""
    step = {t: -(-16 // t.itemsize) for t in DTYPES.values()}
    size, at = {}, []
    for g in grads:
        at.append(size.get(g.dtype, 0))
        size[g.dtype] = at[-1] + -(-g.numel() // step[g.dtype]) * step[g.dtype]
    flats = {t: torch.zeros(n, dtype=t, device="cuda") for t, n in size.items()}
    return list(flats.values()), [flats[g.dtype][a:a + g.numel()] for g, a in zip(grads, at)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "clip":
        grads = [(torch.randn(n, device=dev, generator=g, dtype=torch.float32) * (0.02 * (1 + i % 5))).to(DTYPES[d])
                 for i, (n, d, _) in enumerate(_tensors(case))]
        flats, outs = _flat_outputs(grads)
        return {"case": case, "grads": grads, "outs": outs, "flats": flats,
                "weights": [w for _, _, w in _tensors(case)],
                "result": torch.zeros(2, dtype=torch.float64, device=dev)}
    rows, q_off, p_off, row_len = _geometry(case)
    ragged = q_off is not None
    pitch = row_len if ragged else case["pitch"]
    n = int(p_off[-1]) if ragged else rows * pitch
    v = torch.randn(n, device=dev, generator=g, dtype=torch.float32) * 2.5
    if ragged and case["rule"]:  # a grammar admits about a quarter of the bank; a few rows are left with nothing
        v = torch.where(torch.rand(n, device=dev, generator=g) < 0.75, torch.full_like(v, -1e30), v)
    elif n > 100:
        v[torch.randint(0, n, (max(1, n // 50),), device=dev, generator=g)] = -math.inf
    s = {"case": case, "rows": rows, "max_row": row_len, "pitch": pitch}
    if ragged:
        s["q_off"], s["p_off"] = torch.from_numpy(q_off).to(dev), torch.from_numpy(p_off).to(dev)
    if case["kind"] == "p":  # the distribution that a selection leaves, blocked rows all zero
        idx, ok = _positions(s)
        x = torch.where(ok, v[idx].double(), torch.full_like(idx, -1, dtype=torch.float64) * 1e30)
        m = x.amax(1, keepdim=True) if row_len else x.sum(1, keepdim=True)
        e = torch.exp(x - m) * (x > BLOCKED)
        p = (e / e.sum(1, keepdim=True).clamp_min(1e-20)).float()
        v = torch.zeros(n, device=dev)
        v[idx[ok]] = p[ok]
    s["values"] = v.to(DTYPES[case["dtype"]])
    if case["rows_apart"]:  # each row has its own limits
        r = torch.rand(4, rows, device=dev, generator=g)
        s["temperature"] = (case["temperature"] * (0.5 + r[0])).float()
        s["top_k"] = (case["top_k"] * (0.5 + r[1])).to(torch.int32)
        s["top_p"] = (case["top_p"] * (0.8 + 0.25 * r[2])).clamp_max(1.0).float() if case["top_p"] < 1 else r[2] * 0 + 1
        s["min_p"] = (case["min_p"] * (0.5 + r[3])).float()
    new = lambda t, m=rows: torch.zeros(m, dtype=t, device=dev)  # noqa: E731
    s["logp"] = new(torch.float32)
    if case["op"] == "draw":
        s["uniforms"] = torch.rand(rows, device=dev, generator=g, dtype=torch.float64)
        s["index"], s["kept"] = new(torch.int32), new(torch.int32)
        s["p"] = new(torch.float32, n if ragged else rows * row_len) if case["want_p"] else None
    else:
        length = _lengths(s)
        big = torch.randint(0, 1 << 30, (rows,), device=dev, generator=g)
        top = torch.where(length > 0, big % length.clamp_min(1), torch.zeros_like(big))
        idx, ok = _positions(s)
        if row_len:  # most rows learn from a likely answer, some from any, some have none
            best = torch.where(ok, s["values"][idx].float().nan_to_num(neginf=-3e38), -3.1e38).argmax(1)
            top = torch.where(torch.rand(rows, device=dev, generator=g) < 0.6, best, top)
        none = torch.rand(rows, device=dev, generator=g) < 0.05
        s["actions"] = torch.where(none, torch.full_like(top, -1), top).to(torch.int32)
        s["advantage"] = torch.randn(rows, device=dev, generator=g)
        # the mean over the rows; unscaled gradients of f16 scores would fall below the type's range
        s["row_weight"] = torch.rand(rows, device=dev, generator=g) / (1 if case["dtype"] == "f16" else rows)
        s["loss"], s["entropy"] = new(torch.float32), new(torch.float32)
        s["grad"] = torch.zeros(n if ragged else rows * row_len, dtype=s["values"].dtype, device=dev)
    return s


# --- the plain form ----------------------------------------------------------

def _lengths(s):
    """Entries of each row."""
    if "q_off" not in s:
        return torch.full((s["rows"],), s["max_row"], dtype=torch.int64, device="cuda")
    q = s["q_off"][1:] - s["q_off"][:-1]
    r = (s["p_off"][1:] - s["p_off"][:-1]) // q.clamp_min(1)
    row = torch.arange(s["rows"], device="cuda")
    return r[torch.searchsorted(s["q_off"], row, right=True) - 1]


def _positions(s):
    """Each row's entries in the value buffer, padded to the longest row, and which of them exist."""
    col = torch.arange(s["max_row"], device="cuda")
    row = torch.arange(s["rows"], device="cuda")
    length = _lengths(s)
    if "q_off" in s:
        frame = torch.searchsorted(s["q_off"], row, right=True) - 1
        start = s["p_off"][frame] + (row - s["q_off"][frame]) * length
    else:
        start = row * s["pitch"]
    ok = col[None, :] < length[:, None]
    return torch.where(ok, start[:, None] + col[None, :], 0), ok


def _limit(s, name):
    v = s.get(name)
    if v is None:
        return torch.full((s["rows"], 1), s["case"][name], dtype=torch.float32, device="cuda").double()
    return v.double()[:, None]


def _policy(s, v, ok):
    """The tempered and cut policy of padded rows, in 64 bits: log weights
    against the row's largest, weights, and which entries are kept."""
    case, f16 = s["case"], s["values"].dtype == torch.float16
    v = v.double()
    open_ = ok & ((v > 0) if case["kind"] == "p" else (v > (-65504.0 if f16 else BLOCKED)))
    if case["kind"] == "scores":
        v = v.clamp(max=torch.finfo(torch.float32).max)
    t = _limit(s, "temperature")
    low = torch.full_like(v, -math.inf)
    m = torch.where(open_, v, low).amax(1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.ones_like(m))
    x = (torch.log(v) - torch.log(m)) / t if case["kind"] == "p" else (v - m) / t
    x = torch.where(open_, x, low)
    kept = x >= DROPPED
    w = torch.where(kept, torch.exp(x), torch.zeros_like(x))
    if case["top_k"] or case["top_p"] < 1:
        order = torch.argsort(torch.where(open_, v, low), dim=1, descending=True, stable=True)
        k = _limit(s, "top_k")
        rank = torch.arange(v.shape[1], device=v.device)[None, :]
        ws = w.gather(1, order)
        ws = torch.where((rank < k) | (k <= 0), ws, torch.zeros_like(ws))
        before = ws.cumsum(1)
        before = torch.cat([torch.zeros_like(before[:, :1]), before[:, :-1]], 1)
        total = ws.sum(1, keepdim=True)
        p = _limit(s, "top_p")
        cut = ((rank < k) | (k <= 0)) & ((before < p * total) | (p >= 1) | (rank == 0))
        kept = kept & torch.zeros_like(kept).scatter(1, order, cut)
    if case["min_p"] > 0:
        floor = _limit(s, "min_p")
        same = (case["kind"] == "p") & (t == 1)
        kept = kept & torch.where(same, v >= floor * m, w >= floor)
    return t, x, torch.where(kept, w, torch.zeros_like(w)), kept


def _plain_draw(s):
    idx, ok = _positions(s)
    if s["max_row"] == 0:
        none = torch.full((s["rows"],), -1, dtype=torch.int32, device="cuda")
        return none, none * 0, torch.full((s["rows"],), -math.inf, device="cuda"), s["p"]
    _, _, w, kept = _policy(s, s["values"][idx], ok)
    cum = w.cumsum(1)
    z = cum[:, -1:]
    past = (cum > s["uniforms"][:, None] * z) & kept
    col = torch.arange(w.shape[1], device="cuda")[None, :]
    last = torch.where(kept, col, -1).amax(1)
    j = torch.where(past.any(1), past.to(torch.uint8).argmax(1), last)
    pi = w / torch.where(z > 0, z, torch.ones_like(z))
    logp = torch.where(j >= 0, torch.log(pi.gather(1, j.clamp_min(0)[:, None])[:, 0]), -math.inf)
    p = None
    if s["p"] is not None:
        if "q_off" in s:
            p = torch.zeros_like(s["p"])
            p[idx[ok]] = pi[ok].float()
        else:
            p = pi.float().reshape(-1)
    return j.to(torch.int32), kept.sum(1).to(torch.int32), logp.float(), p


def _plain_loss(s):
    case = s["case"]
    idx, ok = _positions(s)
    v = s["values"][idx]
    a = s["actions"].long()[:, None]
    adv, g, beta = s["advantage"][:, None], s["row_weight"][:, None], case["entropy"]
    whole = case["top_k"] == 0 and case["top_p"] >= 1 and case["min_p"] <= 0
    if whole:  # nothing is cut: 32 bits hold it
        open_ = ok & (v.float() > (-65504.0 if v.dtype == torch.float16 else BLOCKED))
        low = torch.full((1, 1), -math.inf, device="cuda")
        x = torch.where(open_, v.float(), low)
        m = x.amax(1, keepdim=True)
        t = _limit(s, "temperature").float()
        x = (x - torch.where(torch.isfinite(m), m, torch.zeros_like(m))) / t
        kept = x >= DROPPED
        w = torch.where(kept, torch.exp(x), torch.zeros_like(x))
    else:
        t, x, w, kept = _policy(s, v, ok)
    z = w.sum(1, keepdim=True)
    z = torch.where(z > 0, z, torch.ones_like(z))
    pi = w / z
    logpi = torch.where(kept, x, torch.zeros_like(x)) - torch.log(z)
    h = -(pi * logpi).sum(1, keepdim=True)
    safe = a.clamp(0, max(0, v.shape[1] - 1))
    live = (a >= 0) & (a < v.shape[1]) & kept.gather(1, safe)
    logp = torch.where(live, logpi.gather(1, safe), torch.full_like(h, -math.inf))
    loss = torch.where(live, -adv * logp - beta * h, torch.zeros_like(h))
    one = torch.arange(v.shape[1], device="cuda")[None, :] == a
    d = g * (adv * (pi - one.to(pi.dtype)) + beta * pi * (logpi + h)) / t
    d = torch.where(live & kept, d, torch.zeros_like(d))
    logp = torch.where(a < 0, torch.zeros_like(logp), logp)
    h = torch.where(kept.any(1, keepdim=True), h, torch.zeros_like(h))
    if "q_off" in s:
        grad = torch.zeros_like(s["grad"])
        grad[idx[ok]] = d[ok].to(grad.dtype)
    else:
        grad = d.to(s["grad"].dtype).reshape(-1)
    return loss[:, 0].float(), logp[:, 0].float(), h[:, 0].float(), grad


def _plain_clip(s):
    total = sum((w * w) * t.double().square().sum() for t, w in zip(s["grads"], s["weights"]))
    norm = torch.sqrt(total)
    c = s["case"]["max_norm"]
    scale = torch.where(torch.isfinite(norm) & (norm > c), c / norm, torch.ones_like(norm))
    wide = {torch.float64: torch.float64}
    [o.copy_(t.to(wide.get(t.dtype, torch.float32)) * scale.to(wide.get(t.dtype, torch.float32)))
     for o, t in zip(s["outs"], s["grads"])]
    return torch.stack([norm, scale]), s["flats"]


# --- the framework's calls ---------------------------------------------------

_backend = None


def _handle():
    """The handle that a user's program keeps."""
    global _backend
    if _backend is None:
        from krystal_b200 import BRAIN_FORWARD_CONFIG, create_brain_forward_weights, cuda_backend
        cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
        _backend = cuda_backend(0)(cfg, create_brain_forward_weights(cfg, 1337))
    return _backend


def _own(s):
    from krystal_b200 import policy
    be, case = _handle(), s["case"]
    ptr = lambda name: s[name].data_ptr() if s.get(name) is not None else None  # noqa: E731
    if case["op"] == "clip":
        if "list" not in s:  # a program's gradients stay where they are: it lists them once
            s["list"] = policy.GradList(s["grads"], s["outs"], s["weights"])
        be.clip_grads(s["list"], case["max_norm"], ptr("result"))
        return s["result"], s["flats"]
    if "q_off" in s:
        rows = policy.ragged_rows(ptr("values"), case["dtype"], s["rows"], case["frames"], ptr("q_off"),
                                  ptr("p_off"), s["max_row"], case["kind"])
    else:
        rows = policy.dense_rows(ptr("values"), case["dtype"], s["rows"], s["max_row"], s["pitch"], case["kind"])
    sampling = policy.Sampling(case["temperature"], case["top_k"], case["top_p"], case["min_p"],
                               ptr("temperature"), ptr("top_k"), ptr("top_p"), ptr("min_p"))
    if case["op"] == "draw":
        be.draw(rows, sampling, ptr("uniforms"), index=ptr("index"), kept=ptr("kept"), logp=ptr("logp"), p=ptr("p"))
        return s["index"], s["kept"], s["logp"], s["p"]
    be.policy_loss(rows, sampling, ptr("actions"), ptr("advantage"), case["entropy"], ptr("row_weight"),
                   loss=ptr("loss"), logp=ptr("logp"), entropy=ptr("entropy"), grad=ptr("grad"))
    return s["loss"], s["logp"], s["entropy"], s["grad"]


def run(state):
    if own:
        return _own(state)
    return {"draw": _plain_draw, "loss": _plain_loss, "clip": _plain_clip}[state["case"]["op"]](state)


# --- from the definitions, row by row in 64 bits -----------------------------

def _row_policy(case, v, t, k, p, mp):
    """(kept entries in bank order, their probabilities, their log probabilities) of one row."""
    if case["kind"] == "p":
        j = np.flatnonzero(v > 0)
        if not j.size:
            return j, v[:0], v[:0]
        x = (np.log(v[j]) - np.log(v[j].max())) / t
    else:
        j = np.flatnonzero(v > (-65504.0 if case["dtype"] == "f16" else BLOCKED))
        if not j.size:
            return j, v[:0], v[:0]
        u = np.minimum(v[j], float(np.finfo(np.float32).max))
        x = (u - u.max()) / t
    if (0 < k < j.size) or p < 1:
        by = np.lexsort((j, -v[j]))
        if 0 < k:
            by = by[:k]
        if p < 1:
            w = np.exp(x[by])
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            by = by[:max(1, int((before < p * w.sum()).sum()))]
        by = np.sort(by)
        j, x = j[by], x[by]
    if mp > 0:
        fine = v[j] >= mp * v[j].max() if case["kind"] == "p" and t == 1 else np.exp(x) >= mp
        j, x = j[fine], x[fine]
    j, x = j[x >= DROPPED], x[x >= DROPPED]
    w = np.exp(x)
    z = w.sum()
    return j, w / z, x - np.log(z)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        parts = [float(torch.dot(t.double(), t.double())) * w * w for t, w in zip(s["grads"], s["weights"])]
        norm = math.sqrt(math.fsum(parts))
        scale = case["max_norm"] / norm if norm > case["max_norm"] else 1.0
        flats = [t.double() for t in s["flats"]]  # zeros: the places between the tensors stay so
        for o, t in zip(s["outs"], s["grads"]):
            k = [f.dtype for f in s["flats"]].index(t.dtype)
            flats[k][o.storage_offset():o.storage_offset() + t.numel()] = t.double() * scale
        return torch.tensor([norm, scale], dtype=torch.float64), flats
    rows, q_off, p_off, row_len = _geometry(case)
    host = lambda name: s[name].double().cpu().numpy()  # noqa: E731
    values = host("values")
    limits = [host(n) if n in s else np.full(rows, float(np.float32(case[n]))) for n in LIMITS]
    if q_off is not None:
        frame = np.repeat(np.arange(case["frames"]), np.diff(q_off))
        length = (np.diff(p_off) // np.maximum(1, np.diff(q_off)))[frame]
        start = p_off[frame] + (np.arange(rows) - q_off[frame]) * length
        out_start, total = start, int(p_off[-1])
    else:
        length = np.full(rows, row_len)
        start, out_start, total = np.arange(rows) * case["pitch"], np.arange(rows) * row_len, rows * row_len
    out = np.zeros(total)
    logp, second, third = np.full(rows, -np.inf), np.zeros(rows), np.zeros(rows)
    index = np.full(rows, -1, np.int64)
    extra = {n: host(n) for n in ("uniforms", "actions", "advantage", "row_weight") if n in s}
    for i in range(rows):
        t, k, p, mp = limits[0][i], int(limits[1][i]), limits[2][i], limits[3][i]
        j, pi, logpi = _row_policy(case, values[start[i]:start[i] + length[i]], t, k, p, mp)
        if case["op"] == "draw":
            second[i] = j.size
            if j.size:
                at = min(int(np.searchsorted(np.cumsum(pi), extra["uniforms"][i], side="right")), j.size - 1)
                index[i], logp[i] = j[at], logpi[at]
                out[out_start[i] + j] = pi
            continue
        h = -float((pi * logpi).sum())
        third[i] = h
        a = int(extra["actions"][i])
        at = np.flatnonzero(j == a)
        if a < 0:
            logp[i] = 0.0
        if not at.size:
            continue
        logp[i] = logpi[at[0]]
        second[i] = -extra["advantage"][i] * logp[i] - case["entropy"] * h
        d = extra["advantage"][i] * pi + case["entropy"] * pi * (logpi + h)
        d[at[0]] -= extra["advantage"][i]
        out[out_start[i] + j] = extra["row_weight"][i] * d / t
    if case["op"] == "draw":
        # indices and counts are whole numbers: they have to be equal to the plain form's
        return None, None, torch.from_numpy(logp), torch.from_numpy(out) if case["want_p"] else None
    return torch.from_numpy(second), torch.from_numpy(logp), torch.from_numpy(third), torch.from_numpy(out)
