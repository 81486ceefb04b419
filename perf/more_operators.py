"""What the bank cache's operators are measured on: quantising rows as they are
written and reading them back (``write``), attention of questions over cached
rows (``attend``), the same over the blocks that a bound of their scores selects
(``sparse``), and the pointer scores of a bank (``scores``).

A cache is one buffer of pages of 64 rows. A page holds, head after head, two
cells of 32 rows: their 8-bit keys, their 8-bit values, an f32 scale a key and
an f32 scale a value. Behind the pages lie each page's bounds: the smallest and
the largest of its keys, f32, dimension by dimension. A sequence is a list of
pages and a length. ``run`` computes the plain form with elementary torch
operations, or (``own``) calls the backend.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAGE, CELL = 64, 32
TOP = {"i8": 127.0, "e4m3": 448.0}   # the largest code
LEAST = 2.0 ** -100                  # the smallest scale
MOST = 2.0 ** 127                    # what larger values count as
BLOCKED = -1e29                      # a mask entry at or below it, or NaN, shuts a row out


# --- the cases ---------------------------------------------------------------

def _case(name, op, dtype, fmt, heads, kv_heads, dim, seqs, q, r, **more):
    return {"name": name, "op": op, "dtype": dtype, "format": fmt, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "seqs": seqs, "q_lo": q[0], "q_hi": q[1], "r_lo": r[0], "r_hi": r[1], "mask": False, **more}


def listed():
    return [
        # 64 sessions, one new record each: what an interactive turn adds to its bank
        _case("write one record a session", "write", "f32", "i8", 4, 4, 32, 64, (1, 1), (1, 2000)),
        # the banks of a packed batch of frames (ragged_4096's geometry), written whole
        _case("write ragged batch", "write", "f32", "i8", 4, 4, 32, 4096, (8, 240), (0, 0)),
        # long histories in 16 bits, wide heads
        _case("write long bf16 e4m3", "write", "bf16", "e4m3", 8, 8, 128, 8, (30001, 32768), (0, 100)),
        # one turn over a small bank: a 64-record frame with 8 questions
        _case("attend one frame", "attend", "f32", "i8", 4, 4, 32, 1, (8, 8), (56, 56)),
        # a packed batch of frames, the mixer's heads
        _case("attend ragged batch", "attend", "f32", "i8", 4, 4, 32, 4096, (1, 16), (8, 240)),
        # long banks: 64 questions over 4096 records a frame, under a mask
        _case("attend long banks", "attend", "f32", "i8", 4, 4, 32, 64, (64, 64), (4096, 4096), mask=True),
        # single tokens of a ragged serving batch, four heads a key head
        _case("attend single bf16 e4m3", "attend", "bf16", "e4m3", 32, 8, 128, 32, (1, 1), (1, 16384)),
        # one token over one very long history: the work has to be split over its length
        _case("attend one long f16", "attend", "f16", "i8", 16, 4, 64, 1, (1, 1), (400003, 400003)),
        # questions that look at 8 of their bank's blocks, the newest among them
        _case("sparse banks", "sparse", "f32", "i8", 4, 4, 32, 64, (16, 16), (1000, 4096), blocks=8, recent=1),
        # single tokens over long histories, 64 blocks each
        _case("sparse long bf16", "sparse", "bf16", "i8", 32, 8, 128, 8, (4, 4), (100000, 131072), blocks=64, recent=2),
        # the pointer scores of one turn
        _case("scores one frame", "scores", "f32", "i8", 1, 1, 128, 1, (8, 8), (1000, 1000)),
        # the pointer scores of long banks, under a mask
        _case("scores long banks", "scores", "f32", "i8", 1, 1, 128, 64, (64, 64), (4096, 4096), mask=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "sparse", "scores"])
    dim = rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
    dtype, fmt = rng.choice(["f32", "f16", "bf16"]), rng.choice(["i8", "e4m3"])
    if op == "write":
        q_hi = _log_int(rng, 1, 20000)
        seqs = _log_int(rng, 1, max(1, min(2000, 60000000 // (q_hi * kv_heads * dim))))
        return dict(op=op, dtype=dtype, format=fmt, heads=kv_heads, kv_heads=kv_heads, dim=dim, seqs=seqs,
                    q_lo=rng.randint(0, q_hi), q_hi=q_hi, r_lo=0, r_hi=rng.choice([0, 1, 63, 64, 1000]), mask=False)
    if op == "scores":
        heads = kv_heads = 1
    r_hi = _log_int(rng, 1, 100000)
    q_hi = _log_int(rng, 1, 64 if r_hi <= 8192 else 8)
    most = min(200000000 // (r_hi * kv_heads * dim), 100000000 // (r_hi * q_hi * heads))
    seqs = _log_int(rng, 1, max(1, min(1000, most)))
    r_lo = max(0, _log_int(rng, 1, r_hi) - (1 if rng.random() < 0.2 else 0))
    case = dict(op=op, dtype=dtype, format=fmt, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs,
                q_lo=rng.randint(0, q_hi), q_hi=q_hi, r_lo=r_lo, r_hi=r_hi, mask=rng.random() < 0.4)
    if op == "sparse":
        case.update(blocks=_log_int(rng, 1, 100), recent=0)
        case["recent"] = min(case["blocks"], rng.choice([0, 1, 2]))
        most = 300000000 // (case["blocks"] * PAGE * dim * kv_heads * q_hi)
        case["seqs"] = max(1, min(case["seqs"], most))
    return case


# --- geometry ----------------------------------------------------------------

def _geometry(case):
    """Questions (or new rows) and cached rows of each sequence."""
    g = np.random.RandomState((case["seqs"] * 7919 + case["q_hi"] * 131 + case["r_hi"]) % (1 << 31))
    q = g.randint(case["q_lo"], case["q_hi"] + 1, case["seqs"]).astype(np.int64)
    r = g.randint(case["r_lo"], case["r_hi"] + 1, case["seqs"]).astype(np.int64)
    q[-1], r[-1] = case["q_hi"], case["r_hi"]
    return q, (r + q if case["op"] == "write" else r)


def _offsets(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int64)


def work(case):
    q, r = _geometry(case)
    d, h, kv = case["dim"], case["heads"], case["kv_heads"]
    size = 4 if case["dtype"] == "f32" else 2
    row = kv * (2 * d + 8)  # a cached row: 8-bit keys and values, two f32 scales a head
    if case["op"] == "write":  # the rows in, their codes out and in again, the rows out
        n = int(q.sum())
        pages = int((-(-r // PAGE) - (r - q) // PAGE)[q > 0].sum())
        return {"bytes": n * (2 * 2 * kv * d * size + 2 * row) + pages * kv * 2 * d * 4, "flops": n * kv * d * 8}
    nq, pairs = int(q.sum()), int((q * r).sum())
    if case["op"] == "scores":
        return {"bytes": int(r.sum()) * (d + 4) + nq * d * size + pairs * (8 if case["mask"] else 4),
                "flops": 2 * pairs * d}
    io = nq * h * (2 * d * size + 4)
    if case["op"] == "attend":
        return {"bytes": int(r.sum()) * row + io + (4 * pairs if case["mask"] else 0), "flops": 4 * pairs * h * d}
    pages = -(-r // PAGE)
    taken = np.minimum(pages, case["blocks"])  # blocks a question reads, and at most all of a bank's once
    read = int((np.minimum(q * taken * PAGE, r)).sum()) * row
    seen = int((q * np.minimum(taken * PAGE, r)).sum())
    return {"bytes": int(pages.sum()) * kv * 2 * d * 4 + read + io + nq * kv * case["blocks"] * 4
            + (4 * seen if case["mask"] else 0), "flops": 4 * seen * h * d + 4 * int((q * pages).sum()) * h * d}


# --- the storage ---------------------------------------------------------------

def _cell_bytes(d):
    return CELL * 2 * d + CELL * 8


def _places(d, device):
    """Where byte b of row r of a cell's keys and of its values lies: rows are in
    order, and a row's 64-byte halves (keys of 128) and 32-byte quarters (values
    of 64 and 128) change places by the row's number."""
    r = torch.arange(CELL, device=device)[:, None]
    b = torch.arange(d, device=device)[None, :]
    keys = b ^ (((r >> 2) & 1) << 6) if d == 128 else b + 0 * r
    values = b ^ ((r & 3) << 5) if d == 128 else b ^ (((r >> 1) & 1) << 5) if d == 64 else b + 0 * r
    return keys, values


def _quantise(x, fmt):
    """Codes (u8) and scales (f32) of rows x [..., d]: the scale is the row's
    largest magnitude over the largest code, a code the nearest to x / scale."""
    x = x.float().nan_to_num(0.0, MOST, -MOST).clamp(-MOST, MOST)
    top = torch.full((), TOP[fmt], device=x.device)  # by a Python number the quotient would not be the rounded one
    scale = (x.abs().amax(-1) / top).clamp_min(LEAST)
    y = x / scale[..., None]
    if fmt == "i8":
        return (y.round() + 128).to(torch.uint8), scale
    return y.to(torch.float8_e4m3fn).view(torch.uint8), scale


def _decode(codes, fmt):
    return codes.float() - 128 if fmt == "i8" else codes.contiguous().view(torch.float8_e4m3fn).float()


def _split(s):
    """Views of the storage: keys, values [pages, kv, 2, 32, d] u8, their scales
    [pages, kv, 2, 32] f32, and the bounds [pages, kv, 2, d] f32."""
    case = s["case"]
    p, kv, d, cell = s["page_count"], case["kv_heads"], case["dim"], _cell_bytes(case["dim"])
    body = s["storage"][:p * kv * 2 * cell].view(p, kv, 2, cell)
    at = CELL * d
    scales = body.view(torch.float32)
    return (body[..., :at].unflatten(-1, (CELL, d)), body[..., at:2 * at].unflatten(-1, (CELL, d)),
            scales[..., 2 * at // 4:2 * at // 4 + CELL], scales[..., 2 * at // 4 + CELL:],
            s["storage"][p * kv * 2 * cell:].view(torch.float32).view(p, kv, 2, d))


def _fetch(s, pages):
    """Keys and values of whole pages, f32 [..., kv, 64, d]."""
    case, (kc, vc, ks, vs, _) = s["case"], _split(s)
    out = []
    for codes, scales, place in zip((kc, vc), (ks, vs), _places(case["dim"], pages.device)):
        c = codes[pages]
        c = c.gather(-1, place.expand(c.shape)) if case["dim"] > 32 else c
        out.append((_decode(c, case["format"]) * scales[pages][..., None]).flatten(-3, -2))
    return out


# --- inputs ------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    q, r = _geometry(case)
    kv, d, n = case["kv_heads"], case["dim"], case["seqs"]
    pitch = max(1, int(-(-r.max() // PAGE)))
    count = n * pitch + 3
    s = {"case": case, "page_count": count, "max_q": int(q.max()), "max_r": int(r.max()), "pitch": pitch,
         "questions": int(q.sum()), "q_off": torch.from_numpy(_offsets(q)).to(dev),
         "lengths": torch.from_numpy(r.astype(np.int32)).to(dev),
         "storage": torch.zeros(count * kv * (2 * _cell_bytes(d) + 8 * d), dtype=torch.uint8, device=dev)}
    s["pages"] = torch.randperm(count, device=dev, generator=g)[:n * pitch].view(n, pitch).to(torch.int32)
    kc, vc, ks, vs, bounds = _split(s)
    held = s["lengths"] - torch.from_numpy(q.astype(np.int32)).to(dev) if case["op"] == "write" else s["lengths"]
    rows = torch.zeros(count, dtype=torch.int32, device=dev)  # rows that each page holds
    rows[s["pages"].long()] = (held[:, None] - PAGE * torch.arange(pitch, device=dev)).clamp(0, PAGE).to(torch.int32)
    key_place, value_place = _places(d, dev)
    step = max(1, (1 << 27) // (kv * PAGE * d))
    for a in range(0, count, step):  # what earlier turns wrote; a page's records are near one another
        m = min(step, count - a)
        new = lambda *shape: torch.randn(m, kv, *shape, device=dev, generator=g)  # noqa: E731
        for codes, scales, place, drift in ((kc, ks, key_place, 0.7), (vc, vs, value_place, 0.2)):
            x = new(PAGE, d) * (0.4 + new(PAGE, 1).abs()) + drift * new(1, d)
            c, sc = _quantise(x, case["format"])
            if codes is kc:
                y = _decode(c, case["format"]) * sc[..., None]
                ok = (torch.arange(PAGE, device=dev) < rows[a:a + m, None])[:, None, :, None]
                bounds[a:a + m, :, 0] = torch.where(ok, y, math.inf).amin(2)
                bounds[a:a + m, :, 1] = torch.where(ok, y, -math.inf).amax(2)
            c = c.view(m, kv, 2, CELL, d)
            codes[a:a + m] = c.gather(-1, place.expand(c.shape))
            scales[a:a + m] = sc.view(m, kv, 2, CELL)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "write":
        x = torch.randn(2, s["questions"], kv, d, device=dev, generator=g)
        x = x * (0.3 + torch.randn(2, s["questions"], kv, 1, device=dev, generator=g).abs())
        x[:, ::97] = 0.0  # records that encode to nothing
        s["keys"], s["values"] = x[0].to(dt), x[1].to(dt)
        s["keys_out"], s["values_out"] = torch.zeros_like(s["keys"]), torch.zeros_like(s["values"])
        return s
    s["q"] = (torch.randn(s["questions"], case["heads"], d, device=dev, generator=g) * 1.2).to(dt)
    off = _offsets(q * r)
    s["p_off"] = torch.from_numpy(off).to(dev)
    if case["mask"]:  # a grammar admits a quarter of the bank; some questions are left with nothing
        m = torch.rand(int(off[-1]), device=dev, generator=g)
        s["mask"] = torch.where(m < 0.75, torch.full_like(m, -1e30), (m - 0.8) * 4)
        none = torch.from_numpy(np.arange(s["questions"]) % 17 == 5).to(dev)
        none = torch.repeat_interleave(none, torch.from_numpy(np.repeat(r, q)).to(dev))
        s["mask"] = torch.where(none, torch.full_like(m, -1e30), s["mask"])
        s["mask"] = torch.where(m < 0.02, torch.full_like(m, math.nan), s["mask"])
        s["mask"] = torch.where((m > 0.02) & (m < 0.04), torch.full_like(m, -math.inf), s["mask"])
        del none, m
    if case["op"] == "scores":
        s["scores"] = torch.zeros(int(off[-1]), device=dev)
        return s
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(s["questions"], case["heads"], device=dev)
    if case["op"] == "sparse":
        s["blocks"] = torch.zeros(s["questions"], kv, case["blocks"], dtype=torch.int32, device=dev)
    return s


# --- the plain form ----------------------------------------------------------

def _whose(s):
    """Each question's sequence, and its number there."""
    row = torch.arange(s["questions"], device="cuda")
    seq = torch.searchsorted(s["q_off"], row, right=True) - 1
    return seq, row - s["q_off"][seq]


def _padded(s, x):
    """Per-question rows as [seqs, most questions, ...], zeros where there is none."""
    seq, at = _whose(s)
    out = torch.zeros(s["case"]["seqs"], s["max_q"], *x.shape[1:], dtype=x.dtype, device=x.device)
    out[seq, at] = x
    return out


def _entries(s, columns, rows=None):
    """Where columns [..., n] of each question's mask row lie, and which exist."""
    seq, at = _whose(s)
    length = s["lengths"].long()[seq]
    shape = (-1,) + (1,) * (columns.dim() - 1)
    ok = (columns >= 0) & (columns < length.view(shape))
    return torch.where(ok, (s["p_off"][seq] + at * length).view(shape) + columns, 0), ok


def _softmax(score, ok, values):
    """(sum of exp(score) * value over what is open, divided; log sum)."""
    low = torch.full((1,), -math.inf, device=score.device)
    score = torch.where(ok, score, low)
    m = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    z = e.sum(-1, keepdim=True)
    return (e @ values) / torch.where(z > 0, z, torch.ones_like(z)), (m + torch.log(z)).squeeze(-1)


def _mask_of(s, columns):
    """Mask values of every question's columns, and which are open."""
    at, ok = _entries(s, columns)
    if not s["case"]["mask"]:
        return torch.zeros((), device="cuda"), ok
    if s["mask"].numel() == 0:
        return torch.zeros_like(ok, dtype=torch.float32), ok
    m = s["mask"][at]
    return m.clamp_max(-BLOCKED), ok & (m > BLOCKED)


def _plain_attend(s):
    case = s["case"]
    n, kv, d, g, mq = case["seqs"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"], s["max_q"]
    keys, values = (x.transpose(1, 2).flatten(2, 3) for x in _fetch(s, s["pages"].long()))  # [n, kv, rows, d]
    q = _padded(s, s["q"].float()).view(n, mq, kv, g, d).permute(0, 2, 1, 3, 4).reshape(n, kv, mq * g, d)
    score = (q @ keys.transpose(-1, -2)) * (1 / math.sqrt(d))
    col = torch.arange(keys.shape[2], device="cuda")
    m, ok = _mask_of(s, col.expand(s["questions"], -1))
    if m.dim():
        score = score + _padded(s, m)[:, None, :, None, :].expand(-1, 1, -1, g, -1).reshape(n, 1, mq * g, -1)
    ok = _padded(s, ok)[:, None, :, None, :].expand(-1, 1, -1, g, -1).reshape(n, 1, mq * g, -1)
    out, lse = _softmax(score, ok, values)
    seq, at = _whose(s)
    out = out.view(n, kv, mq, g, d).permute(0, 2, 1, 3, 4)[seq, at].reshape(-1, case["heads"], d)
    lse = lse.view(n, kv, mq, g).permute(0, 2, 1, 3)[seq, at].reshape(-1, case["heads"])
    return out.to(s["q"].dtype), lse


def _plain_sparse(s):
    case = s["case"]
    kv, d, g, k = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"], case["blocks"]
    seq, at = _whose(s)
    n = (s["lengths"].long() + PAGE - 1) // PAGE
    bounds = _split(s)[4][s["pages"].long()].double()  # next to one another two scores decide: 64 bits
    bounds = torch.where(torch.isfinite(bounds), bounds, 0.0)
    q = _padded(s, s["q"].double()).view(case["seqs"], s["max_q"], kv, g, d)
    up = torch.einsum("nqhgd,nphd->nqhp", q.clamp_min(0), bounds[:, :, :, 1])
    score = (up + torch.einsum("nqhgd,nphd->nqhp", q.clamp_max(0), bounds[:, :, :, 0]))[seq, at]
    block = torch.arange(s["pitch"], device="cuda")
    n = n[seq][:, None, None]
    score = torch.where(block >= n - case["recent"], math.inf, score)
    score = torch.where(block < n, score, -math.inf)
    order = torch.argsort(score, dim=-1, descending=True, stable=True)[..., :k]
    order = torch.where(order < n, order, 1 << 40).sort(-1).values
    if order.shape[-1] < k:
        order = torch.cat([order, order.new_full((*order.shape[:-1], k - order.shape[-1]), 1 << 40)], -1)
    taken = order < n
    page = s["pages"].long()[seq[:, None, None], torch.where(taken, order, 0)]
    head = torch.arange(kv, device="cuda")[None, :, None]
    kc, vc, ks, vs, _ = _split(s)
    rows = []
    for codes, scales, place in zip((kc, vc), (ks, vs), _places(d, page.device)):
        c = codes[page, head]
        c = c.gather(-1, place.expand(c.shape)) if d > 32 else c
        rows.append((_decode(c, case["format"]) * scales[page, head][..., None]).flatten(2, 4))  # [nq, kv, k * 64, d]
    col = (torch.where(taken, order * PAGE, -PAGE)[..., None] + torch.arange(PAGE, device="cuda")).flatten(2)
    score = (s["q"].float().view(-1, kv, g, d) @ rows[0].transpose(-1, -2)) * (1 / math.sqrt(d))
    m, ok = _mask_of(s, col)
    score = score + (m[:, :, None] if m.dim() else m)
    out, lse = _softmax(score, ok[:, :, None], rows[1])
    blocks = torch.where(taken, order, -1).to(torch.int32)
    return blocks, out.reshape(-1, case["heads"], d).to(s["q"].dtype), lse.reshape(-1, case["heads"])


def _plain_scores(s):
    d = s["case"]["dim"]
    keys = _fetch(s, s["pages"].long())[0].flatten(1, 3)  # one head: [n, rows, d]
    score = (_padded(s, s["q"].float()[:, 0]) @ keys.transpose(-1, -2)) * (1 / math.sqrt(d))
    seq, at = _whose(s)
    col = torch.arange(keys.shape[1], device="cuda").expand(s["questions"], -1)
    place, there = _entries(s, col)
    m, ok = _mask_of(s, col)
    score = torch.where(ok, score[seq, at] + m, -1e30)
    out = torch.zeros_like(s["scores"])
    out[place[there]] = score[there]
    return out


def _plain_write(s):
    case = s["case"]
    fmt, kv, d = case["format"], case["kv_heads"], case["dim"]
    seq, at = _whose(s)
    start = s["lengths"].long() - (s["q_off"][1:] - s["q_off"][:-1])
    pos = start[seq] + at
    page = s["pages"].long()[seq, pos // PAGE][:, None]
    half, row = (pos % PAGE // CELL)[:, None], (pos % CELL)[:, None]
    head = torch.arange(kv, device="cuda")[None, :]
    kc, vc, ks, vs, bounds = _split(s)
    back = []
    for x, codes, scales, place in zip((s["keys"], s["values"]), (kc, vc), (ks, vs), _places(d, pos.device)):
        c, sc = _quantise(x, fmt)
        where = place[row[:, 0]][:, None, :].expand(c.shape)
        codes[page, head, half, row] = c.gather(-1, where) if d > 32 else c
        scales[page, head, half, row] = sc
        c = codes[page, head, half, row]
        c = c.gather(-1, where) if d > 32 else c
        back.append((_decode(c, fmt) * scales[page, head, half, row][..., None]).to(x.dtype))
    # the bounds of the pages that have new rows, over all that they hold
    first, n = start // PAGE, (s["lengths"].long() + PAGE - 1) // PAGE
    block = first[:, None] + torch.arange(s["max_q"] // PAGE + 2, device="cuda")
    touched = (block < n[:, None]) & (s["lengths"].long() > start)[:, None]
    which = torch.arange(case["seqs"], device="cuda")[:, None].expand(block.shape)[touched]
    block = block[touched]
    page = s["pages"].long()[which, block]
    step = max(1, (1 << 28) // (kv * PAGE * d))
    for a in range(0, page.numel(), step):
        p = page[a:a + step]
        c = kc[p]
        c = c.gather(-1, _places(d, p.device)[0].expand(c.shape)) if d > 32 else c
        y = (_decode(c, fmt) * ks[p][..., None]).flatten(2, 3)
        held = s["lengths"].long()[which[a:a + step]] - block[a:a + step] * PAGE
        ok = (torch.arange(PAGE, device="cuda") < held[:, None])[:, None, :, None]
        bounds[p] = torch.stack([torch.where(ok, y, math.inf).amin(2), torch.where(ok, y, -math.inf).amax(2)], 2)
    return back[0], back[1], bounds


# --- the framework's calls ---------------------------------------------------

_backend = None


def _handle():
    """The handle that a user's program keeps, on the stream the program works on."""
    global _backend
    if _backend is None:
        from krystal_b200 import BRAIN_FORWARD_CONFIG, create_brain_forward_weights, cuda_backend
        cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
        _backend = cuda_backend(0)(cfg, create_brain_forward_weights(cfg, 1337))
        _backend.set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: the default stream
    return _backend


def _own(s):
    from krystal_b200 import cache as kc
    be, case = _handle(), s["case"]
    ptr = lambda name: s[name].data_ptr() if s.get(name) is not None else None  # noqa: E731
    if "cache" not in s:  # a program's cache and page table stay where they are
        s["cache"] = kc.BankCache(s["page_count"], case["kv_heads"], case["dim"], case["format"], storage=s["storage"])
        s["table"] = kc.page_table(ptr("pages"), ptr("lengths"), case["seqs"], s["pitch"], s["max_r"])
        if case["op"] == "write":
            s["rows"] = kc.cache_rows(ptr("keys"), ptr("values"), case["dtype"], s["questions"], ptr("q_off"))
            s["rows_out"] = kc.cache_rows(ptr("keys_out"), ptr("values_out"), case["dtype"], s["questions"],
                                          ptr("q_off"))
        else:
            s["ask"] = kc.questions(ptr("q"), case["dtype"], s["questions"], case["heads"], ptr("q_off"), s["max_q"])
        if case["op"] in ("attend", "sparse"):
            size = be.attend_workspace(s["cache"], s["table"], s["ask"], case.get("blocks", 0))
            s["space"] = torch.empty(max(1, size), dtype=torch.uint8, device="cuda")
    c, t = s["cache"], s["table"]
    if case["op"] == "write":
        be.cache_write(c, t, s["rows"])
        be.cache_read(c, t, s["rows_out"])
        return s["keys_out"], s["values_out"], c.bounds()
    mask = {"mask": ptr("mask"), "mask_off": ptr("p_off")} if case["mask"] else {}
    if case["op"] == "scores":
        be.cache_scores(c, t, s["ask"], ptr("scores"), ptr("p_off"), mask=ptr("mask"))
        return s["scores"]
    if case["op"] == "sparse":
        be.cache_blocks(c, t, s["ask"], case["blocks"], case["recent"], ptr("blocks"))
        mask.update(blocks=ptr("blocks"), block_count=case["blocks"])
    be.cache_attend(c, t, s["ask"], ptr("out"), lse=ptr("lse"), workspace=s["space"].data_ptr(),
                    workspace_bytes=s["space"].numel(), **mask)
    return (s["blocks"], s["out"], s["lse"]) if case["op"] == "sparse" else (s["out"], s["lse"])


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "attend": _plain_attend, "sparse": _plain_sparse,
            "scores": _plain_scores}[state["case"]["op"]](state)


# --- from the definitions, sequence by sequence in 64 bits ---------------------

def _meaning(fmt):
    """The 64-bit value of each of the 256 codes."""
    c = np.arange(256)
    if fmt == "i8":
        return c - 128.0
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)
    return np.where(c & 128, -v, v)


def _cached(s, table, pages, n, which):
    """The first n rows of the pages' keys (0) or values (1), f64 [kv, n, d]."""
    case = s["case"]
    kv, d, cell = case["kv_heads"], case["dim"], _cell_bytes(case["dim"])
    row = torch.arange(n, device="cuda")
    base = ((pages.long()[row // PAGE][None] * kv + torch.arange(kv, device="cuda")[:, None]) * 2
            + row % PAGE // CELL) * cell
    r, b = (row % CELL)[:, None], torch.arange(d, device="cuda")[None]
    flip = ((r // 4 % 2 * 64) if d == 128 else 0 * r) if which == 0 else (r % 4 * 32 if d == 128 else
                                                                         r // 2 % 2 * 32 if d == 64 else 0 * r)
    code = s["storage"][base[..., None] + which * CELL * d + r * d + (b ^ flip)]
    at = (base + 2 * CELL * d + which * CELL * 4) // 4 + row % CELL
    end = s["page_count"] * kv * 2 * cell
    return table[code.long()] * s["storage"][:end].view(torch.float32)[at].double()[..., None]


def _exact_write(s):
    case, top = s["case"], TOP[s["case"]["format"]]
    outs = []
    for x in (s["keys"], s["values"]):
        x = x.double()
        # the definition rounds the scale, and the quotient, to f32
        scale = (x.abs().amax(-1, keepdim=True) / top).float().double().clamp_min(LEAST)
        y = (x / scale).float().double()
        if case["format"] == "i8":
            c = y.round()
        else:  # the nearest of 8 steps a power of two, the lowest power 2^-6; halves go to the even
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
            c = ((y / step).round() * step).clamp(-top, top)
        outs.append(c * scale)
    bounds = _split(s)[4].double().clone()
    table = torch.from_numpy(_meaning(case["format"])).cuda()
    q_off, r = s["q_off"].tolist(), s["lengths"].tolist()
    for i in range(case["seqs"]):
        n = q_off[i + 1] - q_off[i]
        if not n:
            continue
        first = (r[i] - n) // PAGE
        old = _cached(s, table, s["pages"][i, first:], r[i] - n - first * PAGE, 0)
        keys = torch.cat([old, (outs[0][q_off[i]:q_off[i + 1]]).float().double().transpose(0, 1)], 1)
        whole = keys.shape[1] // PAGE * PAGE
        p = s["pages"][i, first:first + -(-keys.shape[1] // PAGE)].long()
        if whole:
            k = keys[:, :whole].unflatten(1, (-1, PAGE))
            bounds[p[:whole // PAGE]] = torch.stack([k.amin(2), k.amax(2)], 2).transpose(0, 1)
        if whole < keys.shape[1]:
            k = keys[:, whole:]
            bounds[p[-1]] = torch.stack([k.amin(1), k.amax(1)], 1)
    return outs[0], outs[1], bounds


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(s)
    table = torch.from_numpy(_meaning(case["format"])).cuda()
    kv, d, g = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    q_off, p_off, r = s["q_off"].tolist(), s["p_off"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["questions"], case["heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((s["questions"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    scores = torch.zeros(p_off[-1], dtype=torch.float64, device="cuda")
    chosen = _plain_sparse(s)[0] if case["op"] == "sparse" else None  # whole numbers, equal to the plain form's
    for i in range(case["seqs"]):
        n = q_off[i + 1] - q_off[i]
        if not n or not r[i]:
            continue
        q = s["q"][q_off[i]:q_off[i + 1]].double().view(n, kv, g, d)
        x = torch.einsum("qhgd,hrd->qhgr", q, _cached(s, table, s["pages"][i], r[i], 0)) / math.sqrt(d)
        if case["mask"]:
            m = s["mask"][p_off[i]:p_off[i + 1]].view(n, 1, 1, r[i]).double()
            x = torch.where(m > BLOCKED, x + m.clamp_max(-BLOCKED), -math.inf)
        if case["op"] == "scores":
            scores[p_off[i]:p_off[i + 1]] = torch.where(torch.isinf(x), -1e30, x).flatten()
            continue
        if chosen is not None:
            c = chosen[q_off[i]:q_off[i + 1]].long()
            seen = torch.zeros(n, kv, s["pitch"] + 1, dtype=torch.bool, device="cuda")
            seen.scatter_(2, torch.where(c >= 0, c, s["pitch"]), True)
            block = torch.arange(r[i], device="cuda") // PAGE
            x = torch.where(seen[:, :, block][:, :, None], x, -math.inf)
        z = torch.logsumexp(x, -1)
        w = torch.where(torch.isfinite(z)[..., None], torch.exp(x - z[..., None]), 0.0)
        lse[q_off[i]:q_off[i + 1]] = z.reshape(n, -1)
        y = torch.einsum("qhgr,hrd->qhgd", w, _cached(s, table, s["pages"][i], r[i], 1))
        out[q_off[i]:q_off[i + 1]] = y.reshape(n, -1, d)
    if case["op"] == "scores":
        return scores
    return (None, out, lse) if case["op"] == "sparse" else (out, lse)
