"""Sessions whose banks stay on the device: each turn encodes its own records only.

``BrainSession.think`` (packages/krystal/src/host/session.ts:128-181) encodes a
frame's whole bank every turn. ``SessionBanks`` keeps what earlier turns encoded
to in caches (``cache.BankCache``), hands out their pages, and runs a turn of any
of its sessions through ``CudaBrainBackend.bank_turn``: the turn's bank records
are appended, its questions answered over all that the session has been told.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Hashable, Sequence

import numpy as np

from . import abi
from .cache import PAGE, BankCache, page_table
from .frame import QUERY_BAND, pack_frame_batch
from .policy import Sampling


@dataclass
class TurnAnswers:
    """One session's answers of a turn: its questions in the order they came."""

    index: np.ndarray  # u32 [Q], a bank row counted from the session's first, KC_NO_SELECTION for an empty row
    p: np.ndarray      # [Q, R] over all R rows the session holds
    logp: np.ndarray   # [Q] log probability of the answer


class SessionBanks:
    """Caches for the banks of many sessions, in ``pages`` pages of 64 records
    that the sessions share; a session holds at most ``max_length`` records. The
    brain's weights are those of the turns: records that a weight change finds
    cached keep what they encoded to (``drop`` the sessions to tell them again)."""

    def __init__(self, backend, pages: int, max_length: int, format: str = "i8"):
        import torch
        self.torch = torch
        self.backend, self.max_length = backend, int(max_length)
        if not 1 <= self.max_length <= abi.KC_MAX_ROW:
            raise ValueError(f"a session holds 1 to {abi.KC_MAX_ROW} records")
        c = backend.config
        self.mixer = [BankCache(pages, c.head_count, c.head_dim, format, device=backend.device)
                      for _ in range(c.mixer_blocks)]
        self.selector = BankCache(pages, 1, c.hidden_size, format, device=backend.device)
        self.free = list(range(int(pages)))[::-1]
        self.pages: dict[Hashable, list[int]] = {}
        self.lengths: dict[Hashable, int] = {}

    def length(self, session: Hashable) -> int:
        """Bank records that the session holds."""
        return self.lengths.get(session, 0)

    def drop(self, session: Hashable) -> None:
        """Forgets a session; its pages go to others."""
        self.free.extend(self.pages.pop(session, []))
        self.lengths.pop(session, None)

    def cut(self, session: Hashable, length: int) -> None:
        """Takes the session back to its first ``length`` records."""
        if not 0 <= length <= self.length(session):
            raise ValueError(f"the session holds {self.length(session)} records")
        self._shrink(session, length)

    def _shrink(self, session, length):
        held = self.pages.get(session, [])
        keep = -(-length // PAGE)
        self.free.extend(held[keep:])
        del held[keep:]
        if session in self.lengths:
            self.lengths[session] = length

    def turn(self, turns: Sequence[tuple[Hashable, Sequence]], masks: Sequence[np.ndarray] | None = None,
             uniforms=None, sampling: Sampling | None = None) -> list[TurnAnswers]:
        """A turn of each of ``turns``' sessions, (session, its records of this
        turn: questions in the query band, bank records in the others). masks:
        per turn a [Q, R] selection mask over all rows the session then holds
        (-1e30 blocked, 0 open). uniforms ([all questions] f64) draw the answers,
        by ``sampling`` (host arrays as row limits) or the whole distribution."""
        torch = self.torch
        names = [s for s, _ in turns]
        if len(set(names)) != len(names):
            raise ValueError("a session takes one turn at a time")
        if not turns:
            return []
        if masks is not None and len(masks) != len(turns):
            raise ValueError(f"a mask per turn is needed ({len(turns)})")
        batch = pack_frame_batch([r for _, r in turns])
        rec = np.diff(batch.rec_off.astype(np.int64))
        asks = np.bincount(np.repeat(np.arange(len(turns)), rec), weights=batch.band_ids == QUERY_BAND,
                           minlength=len(turns)).astype(np.int64)
        before = [self.length(s) for s in names]
        after = [n + int(r - q) for n, r, q in zip(before, rec, asks)]
        questions, longest = int(asks.sum()), max(1, max(after))
        if longest > self.max_length:
            raise ValueError(f"a session would hold {longest} records, more than {self.max_length}")
        need = sum(-(-n // PAGE) - len(self.pages.get(s, [])) for s, n in zip(names, after))
        if need > len(self.free):
            raise ValueError(f"the turn needs {need} more pages, {len(self.free)} are free")
        mask = None
        if masks is not None:
            mask = np.zeros((questions, longest), np.float32)
            at = 0
            for m, q, n in zip(masks, asks, after):
                m = np.asarray(m, np.float32)
                if m.size != q * n:
                    raise ValueError(f"a turn's mask must be [{q}, {n}]")
                mask[at:at + q, :n] = m.reshape(q, n)
                at += q
        if uniforms is not None:
            uniforms = np.ascontiguousarray(uniforms, np.float64)
            if uniforms.size != questions:
                raise ValueError(f"uniforms must have one entry per question ({questions})")
        known = [s in self.lengths for s in names]
        try:
            for s, n in zip(names, after):
                held = self.pages.setdefault(s, [])
                held.extend(self.free.pop() for _ in range(-(-n // PAGE) - len(held)))
                self.lengths[s] = n
            pitch = max(1, -(-longest // PAGE))
            table = np.zeros((len(names), pitch), np.uint32)
            for i, s in enumerate(names):
                table[i, :len(self.pages[s])] = self.pages[s]
            device = f"cuda:{self.backend.device}"

            def up(a, dtype):
                return torch.from_numpy(np.ascontiguousarray(a).view(dtype)).to(device)

            keep = [up(table, np.int32), up(np.array(after, np.uint32), np.int32),
                    up(batch.rec_off.astype(np.uint64), np.int64)]
            keep += [up(np.asarray(a, np.uint32), np.int32) for a in (batch.token_ids, batch.field_roles,
                                                                     batch.schema_ids, batch.band_ids)]
            keep += [None if a is None else torch.from_numpy(a).to(device) for a in (uniforms, mask)]
            limits, policy = [], None
            if sampling is not None:
                for name, dtype in (("row_temperature", np.float32), ("row_top_k", np.uint32),
                                    ("row_top_p", np.float32), ("row_min_p", np.float32)):
                    v = getattr(sampling, name)
                    if v is not None:
                        v = np.ascontiguousarray(v, dtype)
                        if v.size != questions:
                            raise ValueError(f"{name} must have one entry per question ({questions})")
                        v = up(v, np.int32)
                    limits.append(v)
                policy = Sampling(sampling.temperature, sampling.top_k, sampling.top_p, sampling.min_p,
                                  *(v.data_ptr() if v is not None else None for v in limits))
            p = torch.empty(max(1, questions), longest, device=device)
            index = torch.empty(max(1, questions), dtype=torch.int32, device=device)
            logp = torch.empty(max(1, questions), device=device)
            ptr = [t.data_ptr() if t is not None else None for t in keep]
            torch.cuda.current_stream(self.backend.device).synchronize()  # the handle may work on another stream
            self.backend.bank_turn(batch.frames, batch.records, *ptr[2:7], self.mixer, self.selector,
                                   page_table(ptr[0], ptr[1], len(names), pitch, longest), p.data_ptr(), questions,
                                   index=index.data_ptr(), logp=logp.data_ptr(), uniforms=ptr[7], mask=ptr[8],
                                   sampling=policy)
            p, index, logp = p.cpu().numpy(), index.cpu().numpy().view(np.uint32), logp.cpu().numpy()
        except BaseException:
            for s, n, had in zip(names, before, known):
                self._shrink(s, n) if had else self.drop(s)
            raise
        out, at = [], 0
        for q, n in zip(asks, after):
            out.append(TurnAnswers(index[at:at + q].copy(), p[at:at + q, :n].copy(), logp[at:at + q].copy()))
            at += int(q)
        return out
