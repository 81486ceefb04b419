"""The policy an answer is drawn from, and the lists its learning clips.

The reference draws from a question's whole distribution (sampleRow,
packages/krystal/src/forward/sampling.ts:41-57). ``Sampling`` names a tempered
and cut policy instead: ``BrainSession.think(sampling=...)``,
``CudaBrainBackend.forward_batch`` / ``select_batch`` / ``draw*`` draw from it,
``policy_loss`` and the backward (``set_policy``, ``LearnOptions.sampling``)
differentiate it. ``GradList`` names the gradients of one global norm
(``clip_grads``, ``LearnOptions.max_update_norm``).

The row and list helpers take raw device pointers, as the backend's other
device entry points do.
"""
from __future__ import annotations

import ctypes as C
import weakref
from dataclasses import dataclass

import numpy as np

from . import abi

DTYPES = {"f32": abi.KC_DTYPE_F32, "f16": abi.KC_DTYPE_F16, "bf16": abi.KC_DTYPE_BF16, "f64": abi.KC_DTYPE_F64}
KINDS = {"scores": abi.KC_ROWS_SCORES, "p": abi.KC_ROWS_P}


@dataclass
class Sampling:
    """kc_sampling: temperature, then top-k, top-p and min-p (the defaults cut
    nothing; temperature 0 is the first largest entry). The row_* limits
    replace a limit row by row: device pointers for the device entry points,
    arrays for the host ones."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    row_temperature: object = None
    row_top_k: object = None
    row_top_p: object = None
    row_min_p: object = None

    @property
    def whole(self) -> bool:
        """Whether every row is drawn from its whole distribution, as it is."""
        rows = (self.row_temperature, self.row_top_k, self.row_top_p, self.row_min_p)
        return (all(r is None for r in rows) and self.temperature == 1 and self.top_k == 0 and self.top_p >= 1
                and self.min_p == 0)

    def device_struct(self) -> abi.KcSampling:
        return abi.KcSampling(self.temperature, self.top_k, self.top_p, self.min_p, self.row_temperature,
                              self.row_top_k, self.row_top_p, self.row_min_p)

    def host_struct(self, rows: int) -> tuple[abi.KcSampling, list]:
        """The struct over host arrays, and what has to outlive the call."""
        keep = []

        def limit(name, dtype):
            v = getattr(self, name)
            if v is None:
                return None
            a = np.ascontiguousarray(v, dtype=dtype)
            if a.size != rows:
                raise ValueError(f"{name} must have one entry per question ({rows})")
            keep.append(a)
            return a.ctypes.data

        s = abi.KcSampling(self.temperature, self.top_k, self.top_p, self.min_p, limit("row_temperature", np.float32),
                           limit("row_top_k", np.uint32), limit("row_top_p", np.float32),
                           limit("row_min_p", np.float32))
        return s, keep


def _dtype(name: str) -> int:
    if name not in DTYPES:
        raise ValueError(f"unknown element type {name!r}: one of {', '.join(DTYPES)}")
    return DTYPES[name]


def _kind(name: str) -> int:
    if name not in KINDS:
        raise ValueError(f"unknown kind of rows {name!r}: one of {', '.join(KINDS)}")
    return KINDS[name]


def dense_rows(values: int, dtype: str, rows: int, row_len: int, row_pitch: int = 0,
               kind: str = "scores") -> abi.KcRowsView:
    """A [rows, row_len] matrix on the device, row i at values + i * row_pitch elements."""
    return abi.KcRowsView(values, None, None, rows, 0, row_len, row_pitch, _dtype(dtype), _kind(kind))


def ragged_rows(values: int, dtype: str, rows: int, frames: int, q_off: int | None, p_off: int, max_row: int = 0,
                kind: str = "scores") -> abi.KcRowsView:
    """A packed batch's rows on the device: frame f's [Q_f, R_f] block at
    p_off[f], its first question at q_off[f] (None: one row a frame). max_row
    bounds the longest row (0: the largest bank a frame may hold)."""
    return abi.KcRowsView(values, q_off, p_off, rows, frames, max_row, 0, _dtype(dtype), _kind(kind))


class GradList:
    """The gradients of one global norm: contiguous CUDA tensors of one device,
    where each clipped gradient goes (None: in place), and each one's factor
    in the norm. The list holds its tensors and its workspace; it is built once
    for gradients that stay where they are. A list dropped while its clip is
    queued leaves both with the backend until the stream has passed them. Two
    captured graphs that may run at once need a list each, and a graph's list
    has to live as long as the graph."""

    def __init__(self, tensors, outs=None, weights=None):
        import torch
        names = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.float64: "f64"}
        tensors = list(tensors)
        outs = tensors if outs is None else list(outs)
        weights = [1.0] * len(tensors) if weights is None else [float(w) for w in weights]
        if len(outs) != len(tensors) or len(weights) != len(tensors):
            raise ValueError("a gradient list needs one output and one weight per tensor")
        if not tensors:
            raise ValueError("a gradient list needs at least one tensor")
        self.device = tensors[0].device
        self.views = (abi.KcGradView * len(tensors))()
        for i, (t, o, w) in enumerate(zip(tensors, outs, weights)):
            if t.dtype not in names:
                raise ValueError(f"gradient {i} is {t.dtype}: f32, f16, bf16 or f64 is needed")
            if o.dtype != t.dtype or o.numel() != t.numel():
                raise ValueError(f"output {i} must have its gradient's type and size")
            for x in (t, o):
                if x.device.type != "cuda" or x.device != self.device:
                    raise ValueError("a gradient list's tensors lie on one CUDA device")
                if not x.is_contiguous():
                    raise ValueError(f"gradient {i} and its output must be contiguous")
            self.views[i] = abi.KcGradView(t.data_ptr(), o.data_ptr(), t.numel(), w, DTYPES[names[t.dtype]])
        self.keep = (tensors, outs)
        self.count = len(tensors)
        self.workspace_bytes = int(abi.load().kc_clip_workspace(self.count))
        self.workspace = torch.empty(self.workspace_bytes // 8, dtype=torch.float64, device=self.device)
        self.address = C.addressof(self.views)
        self.backends = []  # weak references to those that queued a clip of the list

    def queued_on(self, backend) -> None:
        if not any(r() is backend for r in self.backends):
            self.backends.append(weakref.ref(backend))

    def __del__(self):
        for r in getattr(self, "backends", ()):
            backend = r()
            if backend is not None:
                backend.hold_clip((self.keep, self.workspace))
