"""The bank cache: encoded records kept on the device in 8 bits from turn to turn.

The reference encodes a session's whole frame every turn (packages/krystal/src/
host/session.ts:128-147), though what a record encodes to depends on the record
alone. ``BankCache`` holds keys and values of many sessions' records in pages;
``page_table`` names each session's pages and length. ``CudaBrainBackend`` writes
rows to it (``cache_write``), reads them back (``cache_read``), attends questions
over it (``cache_attend``), over the blocks a bound of their scores selects
(``cache_blocks``), and takes pointer scores from it (``cache_scores``).

The helpers take raw device pointers, as the backend's other device entry points
do.
"""
from __future__ import annotations

import weakref

from . import abi
from .policy import _dtype

FORMATS = {"i8": abi.KC_CACHE_I8, "e4m3": abi.KC_CACHE_E4M3}
PAGE = abi.KC_CACHE_PAGE


class BankCache:
    """Pages of 64 rows of ``kv_heads`` keys and values of ``head_dim``
    (kc_cache_view). ``storage``: a CUDA uint8 tensor of at least
    ``BankCache.bytes_for(...)`` bytes, or None for one of its own on ``device``.
    A cache dropped while its calls are queued leaves the storage with their
    backends until the stream has passed them; once a call that waits for the
    stream has returned (synchronize, bank_turn) a drop frees it. A captured
    call's cache has to live as long as its graph."""

    def __init__(self, pages: int, kv_heads: int = 4, head_dim: int = 32, format: str = "i8", storage=None,
                 device: int = 0):
        import torch
        if format not in FORMATS:
            raise ValueError(f"unknown cache format {format!r}: one of {', '.join(FORMATS)}")
        self.pages, self.kv_heads, self.head_dim, self.format = int(pages), int(kv_heads), int(head_dim), format
        if self.pages < 1 or not 1 <= self.kv_heads <= 128 or self.head_dim not in (32, 64, 128):
            raise ValueError("a cache has at least one page, 1 to 128 kv_heads and a head_dim of 32, 64 or 128")
        size = self.bytes_for(pages, kv_heads, head_dim)
        if storage is None:
            storage = torch.empty(size, dtype=torch.uint8, device=f"cuda:{device}")
        if storage.dtype != torch.uint8 or storage.device.type != "cuda" or not storage.is_contiguous():
            raise ValueError("a cache's storage is a contiguous CUDA tensor of uint8")
        if storage.numel() < size:
            raise ValueError(f"a cache of {pages} pages needs {size} bytes of storage")
        self.storage, self.device = storage, storage.device
        self.view = abi.KcCacheView(storage.data_ptr(), storage.numel(), self.pages, self.kv_heads, self.head_dim,
                                    FORMATS[format])
        self.backends = []  # weak references to those that queued a call on it, and each one's last ticket

    @staticmethod
    def bytes_for(pages: int, kv_heads: int = 4, head_dim: int = 32) -> int:
        """kc_cache_bytes."""
        return int(abi.load().kc_cache_bytes(pages, kv_heads, head_dim))

    def bounds(self):
        """[pages, kv_heads, 2, head_dim] f32, a view of the storage: the smallest
        and the largest of the keys that each page held when it was last written to."""
        import torch
        n = self.pages * self.kv_heads * 2 * self.head_dim * 4
        size = self.bytes_for(self.pages, self.kv_heads, self.head_dim)
        return self.storage[size - n:size].view(torch.float32).view(self.pages, self.kv_heads, 2, self.head_dim)

    def queued_on(self, backend) -> None:
        ticket = backend.ticket()
        last = self.backends[-1] if self.backends else None
        if last and last[0]() is backend:
            last[1] = ticket
        else:
            self.backends = [b for b in self.backends if b[0]() is not None and b[0]() is not backend]
            self.backends.append([weakref.ref(backend), ticket])

    def __del__(self):
        for r, ticket in getattr(self, "backends", ()):
            backend = r()
            if backend is not None and not backend.passed(ticket):
                backend.hold_clip((self.storage,))


def page_table(pages: int | None, lengths: int, sequences: int, pitch: int, max_length: int = 0) -> abi.KcPageTable:
    """Where ``sequences`` sequences lie: row i of sequence s in page
    pages[s * pitch + i // 64] (u32 [sequences, pitch]); lengths u32 [sequences].
    max_length bounds the lengths (0: what the pages hold)."""
    return abi.KcPageTable(pages, lengths, sequences, pitch, max_length)


def cache_rows(keys: int | None, values: int | None, dtype: str, rows: int, row_off: int | None = None,
               pitch: int = 0) -> abi.KcCacheRows:
    """[rows, kv_heads, head_dim] keys and values, a sequence's at row_off (u64
    [sequences + 1]; None: one row a sequence)."""
    return abi.KcCacheRows(keys, values, row_off, rows, pitch, _dtype(dtype))


def questions(q: int, dtype: str, questions: int, heads: int, q_off: int | None = None, max_questions: int = 0,
              pitch: int = 0) -> abi.KcQuestionView:
    """[questions, heads, head_dim] questions, a sequence's at q_off (u64
    [sequences + 1]; None: one a sequence); max_questions bounds one sequence's."""
    return abi.KcQuestionView(q, q_off, questions, heads, max_questions, _dtype(dtype), pitch)
