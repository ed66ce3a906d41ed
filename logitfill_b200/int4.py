"""A 4-bit paged Key/Value cache, attention over it, and attention over the
pages that matter.

The tiered cache of :mod:`logitfill_b200.packed` needs a Key policy from an
offline calibration and stores Value at 2 bits.  This one needs none: Key and
Value are both held at 4 bits, quantized token by token as they are written
(an fp16 scale and minimum for every 32 channels: 5 bits per element in all),
in 64-token pages that a page table orders into sequences.

* :func:`int4_write` / :func:`int4_read` quantize tokens into the pages and
  read them back;
* :func:`int4_attention` attends query tokens over the cached tokens;
* :func:`int4_select` scores a sequence's pages by a bound on their attention
  scores and picks the best for each query token and KV head, and
  :func:`int4_sparse_attention` attends over the picked pages only;
* :class:`Int4KVCache` keeps the pools, the page table and the lengths of a
  batch of sequences, for every layer of a model.

The functions take the tensors themselves: ``pages`` int32 ``[n_pages, n_kv,
20 * head_dim]`` (see ``include/logitfill_b200.h`` for the record),
``page_table`` int32 ``[batch, width]``, lengths and positions int32
``[batch]``, all on the GPU.  Sequences may share pages that are not written
any more (a common prefix); a page that a call writes belongs to one of its
sequences.  A page table entry outside the pool is never followed; with
``status`` (int32 ``[1]`` on the GPU) given, such an access sets it to a
non-zero ``lf_status``.  Every launch goes to the current stream.  There is no
CPU or dense fallback; what the kernels do not implement raises
``NotImplementedError``, malformed arguments ``ValueError``.
"""
from __future__ import annotations

import numpy as np
import torch

from logitfill_b200 import _lib

PAGE_TOKENS = 64   # tokens of a page
GROUP = 32         # channels that share a scale and a minimum


def record_words(head_dim: int) -> int:
    """int32 words of one page and KV head."""
    return 20 * int(head_dim)


def bounds_bytes(head_dim: int) -> int:
    """int8 entries of the bounds record of one page and KV head."""
    return 2 * int(head_dim) + 16


def alloc_pages(n_pages: int, n_kv: int, head_dim: int, device="cuda") -> torch.Tensor:
    """An empty pool (zeros) of ``n_pages`` pages."""
    return torch.zeros(n_pages, n_kv, record_words(head_dim), dtype=torch.int32, device=device)


def alloc_bounds(n_pages: int, n_kv: int, head_dim: int, device="cuda") -> torch.Tensor:
    """Bounds records (zeros) of ``n_pages`` pages."""
    return torch.zeros(n_pages, n_kv, bounds_bytes(head_dim), dtype=torch.int8, device=device)


def int4_write(key: torch.Tensor, value: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor,
               start: torch.Tensor, counts: torch.Tensor | None = None, bounds: torch.Tensor | None = None,
               status: torch.Tensor | None = None) -> None:
    """Quantize ``key``/``value`` ``[batch, n_kv, T, head_dim]`` (fp32, fp16 or
    bf16, any strides) into the pages: token ``i`` of sequence ``b`` goes to
    position ``start[b] + i``, for ``i < counts[b]`` (all ``T`` where ``counts``
    is None).  With ``bounds`` given, the record of every page whose last slot
    is written is brought up to date (a sparse call needs it).  A group of 32
    channels whose scale or minimum is no finite fp16 number (a NaN, an
    infinity, a range past 15 * 65504) reads back as NaN."""
    _lib.int4_binding().write(key, value, pages, page_table, start, counts, bounds, status)


def int4_read(pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor, tokens: int,
              counts: torch.Tensor | None = None, dtype=torch.float32, status: torch.Tensor | None = None):
    """Positions ``start[b] .. start[b] + tokens - 1`` of every sequence as Key and
    Value ``[batch, n_kv, tokens, head_dim]`` in ``dtype`` (fp32, fp16 or
    bf16); tokens ``i >= counts[b]`` are zeros."""
    return _lib.int4_binding().read(pages, page_table, start, tokens, counts, dtype, status)


def int4_read_bounds(bounds: torch.Tensor) -> torch.Tensor:
    """fp32 ``[n_pages, n_kv, 2, head_dim]`` of the bounds records: every Key
    channel's upper, then its lower bound over a page's tokens."""
    return _lib.int4_binding().read_bounds(bounds)


def int4_attention(query: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                   scaling: float, counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``query`` ``[batch, n_q, head_dim]`` (one token per
    sequence) or ``[batch, n_q, q_len, head_dim]`` over the cached tokens, fp16
    or bf16, in the query's shape and type.  ``lengths[b]`` tokens are cached,
    the query's own among them (written first): query token ``i`` sees
    positions ``0 .. lengths[b] - q_len + i``.  With ``counts`` (int32
    ``[batch]``) sequence ``b`` has only its first ``counts[b]`` query tokens;
    the others, and those that see nothing, get zeros."""
    return _lib.int4_binding().attend(query, pages, page_table, lengths, scaling, counts, out, status)


def int4_select(query: torch.Tensor, pages: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor,
                lengths: torch.Tensor, top_pages: int, sink_pages: int = 1, recent_pages: int = 2,
                counts: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """The logical pages each query token and KV head reads in a sparse call:
    int32 ``[batch, q_len, n_kv, sink + recent + top]``, ascending, -1 after the
    last.  The first ``sink_pages`` and the last ``recent_pages`` (at least 1:
    the page being filled) are always in; of the rest the ``top_pages`` with
    the largest bound on the scores of the KV head's queries (summed over its
    query heads; ties to the lower page)."""
    return _lib.int4_binding().attend(query, pages, page_table, lengths, 0.0, counts, None, status, bounds, top_pages,
                                      sink_pages, recent_pages, True)


def int4_sparse_attention(query: torch.Tensor, pages: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor,
                          lengths: torch.Tensor, scaling: float, top_pages: int, sink_pages: int = 1,
                          recent_pages: int = 2, counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                          status: torch.Tensor | None = None):
    """:func:`int4_select` (of the negated query where ``scaling`` is negative),
    then :func:`int4_attention` over the picked pages only: ``(out, picked)``.  With ``sink + recent + top`` pages or fewer
    visible, every page is read and the result is the dense one."""
    return _lib.int4_binding().attend(query, pages, page_table, lengths, scaling, counts, out, status, bounds, top_pages,
                                      sink_pages, recent_pages)


class Int4KVCache:
    """4-bit cache of ``batch`` sequences for ``n_layers`` layers: a pool of
    ``n_pages`` 64-token pages per layer, shared by the sequences through one
    page table (a sequence's token positions are the same in every layer).

    A step is ``extend(counts)``, then for every layer ``write(layer, key,
    value)`` and ``attend(layer, query, scaling)``: ``extend`` makes room for
    the step's tokens, ``write`` stores them behind the tokens of the steps
    before, ``attend`` sees both.  Pages come from a free list and go back with
    ``release``.

    Capturing a step in a CUDA graph: ``reserve`` pages for all tokens to come,
    capture ``extend(n)`` (an int) with the rest of the step, and call
    ``advance_host(n)`` for each replay."""

    def __init__(self, n_layers: int, batch: int, n_q: int, n_kv: int, head_dim: int, n_pages: int,
                 max_tokens: int, device="cuda", bounds: bool = True):
        if n_q % n_kv:
            raise ValueError("query heads must divide into KV heads")
        if head_dim not in (64, 128):
            raise NotImplementedError(f"the 4-bit cache takes head_dim 64 or 128, got {head_dim}")
        if n_layers < 1 or batch < 1 or n_pages < 1 or max_tokens < 1:
            raise ValueError("layers, batch, pages and max_tokens must be positive")
        self.batch, self.n_q, self.n_kv, self.head_dim = int(batch), int(n_q), int(n_kv), int(head_dim)
        self.n_pages = int(n_pages)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.width = -(-int(max_tokens) // PAGE_TOKENS)
        self.pages = [alloc_pages(n_pages, n_kv, head_dim, self.device) for _ in range(n_layers)]
        self.bounds = [alloc_bounds(n_pages, n_kv, head_dim, self.device) for _ in range(n_layers)] if bounds else None
        self.page_table = torch.full((batch, self.width), -1, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        spans = torch.zeros(3, batch, dtype=torch.int32, device=self.device)
        self.start, self.end, self.counts = spans.unbind(0)     # device: first new position, length, new tokens
        self._spans = spans
        self._table = np.full((batch, self.width), -1, np.int32)  # host, authoritative
        self._owned = np.zeros(batch, np.int64)                   # pages each sequence holds
        self._end = np.zeros(batch, np.int64)
        self._start = np.zeros(batch, np.int64)
        self._step = 0                                            # tokens of the step, at most
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def n_layers(self) -> int:
        return len(self.pages)

    @property
    def lengths(self) -> np.ndarray:
        """Tokens of each sequence, the current step's among them (host)."""
        return self._end.copy()

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, tokens) -> None:
        """Hold pages for ``tokens`` tokens in all (an int, or one per
        sequence).  Raises ``RuntimeError`` when the pool has too few; nothing
        changes then."""
        want = -(-np.broadcast_to(np.asarray(tokens, np.int64), (self.batch,)) // PAGE_TOKENS)
        if want.max(initial=0) > self.width:
            raise ValueError(f"{int(np.max(tokens))} tokens exceed the cache's {self.width * PAGE_TOKENS} per sequence")
        need = np.maximum(want - self._owned, 0)
        if not need.any():
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("reserve the pages before the capture")
        if need.sum() > len(self._free):
            raise RuntimeError(f"{int(need.sum())} pages are needed, {len(self._free)} are free")
        for b in np.flatnonzero(need):
            for j in range(int(self._owned[b]), int(want[b])):
                self._table[b, j] = self._free.pop()
            self._owned[b] = want[b]
        self._upload(self.page_table, self._table)

    def _upload(self, device_tensor: torch.Tensor, host: np.ndarray) -> None:
        # Pinned, non-blocking: ordered on the stream without stalling the host.
        device_tensor.copy_(torch.from_numpy(host.astype(np.int32)).pin_memory(), non_blocking=True)

    def extend(self, counts) -> None:
        """Open a step of ``counts`` new tokens (an int, or one per sequence,
        0 for a sequence that pauses) behind those of the step before."""
        uniform = np.ndim(counts) == 0
        n = np.broadcast_to(np.asarray(counts, np.int64), (self.batch,))
        if (n < 0).any():
            raise ValueError("counts must not be negative")
        self.reserve(self._end + n)
        self._step = int(n.max())
        if torch.cuda.is_current_stream_capturing():
            if not uniform:
                raise RuntimeError("a captured step takes the same number of tokens for every sequence")
        else:
            self._start, self._end = self._end, self._end + n
            if not uniform:
                self._upload(self._spans, np.stack([self._start, self._end, n]))
                return
        self.start.copy_(self.end)
        self.end.add_(int(counts))
        self.counts.fill_(int(counts))

    def advance_host(self, count: int) -> None:
        """Mirror one replay of a captured ``extend(count)`` in the host lengths."""
        self._start, self._end = self._end, self._end + int(count)

    def truncate(self, lengths) -> None:
        """Drop the tokens past ``lengths`` (an int, or one per sequence), e.g.
        rejected drafts; the pages stay with their sequences."""
        n = np.broadcast_to(np.asarray(lengths, np.int64), (self.batch,))
        if (n < 0).any() or (n > self._end).any():
            raise ValueError("truncate() takes lengths between 0 and the present ones")
        self._start, self._end, self._step = n.copy(), n.copy(), 0
        self._upload(self._spans, np.stack([self._start, self._end, np.zeros_like(n)]))

    def release(self, seqs=None) -> None:
        """Empty the sequences ``seqs`` (default: all) and return their pages."""
        every = range(self.batch)
        for b in every if seqs is None else [every[s] for s in seqs]:   # all are looked up before the first is emptied
            for j in range(int(self._owned[b]) - 1, -1, -1):
                self._free.append(int(self._table[b, j]))
            self._table[b, :] = -1
            self._owned[b] = self._start[b] = self._end[b] = 0
        self._step = int((self._end - self._start).max())
        self._upload(self.page_table, self._table)
        self._upload(self._spans, np.stack([self._start, self._end, self._end - self._start]))

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Store this step's tokens of one layer: ``[batch, n_kv, T, head_dim]``,
        the first ``counts[b]`` of sequence ``b`` (``T`` is the largest count at
        least)."""
        if key.dim() == 4:
            self._check_step("key", key.shape[2])
        int4_write(key, value, self.pages[layer], self.page_table, self.start, self.counts,
                   None if self.bounds is None else self.bounds[layer], self.status)

    def read(self, layer: int, start: int = 0, stop: int | None = None, dtype=torch.float32):
        """Positions ``start .. stop - 1`` (default: to the longest sequence's
        end) of every sequence as ``[batch, n_kv, stop - start, head_dim]``;
        zeros past a sequence's end."""
        stop = int(self._end.max()) if stop is None else int(stop)
        if start < 0 or stop < start:
            raise ValueError(f"cannot read positions {start} .. {stop}")
        first = torch.full_like(self.start, start)
        return int4_read(self.pages[layer], self.page_table, first, stop - start, self.end - first, dtype, self.status)

    def attend(self, layer: int, query: torch.Tensor, scaling: float, out: torch.Tensor | None = None) -> torch.Tensor:
        """:func:`int4_attention` of this step's query tokens (the first
        ``counts[b]`` of sequence ``b``; all of the step's)."""
        self._check_query(query)
        return int4_attention(query, self.pages[layer], self.page_table, self.end, scaling, self.counts, out, self.status)

    def attend_sparse(self, layer: int, query: torch.Tensor, scaling: float, top_pages: int, sink_pages: int = 1,
                      recent_pages: int = 2, out: torch.Tensor | None = None):
        """:func:`int4_sparse_attention` of this step's query tokens."""
        if self.bounds is None:
            raise RuntimeError("a sparse call needs a cache made with bounds=True")
        self._check_query(query)
        return int4_sparse_attention(query, self.pages[layer], self.bounds[layer], self.page_table, self.end, scaling,
                                     top_pages, sink_pages, recent_pages, self.counts, out, self.status)

    def _check_query(self, query: torch.Tensor) -> None:
        if query.dim() < 3 or query.shape[1] != self.n_q:
            raise ValueError(f"query must have {self.n_q} heads, got {tuple(query.shape)}")
        self._check_step("query", query.shape[2] if query.dim() == 4 else 1)

    def _check_step(self, name: str, tokens: int) -> None:
        # extend() has counted the step's tokens already
        if tokens < self._step:
            raise ValueError(f"{name} has {tokens} tokens per sequence, the step has {self._step}")

    def check_status(self) -> None:
        """Raise if a kernel met a position outside its sequence's pages (synchronises)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            _lib.check(code, "4-bit cache kernel")


__all__ = ["PAGE_TOKENS", "GROUP", "record_words", "bounds_bytes", "alloc_pages", "alloc_bounds", "int4_write",
           "int4_read", "int4_read_bounds", "int4_attention", "int4_select", "int4_sparse_attention", "Int4KVCache"]
