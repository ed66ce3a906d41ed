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
* :func:`int4_prefix_attention` reads the pages that sequences share once for
  all of them;
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
from logitfill_b200.prompt import rotary_embed

PAGE_TOKENS = 64   # tokens of a page
GROUP = 32         # channels that share a scale and a minimum
MAX_GROUPS = 4096  # groups of sequences that share pages, of one call


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


def int4_prefix_attention(query: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                          scaling: float, prefix_group: torch.Tensor, prefix_pages: torch.Tensor,
                          counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                          status: torch.Tensor | None = None, always: bool = False) -> torch.Tensor:
    """:func:`int4_attention` where sequences share their first pages (a system
    prompt, a document that several ask about, or, for one sequence with many
    query tokens, its own history): the shared pages are read and unpacked once
    for all of a group's queries.

    ``prefix_group`` (int32 ``[batch]``) names each sequence's group (outside ``0 ..
    groups - 1``: none), ``prefix_pages`` (int32 ``[groups]``, ``MAX_GROUPS`` at most) how many of their
    first page table entries a group's sequences have in common; the entries of
    its lowest sequence are read.  Both are read on the GPU.  The result is
    :func:`int4_attention`'s within roundings, for any lengths: shared Keys, Values
    and softmax weights enter their products as fp16 numbers (a score is off by up
    to 2^-11 of ``scaling * sum |q k|``), Keys and weights of an fp16 result as the
    sums of two (error against 64 bits, of the result's size: bf16 0.0017, as its own
    rounding; fp16 0.00028, 0.0002 its own).  Where few
    sequences share few pages, each reads them itself, which is faster then
    (``always``: never).  No gradient is recorded: a query that requires one, or
    has a forward-mode tangent, raises ``NotImplementedError``."""
    return _lib.int4_binding().attend_prefix(query, pages, page_table, lengths, scaling, prefix_group, prefix_pages, counts, out,
                                             status, always)


class Int4KVCache:
    """4-bit cache of ``batch`` sequences for ``n_layers`` layers: a pool of
    ``n_pages`` 64-token pages per layer, shared by the sequences through one
    page table (a sequence's token positions are the same in every layer).

    A step is ``extend(counts)``, then for every layer ``write(layer, key,
    value)`` and ``attend(layer, query, scaling)``: ``extend`` makes room for
    the step's tokens, ``write`` stores them behind the tokens of the steps
    before, ``attend`` sees both.  Pages come from a free list and go back with
    ``release``.  ``rotate`` turns a step's queries and Keys to their positions;
    ``share`` gives a sequence's complete pages to others that begin as it does,
    and ``attend_shared`` reads such pages once for all of them.

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
        self._refs = np.zeros(n_pages, np.int64)                  # sequences that hold each page
        self._common = np.zeros(batch, np.int64)                  # first pages of each that others hold too
        self.prefix_pages = torch.zeros(min(batch, MAX_GROUPS), dtype=torch.int32, device=self.device)   # for int4_prefix_attention
        self.prefix_group = torch.from_numpy(self._numbered(np.arange(batch))[0].astype(np.int32)).to(self.device)

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
                self._table[b, j] = page = self._free.pop()
                self._refs[page] = 1
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
        cut = np.flatnonzero(n // PAGE_TOKENS < self._common)   # what comes next would be written over these
        if len(cut):
            raise ValueError(f"sequence {cut[0]} shares pages past token {int(n[cut[0]])}")
        self._start, self._end, self._step = n.copy(), n.copy(), 0
        self._upload(self._spans, np.stack([self._start, self._end, np.zeros_like(n)]))

    def release(self, seqs=None) -> None:
        """Empty the sequences ``seqs`` (default: all) and return the pages that no
        other sequence shares."""
        every = range(self.batch)
        for b in every if seqs is None else [every[s] for s in seqs]:   # all are looked up before the first is emptied
            for j in range(int(self._owned[b]) - 1, -1, -1):
                page = int(self._table[b, j])
                self._refs[page] -= 1
                if self._refs[page] == 0:
                    self._free.append(page)
            self._table[b, :] = -1
            self._owned[b] = self._start[b] = self._end[b] = 0
        self._step = int((self._end - self._start).max())
        self._upload(self.page_table, self._table)
        self._upload(self._spans, np.stack([self._start, self._end, self._end - self._start]))
        self._regroup()

    def share(self, source: int, seqs, tokens: int | None = None) -> int:
        """Let the empty sequences ``seqs`` begin with the first ``tokens`` tokens of
        ``source`` (default: all it has), in whole pages: they hold the same pages,
        which are written no more.  Returns the tokens that are shared; the others
        go on behind them.  The pages' tokens must have been written, or be written
        on this stream before they are read."""
        every = range(self.batch)
        source, seqs = every[source], [every[s] for s in seqs]
        if len(set(seqs)) < len(seqs) or source in seqs:
            raise ValueError("a sequence is named twice")
        if any(self._owned[b] or self._end[b] for b in seqs):
            raise ValueError("sequences that begin with shared pages must be empty (release them first)")
        have = int(self._end[source])
        tokens = have if tokens is None else int(tokens)
        if tokens < 0 or tokens > have:
            raise ValueError(f"sequence {source} has {have} tokens, {tokens} were to be shared")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("share the pages before the capture")
        n = tokens // PAGE_TOKENS
        for b in seqs:
            self._table[b, :n] = self._table[source, :n]
            self._refs[self._table[source, :n]] += 1
            self._owned[b] = n
            self._start[b] = self._end[b] = n * PAGE_TOKENS
        self._upload(self.page_table, self._table)
        self._upload(self._spans, np.stack([self._start, self._end, self._end - self._start]))
        self._regroup()
        return n * PAGE_TOKENS

    def _regroup(self) -> None:
        """Sequences that begin with the same page are one group, named by its lowest;
        the pages that all of it have in common are read once."""
        first = self._table[:, 0]
        rows = np.flatnonzero((first >= 0) & (self._refs[first] > 1))
        if not len(rows) and not self._common.any():
            return   # as before: no sequence shares anything
        group, pages = np.arange(self.batch), np.zeros(self.batch, np.int64)
        self._common[:] = 0
        if len(rows):
            _, leader, which = np.unique(first[rows], return_index=True, return_inverse=True)
            leader = rows[leader[which]]   # each row's group: its lowest sequence
            table = self._table[:, :int(self._owned[rows].max())]
            held = table[rows] >= 0

            def leading(yes):   # how many of a row's first entries are so
                return np.where(yes.all(1), yes.shape[1], np.argmin(yes, 1))

            self._common[rows] = leading(held & (self._refs[table[rows]] > 1))
            group[rows] = leader
            pages[leader] = self.width
            np.minimum.at(pages, leader, leading(held & (table[rows] == table[leader])))
        group, names = self._numbered(group)
        self._upload(self.prefix_group, group)
        self._upload(self.prefix_pages, pages[names])

    def _numbered(self, group: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        """(each sequence's group as a call takes it, the lowest sequence of each group).
        Groups that go by their lowest sequence's number as long as there are numbers for
        all; else groups of several come first, and what is past the last number is in none
        (its sequences read their pages themselves)."""
        if self.batch <= MAX_GROUPS:
            return group, np.arange(self.batch)
        size = np.bincount(group, minlength=self.batch)
        names = np.argsort(-np.minimum(size, 2), kind="stable")[:MAX_GROUPS]   # (sequences that lead no group: size 0, last)
        number = np.full(self.batch, -1)
        number[names] = np.arange(len(names))
        return number[group], names

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

    def rotate(self, query: torch.Tensor, key: torch.Tensor | None, freqs: torch.Tensor, magnitude: float = 1.0,
               interleaved: bool = False, out: tuple | None = None):
        """:func:`logitfill_b200.prompt.rotary_embed` of this step's queries and Keys, ``[batch,
        heads, T, head_dim]``, to their positions in the sequences (read on the GPU)."""
        return rotary_embed(query, key, freqs, start=self.start, magnitude=magnitude, interleaved=interleaved, out=out)

    def attend_shared(self, layer: int, query: torch.Tensor, scaling: float, out: torch.Tensor | None = None) -> torch.Tensor:
        """:meth:`attend` by way of :func:`int4_prefix_attention`: pages that sequences
        share are read once for all of them.  (For a chunk of a prompt, many query
        tokens of one sequence, its own pages are read once for all of those.)"""
        self._check_query(query)
        return int4_prefix_attention(query, self.pages[layer], self.page_table, self.end, scaling, self.prefix_group,
                                     self.prefix_pages, self.counts, out, self.status)

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
            with torch.inference_mode():   # (the word may have been made in it)
                self.status.zero_()
            _lib.check(code, "4-bit cache kernel")


__all__ = ["PAGE_TOKENS", "GROUP", "MAX_GROUPS", "record_words", "bounds_bytes", "alloc_pages", "alloc_bounds", "int4_write",
           "int4_read", "int4_read_bounds", "int4_attention", "int4_select", "int4_sparse_attention", "int4_prefix_attention", "Int4KVCache"]
