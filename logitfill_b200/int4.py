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
``[batch]``, all on the GPU.  A page table entry outside the pool is never
followed; with ``status`` (int32 ``[1]`` on the GPU) given, such an access sets
it to a non-zero ``lf_status``.  Every launch goes to the current stream.
There is no CPU or dense fallback; what the kernels do not implement raises
``NotImplementedError``, malformed arguments ``ValueError``.
"""
from __future__ import annotations

import numpy as np
import torch

from logitfill_b200 import _lib

PAGE_TOKENS = 64   # tokens of a page
GROUP = 32         # channels that share a scale and a minimum
_CODE = {torch.float32: _lib.LF_F32, torch.float16: _lib.LF_F16, torch.bfloat16: _lib.LF_BF16}


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


def _pool(pages: torch.Tensor, page_table: torch.Tensor):
    """The C ABI's pool of ``pages`` and ``page_table`` as a tuple (batch and
    KV heads last), the head_dim and the device."""
    shape, strides = pages.shape, pages.stride()
    if len(shape) != 3 or pages.dtype != torch.int32 or strides[2] != 1:
        raise ValueError(f"pages must be int32 [n_pages, n_kv, words] with word stride 1, got {pages.dtype} {tuple(shape)}")
    table_shape, table_strides = page_table.shape, page_table.stride()
    if len(table_shape) != 2 or page_table.dtype != torch.int32 or table_strides[1] != 1:
        raise ValueError(f"page_table must be int32 [batch, width] with entry stride 1, got {page_table.dtype} "
                         f"{tuple(table_shape)}")
    device = pages.device
    if device.type != "cuda":
        raise RuntimeError("the 4-bit cache needs CUDA tensors (there is no CPU path)")
    if page_table.device != device:
        raise RuntimeError(f"page_table is on {page_table.device}, pages on {device}")
    n, H, words = shape
    B, W = table_shape
    if words % 20:
        raise ValueError(f"a record of {words} words belongs to no head_dim (20 * head_dim words)")
    return (pages.data_ptr(), page_table.data_ptr(), strides[0] if n > 1 else H * words, strides[1] if H > 1 else words,
            table_strides[0] if B > 1 else W, W, n, H, B), words // 20, device


def _per_sequence(name: str, t: torch.Tensor | None, batch: int, device) -> int:
    """Address of an int32 [batch] tensor (0 for None)."""
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.shape != (batch,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 [{batch}] tensor on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _status(t: torch.Tensor | None, device) -> int:
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.numel() < 1 or t.device != device:
        raise ValueError(f"status must be an int32 tensor on {device}")
    return t.data_ptr()


def _bounds(bounds: torch.Tensor, pages: torch.Tensor, head_dim: int):
    n, H = pages.shape[0], pages.shape[1]
    if (bounds.dtype != torch.int8 or bounds.dim() != 3 or bounds.shape[0] != n or bounds.shape[1] != H
            or bounds.shape[2] != 2 * head_dim + 16 or bounds.stride(2) != 1 or bounds.device != pages.device):
        raise ValueError(f"bounds must be int8 [{n}, {H}, {bounds_bytes(head_dim)}] on {pages.device}, got {bounds.dtype} "
                         f"{tuple(bounds.shape)} on {bounds.device}")
    return bounds.data_ptr(), bounds.stride(0) if n > 1 else H * bounds.shape[2], \
        bounds.stride(1) if H > 1 else bounds.shape[2]


def _aligned_rows(t: torch.Tensor):
    """``t`` [B, H, T, D] with 16-byte aligned rows of channel stride 1 (a copy
    where it is not), and its first three strides (0 where the extent is 1)."""
    (s0, s1, s2, s3), (n0, n1, n2, _) = t.stride(), t.shape
    s0, s1, s2 = s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0
    if s3 != 1 or t.data_ptr() % 16 or (s0 | s1 | s2) * t.element_size() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, s2, _ = t.stride()
    return t, s0, s1, s2


def _stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _launch(entry: str, device, *args) -> None:
    """Call ``entry`` of the library with ``args`` and the current stream of ``device``."""
    fn = _entries.get(entry)
    if fn is None:
        fn = _entries[entry] = getattr(_lib.lib(), entry)
    index = device.index
    if torch._C._cuda_getDevice() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _lib.check(status, entry)


_entries: dict = {}


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
    pool, D, dev = _pool(pages, page_table)
    H, B = pool[-2:]
    if key.dim() != 4 or key.shape != value.shape or (key.shape[0], key.shape[1], key.shape[3]) != (B, H, D):
        raise ValueError(f"key and value must be [{B}, {H}, T, {D}], got {tuple(key.shape)} and {tuple(value.shape)}")
    if key.dtype != value.dtype:
        raise ValueError(f"key is {key.dtype}, value {value.dtype}")
    if key.device != dev or value.device != dev:
        raise RuntimeError(f"key and value must be on {dev}")
    code = _lib.dtype_code(key.dtype)
    key, *ks = _aligned_rows(key)
    value, *vs = _aligned_rows(value)
    args = _lib.INT4_TOKENS.pack(
        *pool, key.data_ptr(), value.data_ptr(), *ks, *vs, _per_sequence("start", start, B, dev),
        _per_sequence("counts", counts, B, dev), *((0, 0, 0) if bounds is None else _bounds(bounds, pages, D)),
        _status(status, dev), D, code, key.shape[2])
    _launch("lf_int4_write", dev, args)


def int4_read(pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor, tokens: int,
              counts: torch.Tensor | None = None, dtype=torch.float32, status: torch.Tensor | None = None):
    """Positions ``start[b] .. start[b] + tokens - 1`` of every sequence as Key and
    Value ``[batch, n_kv, tokens, head_dim]`` in ``dtype`` (fp32, fp16 or
    bf16); tokens ``i >= counts[b]`` are zeros."""
    pool, D, dev = _pool(pages, page_table)
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"cannot read {tokens} tokens")
    code = _lib.dtype_code(dtype)
    H, B = pool[-2:]
    key = torch.empty((B, H, tokens, D), dtype=dtype, device=dev)
    value = torch.empty_like(key)
    strides = H * tokens * D, tokens * D, D
    args = _lib.INT4_TOKENS.pack(
        *pool, key.data_ptr(), value.data_ptr(), *strides, *strides, _per_sequence("start", start, B, dev),
        _per_sequence("counts", counts, B, dev), 0, 0, 0, _status(status, dev), D, code, tokens)
    _launch("lf_int4_read", dev, args)
    return key, value


def int4_read_bounds(bounds: torch.Tensor) -> torch.Tensor:
    """fp32 ``[n_pages, n_kv, 2, head_dim]`` of the bounds records: every Key
    channel's upper, then its lower bound over a page's tokens."""
    if bounds.dim() != 3 or bounds.dtype != torch.int8 or bounds.stride(2) != 1 or bounds.shape[2] % 2:
        raise ValueError(f"bounds must be int8 [n_pages, n_kv, 2 * head_dim + 16], got {bounds.dtype} {tuple(bounds.shape)}")
    if not bounds.is_cuda:
        raise RuntimeError("the 4-bit cache needs CUDA tensors (there is no CPU path)")
    n, H, width = bounds.shape
    D = (width - 16) // 2
    out = torch.empty(n, H, 2, D, dtype=torch.float32, device=bounds.device)
    _launch("lf_int4_read_bounds", bounds.device, bounds.data_ptr(), bounds.stride(0) if n > 1 else H * width,
            bounds.stride(1) if H > 1 else width, n, H, D, out.data_ptr())
    return out


_workspaces: dict = {}


def _workspace(pool, n_q: int, q_len: int, head_dim: int, device):
    """Scratch of an attention call, its address and bytes: partial results,
    then tickets that are zero between calls.  Calls on one stream share one
    buffer (they run in order); a call being captured in a CUDA graph gets its
    own, which the graph keeps and clears, so replays on any stream do not
    meet."""
    H, B = pool[-2:]
    key = (device.index, _stream(device))
    # a ticket for each column tile of 16 at most, of each query token and KV head
    units = B * H * q_len * (n_q // H + 15)
    held = _workspaces.get(key)
    capturing = torch.cuda.is_current_stream_capturing()
    if held is not None and held[1] >= units and not capturing:
        return held[0], held[2], held[3]
    so = _lib.lib()
    with torch.cuda.device(device):
        need, clear_from = so.lf_int4_workspace_bytes(B, H, n_q, q_len, head_dim), so.lf_int4_workspace_clear_from()
    if capturing:
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[clear_from:].zero_()
        return ws, ws.data_ptr(), need
    units = max(units, 1 << 16)
    need = max(need, clear_from + 4 * units)
    ws = torch.zeros(need, dtype=torch.uint8, device=device)
    _workspaces[key] = ws, units, ws.data_ptr(), need
    return ws, ws.data_ptr(), need


def _query(query: torch.Tensor, pool, head_dim: int, device):
    """The query, checked, as [B, n_q, q_len, D] with 16-byte aligned rows of
    channel stride 1, and its first three strides."""
    q = query if query.dim() == 4 else query.unsqueeze(2)
    H, batch = pool[-2:]
    if q.dim() != 4:
        raise ValueError(f"query must be [batch, n_q, head_dim] or [batch, n_q, q_len, head_dim], got {tuple(query.shape)}")
    B, n_q, q_len, D = q.shape
    if B != batch or D != head_dim or n_q < 1 or q_len < 1:
        raise ValueError(f"query must be [{batch}, n_q, {head_dim}] or [{batch}, n_q, q_len, {head_dim}], got "
                         f"{tuple(query.shape)}")
    if n_q % H:
        raise ValueError(f"{n_q} query heads do not divide into {H} KV heads")
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        raise NotImplementedError(f"the 4-bit cache's attention takes fp16 or bf16 queries, got {q.dtype}")
    if q.device != device:
        raise RuntimeError(f"query is on {q.device}, pages on {device}")
    return _aligned_rows(q)


def _budget(top_pages: int, sink_pages: int, recent_pages: int):
    top, sink, recent = int(top_pages), int(sink_pages), int(recent_pages)
    if top < 0 or sink < 0 or recent < 1:
        raise ValueError(f"top {top} and sink {sink} must not be negative, recent {recent} at least 1")
    return top + sink + recent, sink, recent


def _attend(entry: str, query, pages, page_table, lengths, scaling, counts, out, status, bounds=None, budget=(0, 0, 0)):
    """The dense (``lf_int4_attend``), the sparse (``lf_int4_attend_sparse``) or
    only the page choice's (``lf_int4_select``) call: ``(out, picked)``."""
    pool, D, dev = _pool(pages, page_table)
    q, s0, s1, s2 = _query(query, pool, D, dev)
    H, B = pool[-2:]
    n_q, q_len = q.shape[1], q.shape[2]
    if entry == "lf_int4_select":
        out_args = workspace = (0, 0, 0, 0)
    else:
        if out is None:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
        elif out.shape != query.shape or out.dtype != query.dtype or out.device != dev or out.stride(-1) != 1:
            raise ValueError(f"out must be {query.dtype} {tuple(query.shape)} on {dev} with channel stride 1")
        o = out.stride()
        out_args = out.data_ptr(), o[0], o[1], o[2] if len(o) == 4 else 0
        workspace = _workspace(pool, n_q, q_len, D, dev)
    picked, picked_at, bounds_args = None, 0, (0, 0, 0)
    if bounds is not None:
        bounds_args = _bounds(bounds, pages, D)
        picked = torch.empty((B, q_len, H, budget[0]), dtype=torch.int32, device=dev)
        picked_at = picked.data_ptr()
    args = _lib.INT4_QUERY.pack(
        *pool, q.data_ptr(), s0, s1, s2, *out_args, _per_sequence("lengths", lengths, B, dev),
        0 if counts is None else _per_sequence("counts", counts, B, dev), *bounds_args, picked_at, workspace[1],
        workspace[2], 0 if status is None else _status(status, dev),
        scaling, D, _CODE[q.dtype], n_q, q_len, *budget)
    _launch(entry, dev, args)
    return out, picked


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
    return _attend("lf_int4_attend", query, pages, page_table, lengths, scaling, counts, out, status)[0]


def int4_select(query: torch.Tensor, pages: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor,
                lengths: torch.Tensor, top_pages: int, sink_pages: int = 1, recent_pages: int = 2,
                counts: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """The logical pages each query token and KV head reads in a sparse call:
    int32 ``[batch, q_len, n_kv, sink + recent + top]``, ascending, -1 after the
    last.  The first ``sink_pages`` and the last ``recent_pages`` (at least 1:
    the page being filled) are always in; of the rest the ``top_pages`` with
    the largest bound on the scores of the KV head's queries (summed over its
    query heads; ties to the lower page)."""
    return _attend("lf_int4_select", query, pages, page_table, lengths, 0.0, counts, None, status, bounds,
                   _budget(top_pages, sink_pages, recent_pages))[1]


def int4_sparse_attention(query: torch.Tensor, pages: torch.Tensor, bounds: torch.Tensor, page_table: torch.Tensor,
                          lengths: torch.Tensor, scaling: float, top_pages: int, sink_pages: int = 1,
                          recent_pages: int = 2, counts: torch.Tensor | None = None, out: torch.Tensor | None = None,
                          status: torch.Tensor | None = None):
    """:func:`int4_select`, then :func:`int4_attention` over the picked pages
    only: ``(out, picked)``.  With ``sink + recent + top`` pages or fewer
    visible, every page is read and the result is the dense one."""
    return _attend("lf_int4_attend_sparse", query, pages, page_table, lengths, scaling, counts, out, status, bounds,
                   _budget(top_pages, sink_pages, recent_pages))


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
        self._start, self._end = n.copy(), n.copy()
        self._upload(self._spans, np.stack([self._start, self._end, np.zeros_like(n)]))

    def release(self, seqs=None) -> None:
        """Empty the sequences ``seqs`` (default: all) and return their pages."""
        for b in range(self.batch) if seqs is None else seqs:
            for j in range(int(self._owned[b]) - 1, -1, -1):
                self._free.append(int(self._table[b, j]))
            self._table[b, :] = -1
            self._owned[b] = self._start[b] = self._end[b] = 0
        self._upload(self.page_table, self._table)
        self._upload(self._spans, np.stack([self._start, self._end, self._end - self._start]))

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Store this step's tokens of one layer: ``[batch, n_kv, T, head_dim]``,
        the first ``counts[b]`` of sequence ``b``."""
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
        ``counts[b]`` of sequence ``b``)."""
        self._check_heads(query)
        return int4_attention(query, self.pages[layer], self.page_table, self.end, scaling, self.counts, out, self.status)

    def attend_sparse(self, layer: int, query: torch.Tensor, scaling: float, top_pages: int, sink_pages: int = 1,
                      recent_pages: int = 2, out: torch.Tensor | None = None):
        """:func:`int4_sparse_attention` of this step's query tokens."""
        self._check_heads(query)
        if self.bounds is None:
            raise RuntimeError("a sparse call needs a cache made with bounds=True")
        return int4_sparse_attention(query, self.pages[layer], self.bounds[layer], self.page_table, self.end, scaling,
                                     top_pages, sink_pages, recent_pages, self.counts, out, self.status)

    def _check_heads(self, query: torch.Tensor) -> None:
        if query.dim() < 3 or query.shape[1] != self.n_q:
            raise ValueError(f"query must have {self.n_q} heads, got {tuple(query.shape)}")

    def check_status(self) -> None:
        """Raise if a kernel met a position outside its sequence's pages (synchronises)."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            _lib.check(code, "4-bit cache kernel")


__all__ = ["PAGE_TOKENS", "GROUP", "record_words", "bounds_bytes", "alloc_pages", "alloc_bounds", "int4_write",
           "int4_read", "int4_read_bounds", "int4_attention", "int4_select", "int4_sparse_attention", "Int4KVCache"]
