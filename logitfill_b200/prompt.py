"""A prompt's way into the cache: rotary positions of its queries and Keys, and
its attention over its own tokens.

:func:`rotary_embed` turns the queries and Keys of a step to their positions,
next to the caches' own attention: what :func:`logitfill_b200.int4.int4_write`
or a layer's ``commit`` stores are turned Keys.  :func:`rotary_frequencies`
makes the table it reads.  :func:`prompt_attention` is the causal attention of
whole prompts in their original type, which both caches leave to their caller
(:mod:`logitfill_b200.adapter` can run it).

Tensors are ``[batch, heads, tokens, head_dim]``, or packed ``[tokens, heads,
head_dim]``: the tokens of all sequences behind one another.  Every launch goes
to the current stream.  There is no CPU or dense fallback and no backward pass
(a tensor that requires a gradient, or has a forward-mode tangent, is refused); what the
kernels do not implement raises ``NotImplementedError``, malformed arguments ``ValueError``.
"""
from __future__ import annotations

import math

import torch

from logitfill_b200 import _lib


def rotary_frequencies(part: int, base: float = 10000.0, scaling: dict | None = None, device="cuda"):
    """``(freqs, magnitude)`` for :func:`rotary_embed`: int64 ``[part / 2]``, the
    turns per position of pair ``i`` in units of 2^-64 turn, of ``base ** (-2 i /
    part)`` radians, and the factor on the rotated channels.

    ``scaling`` is a model configuration's dictionary (``rope_type`` or
    ``type``): ``"default"``; ``"linear"``, all frequencies divided by
    ``factor``; ``"yarn"`` (Peng et al., arXiv:2309.00071), where pairs that turn
    more than ``beta_fast`` (32) times over ``original_max_position_embeddings``
    positions keep their frequency, those that turn less than ``beta_slow`` (1)
    times are divided by ``factor``, and between them the two are mixed in
    proportion to the pair's number; the magnitude is ``attention_factor``, or
    ``0.1 ln(factor) + 1``."""
    part = int(part)
    if part < 2 or part % 2:
        raise ValueError(f"the rotated channels are an even number from 2 on, got {part}")
    if not (math.isfinite(base) and base > 0):
        raise ValueError(f"base must be a positive number, got {base}")
    n, magnitude = part // 2, 1.0
    turns = [base ** (-2.0 * i / part) / (2.0 * math.pi) for i in range(n)]
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in ("default", "linear", "yarn"):
        raise NotImplementedError(f"rotary scaling {kind!r} is not implemented (default, linear, yarn)")
    if kind != "default":
        factor = float(scaling["factor"])
        if not (math.isfinite(factor) and factor >= 1.0):
            raise ValueError(f"factor must be 1 or more, got {factor}")
        keep = [0.0] * n   # how much of a pair's own frequency stays
        if kind == "yarn":
            unknown = [k for k in ("mscale", "mscale_all_dim") if scaling.get(k) is not None] + (
                ["truncate"] if scaling.get("truncate", True) is not True else [])
            if unknown:
                raise NotImplementedError(f"rotary scaling with {', '.join(unknown)} is not implemented")
            if base <= 1.0:
                raise ValueError(f"yarn scaling needs a base above 1, got {base}")
            original = float(scaling["original_max_position_embeddings"])
            fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)
            if not (original > 0 and fast > 0 and slow > 0):
                raise ValueError(f"yarn scaling of {original} positions between {fast} and {slow} turns")

            def pair_of(times):   # the pair, counted in fractions, that turns `times` times over the original positions
                return part * math.log(original / (times * 2.0 * math.pi)) / (2.0 * math.log(base))

            low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), part - 1)
            keep = [1.0 - min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(n)]
            given = scaling.get("attention_factor")
            magnitude = 0.1 * math.log(factor) + 1.0 if given is None else float(given)
        turns = [t * k + t / factor * (1.0 - k) for t, k in zip(turns, keep)]
    whole = [int(round(t * 2.0 ** 64)) % (1 << 64) for t in turns]
    return torch.tensor([w - (1 << 64) if w >= 1 << 63 else w for w in whole], dtype=torch.int64, device=device), magnitude


def rotary_embed(query: torch.Tensor, key: torch.Tensor | None, freqs: torch.Tensor, positions: torch.Tensor | None = None,
                 start: torch.Tensor | None = None, magnitude: float = 1.0, interleaved: bool = False,
                 transposed: bool = False, out: tuple | None = None):
    """``query`` and ``key`` (which may be None) turned to their positions:
    ``(query, key)`` of the same shapes, types (fp32, fp16 or bf16) and strides.

    The first ``2 * len(freqs)`` channels of a head are rotated, the others
    copied.  Pair ``i`` of them, channels ``i`` and ``i + len(freqs)`` (or ``2 i``
    and ``2 i + 1`` with ``interleaved``), turns by ``freqs[i]`` a position and is
    multiplied by ``magnitude``.  The angle is exact for any position (64-bit
    whole numbers modulo one turn); the rotation is fp32, rounded once.

    ``positions``: int32 or int64, ``[batch, tokens]`` or packed ``[tokens]``;
    or ``start``: int32 ``[batch]``, token ``t`` of sequence ``b`` being at
    ``start[b] + t`` (the cache's ``start``).  ``transposed`` turns the other way,
    which takes the rotation back (with ``1 / magnitude``) and is how a gradient
    goes back through it.  ``out``: ``(query, key)`` tensors to write, which may
    be the inputs themselves (in place) but must not overlap them otherwise."""
    return _lib.prompt_binding().rotary(query, key, freqs, positions, start, magnitude, interleaved, transposed, out)


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scaling: float,
                     starts: torch.Tensor | None = None, counts: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of whole prompts over their own tokens: token ``i`` of a sequence
    sees its tokens ``0 .. i``.  fp16 or bf16, ``head_dim`` 64 or 128, query head
    ``j`` reading KV head ``j // (n_q // n_kv)`` (128 query heads to a KV head at
    most); the result has the query's shape and type.

    Packed, ``query`` ``[tokens, n_q, head_dim]`` and ``key``, ``value`` ``[tokens,
    n_kv, head_dim]``: sequence ``b`` is rows ``starts[b] .. starts[b + 1] - 1``
    (int32 ``[batch + 1]`` on the GPU; None: one sequence); sequences do not share
    rows, and rows of no sequence are left as they were in ``out`` (undefined in a
    new result).  Padded, ``[batch, heads, tokens, head_dim]``: sequence ``b`` has its
    first ``counts[b]`` tokens (int32 ``[batch]``; None: all), and the rows behind
    them become 0.  What lies in rows that a token does not see does not matter, NaN
    and infinities included.  ``out`` may not share memory with an input.

    Scores and sums are fp32; a softmax weight is rounded to the Value's type for its
    product (error against 64 bits, of the result's size: bf16 0.0021, fp16 0.00026, the
    results' own rounding being 0.0016 and 0.0002).  The sums are taken before the
    division, with weights up to 2^8: bf16 Values past some 2^119 / ``tokens`` may overflow.
    ``status`` (int32 ``[1]`` on the GPU): a wait of the kernel that gives up sets it to a
    non-zero ``lf_status``."""
    return _lib.prompt_binding().attend(query, key, value, scaling, starts, counts, out, status)


__all__ = ["rotary_frequencies", "rotary_embed", "prompt_attention"]
