"""Serve a batch of prompts from the 4-bit paged cache.

A small decoder-only model with grouped heads and rotary positions (random
weights: no checkpoint is needed) takes prompts of different lengths, writes
their Key and Value into an :class:`logitfill_b200.Int4KVCache` and decodes
greedily, attending over every page or (``--top``) over the pages that the
bound selects.  The same tokens go through the model with the uncompressed
Key and Value beside it, and the run reports how far the logits are apart and
what the cache holds.

    python examples/int4_decode.py                       # 4 prompts, dense
    python examples/int4_decode.py --prompt 6000 --top 24
    python examples/int4_decode.py --draft 4             # verify drafts of 4 tokens per step
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from logitfill_b200 import Int4KVCache  # noqa: E402


class Decoder:
    """Random-weight decoder: RMS norm, rotary grouped-query attention, SiLU MLP."""

    def __init__(self, layers=2, hidden=512, n_q=8, n_kv=2, head_dim=64, vocab=1000, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, generator=g, device=device) * shape[-1] ** -0.5).to(torch.bfloat16)

        self.n_q, self.n_kv, self.head_dim, self.device = n_q, n_kv, head_dim, torch.device(device)
        self.embed, self.head = weight(vocab, hidden) * hidden ** 0.5, weight(vocab, hidden)
        self.blocks = [dict(q=weight(n_q * head_dim, hidden), k=weight(n_kv * head_dim, hidden),
                            v=weight(n_kv * head_dim, hidden), o=weight(hidden, n_q * head_dim),
                            up=weight(2 * hidden, hidden), gate=weight(2 * hidden, hidden), down=weight(hidden, 2 * hidden))
                       for _ in range(layers)]
        self.inv_freq = 10000.0 ** (-torch.arange(0, head_dim, 2, device=device) / head_dim)

    def _rotate(self, x, positions):
        """Rotary embedding of ``[B, heads, T, D]`` at ``positions`` ``[B, T]``."""
        angle = positions[:, None, :, None].float() * self.inv_freq
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1).to(x.dtype)

    def forward(self, tokens, positions, attend):
        """Logits ``[B, T, vocab]``; ``attend(layer, q, k, v)`` does the attention
        of ``[B, heads, T, D]`` states."""
        B, T = tokens.shape
        x = self.embed[tokens]
        for layer, w in enumerate(self.blocks):
            y = F.rms_norm(x, x.shape[-1:])
            q, k, v = ((y @ w[n].T).view(B, T, -1, self.head_dim).transpose(1, 2) for n in "qkv")
            out = attend(layer, self._rotate(q, positions), self._rotate(k, positions), v)
            x = x + out.transpose(1, 2).reshape(B, T, -1) @ w["o"].T
            y = F.rms_norm(x, x.shape[-1:])
            x = x + (F.silu(y @ w["gate"].T) * (y @ w["up"].T)) @ w["down"].T
        return F.rms_norm(x, x.shape[-1:]) @ self.head.T


def dense_attention(q, k, v, scaling, lengths, counts):
    """Reference attention over uncompressed ``k``/``v`` ``[B, n_kv, S, D]``."""
    group = q.shape[1] // k.shape[1]
    k, v = (x.float().repeat_interleave(group, 1) for x in (k, v))
    i = torch.arange(q.shape[2], device=q.device)
    seen = (lengths - counts).view(-1, 1) + 1 + i                                    # [B, T]
    mask = torch.arange(k.shape[2], device=q.device) < seen[:, None, :, None]
    p = (q.float() @ k.transpose(-1, -2) * scaling).masked_fill(~mask, -1e30).softmax(-1)
    return (p @ v).to(q.dtype)


def serve(prompts, steps=32, draft=1, top=None, layers=2, n_q=8, n_kv=2, head_dim=64, seed=0):
    """Prefill ``prompts`` (a list of lengths), then ``steps`` steps of ``draft``
    tokens each.  Returns the root mean square of the logits' differences from the
    uncompressed run over that of the logits, the share of equal greedy tokens
    and the cache."""
    model = Decoder(layers, n_q=n_q, n_kv=n_kv, head_dim=head_dim, seed=seed)
    B, scaling = len(prompts), head_dim ** -0.5
    longest = max(prompts) + steps * draft
    cache = Int4KVCache(layers, B, n_q, n_kv, head_dim, n_pages=sum(-(-(n + steps * draft) // 64) for n in prompts),
                        max_tokens=longest)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    tokens = torch.randint(0, model.embed.shape[0], (B, max(prompts)), generator=g, device="cuda")
    full = [torch.zeros(2, B, n_kv, longest, head_dim, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]
    length = torch.zeros(B, dtype=torch.long, device="cuda")

    def step(tokens, counts):
        nonlocal length
        n = torch.tensor(counts, device="cuda")
        T = tokens.shape[1]
        prefill = not int(length.max())
        positions = length.view(-1, 1) + torch.arange(T, device="cuda")
        rows = torch.arange(B, device="cuda").view(-1, 1).expand(B, T)
        live = torch.arange(T, device="cuda") < n.view(-1, 1)

        def uncompressed(layer, q, k, v):
            for x, kept in ((k, full[layer][0]), (v, full[layer][1])):
                kept[rows[live], :, positions[live]] = x.transpose(1, 2)[live]
            return dense_attention(q, full[layer][0], full[layer][1], scaling, length + n, n)

        def cached(layer, q, k, v):
            cache.write(layer, k, v)
            if prefill:   # the prompt itself attends in the original type, as the tiered cache's does
                return dense_attention(q, k, v, scaling, n, n)
            if top is None:
                return cache.attend(layer, q, scaling)
            return cache.attend_sparse(layer, q, scaling, top_pages=top)[0]

        cache.extend(counts if len(set(counts)) > 1 else counts[0])
        want, got = model.forward(tokens, positions, uncompressed), model.forward(tokens, positions, cached)
        length = length + n
        return want[live].float(), got[live].float(), got

    apart, size, same = 0.0, 0.0, []
    counts = list(prompts)
    for s in range(steps + 1):
        want, got, logits = step(tokens, counts)
        if s:
            apart += float((want - got).square().sum())
            size += float(want.square().sum())
            same.append((want.argmax(-1) == got.argmax(-1)).float().mean())
        last = torch.tensor([c - 1 for c in counts], device="cuda")
        nxt = logits[torch.arange(B, device="cuda"), last].argmax(-1)
        # the next step's draft: the chosen token, then guesses
        guesses = torch.randint(0, logits.shape[-1], (B, draft - 1), generator=g, device="cuda")
        tokens, counts = torch.cat([nxt.view(-1, 1), guesses], 1), [draft] * B
    cache.check_status()
    return (apart / size) ** 0.5 if size else 0.0, float(torch.stack(same).mean()) if same else 1.0, cache


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompt", type=int, default=900, help="tokens of the longest prompt")
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--draft", type=int, default=1, help="tokens per step")
    ap.add_argument("--top", type=int, default=None, help="selected pages per KV head (default: all pages)")
    a = ap.parse_args()
    prompts = [max(1, a.prompt - 137 * b) for b in range(a.batch)]
    apart, same, cache = serve(prompts, a.steps, a.draft, a.top)
    held = sum(cache.lengths) * cache.n_layers * cache.n_kv * cache.head_dim * 2
    used = (cache.n_pages - cache.free_pages) * cache.n_layers * cache.n_kv * 20 * cache.head_dim * 4
    print(f"prompts {prompts}, {a.steps} steps of {a.draft}: logits {100 * apart:.1f} % apart, {100 * same:.1f} % equal greedy tokens; "
          f"cache {used / 2 ** 20:.1f} MiB for {held * 2 / 2 ** 20:.1f} MiB of bf16 Key and Value")


if __name__ == "__main__":
    main()
