"""A prompt's operators and the cache's in a run, as a server uses them: a shared system
prompt and each sequence's own, rotary positions, prompt attention, the 4-bit cache
with shared pages, decoding; against the formulas in 64 bits over the values that the
cache holds (read back), step by step on the same inputs."""
from __future__ import annotations

import math

import pytest
import torch

from logitfill_b200 import Int4KVCache, prompt_attention, rotary_frequencies
from logitfill_b200.adapter import DeepSeekQwenKVAdapter
from logitfill_b200.synthetic import synthetic_levels
from tests.qwen_cases import tiny_qwen2

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
U = 2.0 ** -8


def _turned(x, at, freqs, magnitude):
    """[B, heads, T, D] in 64 bits at positions [B][T]."""
    n = freqs.numel()
    whole = freqs.tolist()
    phase = torch.tensor([[[(p * f) % (1 << 64) / 2.0 ** 64 for f in whole] for p in row] for row in at], dtype=torch.float64).cuda()
    c, s = ((2 * math.pi * phase).cos() * magnitude).unsqueeze(1), ((2 * math.pi * phase).sin() * magnitude).unsqueeze(1)
    a, b = x[..., :n].double(), x[..., n:2 * n].double()
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * n:].double()], -1)


def _attended(q, k, v, scaling, sees):
    """(out, bound) of q [n_q, T, D] over k, v [n_kv, S, D]; query i sees the first sees[i]."""
    group = q.shape[0] // k.shape[0]
    k, v = (x.double().repeat_interleave(group, 0) for x in (k, v))
    logits = q.double() @ k.transpose(1, 2) * scaling
    hidden = torch.arange(k.shape[1], device="cuda") >= torch.tensor(sees, device="cuda").view(-1, 1)
    p = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
    # weights in bf16 at most (2^-8), Keys in fp16 (2^-11), as the operators' own tests derive it
    e = (q.double().abs() @ k.abs().transpose(1, 2) * scaling).masked_fill(hidden, 0).amax(-1, keepdim=True) * 2.0 ** -11
    out = p @ v
    return out, U * out.abs() + (U + 2 * e + 2.0 ** -10) * (p @ v.abs()) + 2.0 ** -20


def _inside(got, want):
    off = (got.double() - want[0]).abs() - want[1]
    assert bool((off <= 0).all()), float(off.max())


def test_serving_behind_a_shared_prompt():
    B, n_q, H, D, system = 5, 14, 2, 128, 517
    own = [70, 1, 200, 64, 33]
    freqs, magnitude = rotary_frequencies(64, scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096))
    cache = Int4KVCache(1, B, n_q, H, D, n_pages=64, max_tokens=1200)
    g = torch.Generator(device="cuda").manual_seed(0)
    scaling = D ** -0.5

    def projected(batch, T):
        return [torch.randn(batch, T, h, D, generator=g, device="cuda").to(BF16).transpose(1, 2) for h in (n_q, H, H)]

    # The system prompt, once, as sequence 0's: the others idle.
    q, k, v = projected(B, system)
    cache.extend([system] + [0] * (B - 1))
    qr, kr = cache.rotate(q, k, freqs, magnitude)
    want = _turned(k[:1], [range(system)], freqs, magnitude)
    assert bool(((kr[:1].double() - want).abs() <= U * want.abs() + 2.0 ** -17 * want.abs().amax()).all())
    out = prompt_attention(qr, kr, v, scaling, counts=cache.counts)
    _inside(out[0], _attended(qr[0], kr[0], v[0], scaling, range(1, system + 1)))
    assert not bool(out[1:].any())
    cache.write(0, kr, v)
    assert cache.share(0, range(1, B)) == 512

    # Each sequence's own prompt behind it: a step of different lengths, over the shared pages.
    q, k, v = projected(B, max(own))
    before = cache.lengths.tolist()
    cache.extend(own)
    qr, kr = cache.rotate(q, k, freqs, magnitude)
    cache.write(0, kr, v)
    out = cache.attend_shared(0, qr, scaling)
    hk, hv = cache.read(0)
    for b in range(B):
        _inside(out[b, :, :own[b]], _attended(qr[b, :, :own[b]], hk[b, :, :before[b] + own[b]], hv[b, :, :before[b] + own[b]], scaling,
                                              range(before[b] + 1, before[b] + own[b] + 1)))
        assert not bool(out[b, :, own[b]:].any())

    # Decoding, across page borders; both ways of attending, and a graph's replays.
    for _ in range(3):
        q, k, v = projected(B, 1)
        cache.extend(1)
        qr, kr = cache.rotate(q, k, freqs, magnitude)
        cache.write(0, kr, v)
        shared, plain = cache.attend_shared(0, qr, scaling), cache.attend(0, qr, scaling)
        hk, hv = cache.read(0)
        for b in range(B):
            n = int(cache.lengths[b])
            for got in (shared, plain):
                _inside(got[b], _attended(qr[b], hk[b, :, :n], hv[b, :, :n], scaling, [n]))
    cache.reserve([n + 70 for n in cache.lengths])
    q, k, v = projected(B, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(1)
        qr, kr = cache.rotate(q, k, freqs, magnitude)
        cache.write(0, kr, v)
        out = cache.attend_shared(0, qr, scaling)
    for i in range(66):
        graph.replay()
        cache.advance_host(1)
    hk, hv = cache.read(0)
    for b in range(B):
        n = int(cache.lengths[b])
        _inside(out[b], _attended(qr[b], hk[b, :, :n], hv[b, :, :n], scaling, [n]))
    # The owner of the shared pages goes; the others still read them.
    cache.release([0])
    assert cache.prefix_group.tolist()[1:] == [1] * 4 and int(cache.prefix_pages[1]) == 8
    q, k, v = projected(B, 1)
    cache.extend([0, 1, 1, 1, 1])
    qr, kr = cache.rotate(q, k, freqs, magnitude)
    cache.write(0, kr, v)
    out = cache.attend_shared(0, qr, scaling)
    hk, hv = cache.read(0)
    assert not bool(out[0].any())
    for b in range(1, B):
        n = int(cache.lengths[b])
        _inside(out[b], _attended(qr[b], hk[b, :, :n], hv[b, :, :n], scaling, [n]))
    cache.check_status()


def test_a_long_prompt_in_chunks():
    """One sequence whose prompt comes in chunks: each attends over all before it by way of its own pages."""
    n_q, H, D, chunk = 8, 2, 64, 300
    cache = Int4KVCache(1, 1, n_q, H, D, n_pages=40, max_tokens=2000)
    g = torch.Generator(device="cuda").manual_seed(1)
    for _ in range(5):
        q, k, v = (torch.randn(1, h, chunk, D, generator=g, device="cuda").to(BF16) for h in (n_q, H, H))
        cache.extend(chunk)
        cache.write(0, k, v)
        out = cache.attend_shared(0, q, 0.125)
        hk, hv = cache.read(0)
        n = int(cache.lengths[0])
        _inside(out[0], _attended(q[0], hk[0], hv[0], 0.125, range(n - chunk + 1, n + 1)))
    cache.check_status()


def test_model_prefill_by_the_prompt_kernel():
    """The adapter's prompt="kernel": logits of a prompt and of decode steps next to the dense prefill's."""
    layers = 2
    model = tiny_qwen2(n_q=8, n_kv=2, head_dim=128, layers=layers, vocab=512, seed=31, device="cuda", dtype=BF16, attn="sdpa")
    ids = torch.randint(0, 512, (1, 333), generator=torch.Generator().manual_seed(31)).cuda()
    seen = {}

    def run(prompt):
        a = DeepSeekQwenKVAdapter(model, prompt=prompt).attach()
        a.set_k_levels(list(synthetic_levels(layers, 2, 128, 3.0, seed=31)))
        a.capture = True
        with torch.inference_mode():
            out = model(input_ids=ids, use_cache=True, past_key_values=a.make_cache())
            seen[prompt] = {n: dict(a.captured[n]) for n in "QKV"}
            token = torch.zeros(1, 1, dtype=torch.long, device="cuda")
            after = model(input_ids=token, use_cache=True, past_key_values=out.past_key_values)
        a.packed_manager().cache.check_status()
        a.detach()
        return out.logits, after.logits

    dense, kernel = run("dense"), run("kernel")
    # the first layer's inputs are the same; its attention is within the operator's bound of 64 bits
    q, k, v = (seen["kernel"][n][0] for n in "QKV")
    assert all(torch.equal(seen["dense"][n][0], seen["kernel"][n][0]) for n in "QKV")
    got = prompt_attention(q, k, v, 128 ** -0.5)
    _inside(got[0], _attended(q[0], k[0], v[0], 128 ** -0.5, range(1, 334)))
    assert torch.isfinite(kernel[0]).all() and torch.isfinite(kernel[1]).all()
    # Two bf16 forwards of two layers that differ by roundings: a dozen roundings of 2^-8 in all, of the logits' size.
    # (Not the decode step's: a last-bit difference of a Key moves its 2-bit code, which is no rounding.)
    assert float((dense[0].float() - kernel[0].float()).norm() / dense[0].float().norm()) <= 12 * U
    masked = torch.ones(1, 333, dtype=torch.long, device="cuda")
    masked[0, :3] = 0
    a = DeepSeekQwenKVAdapter(model, prompt="kernel").attach()
    with torch.inference_mode(), pytest.raises(NotImplementedError, match="mask"):
        model(input_ids=ids, attention_mask=masked, use_cache=True, past_key_values=a.make_cache())
    a.detach()
    a = DeepSeekQwenKVAdapter(model, prompt="kernel").attach()
    with pytest.raises(NotImplementedError, match="gradient"):
        model(input_ids=ids, use_cache=True, past_key_values=a.make_cache())
    a.detach()


def test_more_sequences_than_groups_of_a_call():
    """attend_shared takes any batch that attend takes."""
    B = 4096 + 37
    cache = Int4KVCache(1, B, 2, 1, 64, n_pages=B + 40, max_tokens=192)
    g = torch.Generator(device="cuda").manual_seed(4)

    def step(counts, T):
        q, k, v = (torch.randn(B, h, T, 64, generator=g, device="cuda").to(BF16) for h in (2, 1, 1))
        cache.extend(counts)
        cache.write(0, k, v)
        return q

    step([130 if b == 4100 else 0 for b in range(B)], 130)
    cache.share(4100, range(20, 50), 128)
    q = step(1, 1)
    shared, plain = cache.attend_shared(0, q, 0.125), cache.attend(0, q, 0.125)
    hk, hv = cache.read(0)
    for b in (0, 19, 20, 49, 50, 4095, 4096, 4100, B - 1):
        n = int(cache.lengths[b])
        for got in (shared, plain):
            _inside(got[b], _attended(q[b], hk[b, :, :n], hv[b, :, :n], 0.125, [n]))
    assert float((shared.float() - plain.float()).abs().max()) <= 2.0 ** -5    # (either within the bound above: a few units)
    cache.check_status()
