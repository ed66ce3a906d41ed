"""GPU tests of a prompt's operators against their formulas in 64 bits.

Rotary positions: the angle is exact up to 2^-31 turns (the phase is cut to 2^-32
turns, fp32 holds it to 2^-25 of at most 1/8 turn, sincospif is within 2 ulp: 2^-22
of the sine and cosine in all, relative to the pair's length), the rotation has two
fp32 roundings (2^-23 of the length), then the output's own rounding.
"""
from __future__ import annotations

import math

import pytest
import torch

from logitfill_b200 import prompt

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


# ------------------------------------------------------------ rotary positions

def _turned(x, at, freqs, magnitude, interleaved, sign=1):
    """(rotated x in 64 bits, each channel's pair length) of packed x [tokens, heads, D]
    at positions `at` (a list)."""
    n = freqs.numel()
    whole = freqs.tolist()
    phase = torch.tensor([[(p * f) % (1 << 64) / 2.0 ** 64 for f in whole] for p in at], dtype=torch.float64).view(len(at), 1, n)
    c, s = (2 * math.pi * phase).cos() * magnitude, (2 * math.pi * phase).sin() * magnitude * sign
    x = x.double().cpu()
    out, size = x.clone(), torch.zeros_like(x)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a * a + b * b).sqrt() * abs(magnitude)
    return out, size


def _check_turned(got, x, at, freqs, magnitude=1.0, interleaved=False, sign=1):
    want, size = _turned(x, at, freqs, magnitude, interleaved, sign)
    got = got.double().cpu()
    tiny = 2.0 ** -24 if x.dtype == F16 else 0.0          # fp16's smallest steps
    bound = HALF_STEP[x.dtype] * (want.abs() + 2.0 ** -20 * size) + 2.0 ** -20 * size + tiny
    bound[..., 2 * freqs.numel():] = 0.0                  # the other channels are copied
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() - bound).max())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,part", [(128, 128), (64, 64), (64, 16), (128, 34), (80, 80), (96, 32), (256, 64), (6, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_is_the_rotation(dtype, D, part, interleaved):
    g = torch.Generator().manual_seed(D + part)
    tokens, n_q, n_kv = 37, 7, 3
    q, k = (torch.randn(tokens, h, D, generator=g).to(dtype).cuda() for h in (n_q, n_kv))
    at = torch.randint(0, 200000, (tokens,), generator=g)
    freqs, m = prompt.rotary_frequencies(part, scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096))
    gq, gk = prompt.rotary_embed(q, k, freqs, positions=at.cuda(), magnitude=m, interleaved=interleaved)
    _check_turned(gq, q, at.tolist(), freqs, m, interleaved)
    _check_turned(gk, k, at.tolist(), freqs, m, interleaved)
    for same in (at.int().cuda(), torch.stack([at, at], 1).cuda()[:, 0]):    # int32, and a stride of its own
        assert torch.equal(prompt.rotary_embed(q, k, freqs, positions=same, magnitude=m, interleaved=interleaved)[0], gq)


@pytest.mark.parametrize("at", [0, 1, -1, -70001, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 3])
def test_far_positions_keep_their_angle(at):
    g = torch.Generator().manual_seed(3)
    q = torch.randn(1, 2, 128, generator=g).cuda()
    freqs, _ = prompt.rotary_frequencies(128, base=1e6)
    got, none = prompt.rotary_embed(q, None, freqs, positions=torch.tensor([at]).cuda())
    assert none is None
    _check_turned(got, q, [at], freqs)


@pytest.mark.parametrize("B,T", [(1, 1), (16, 1), (3, 5), (2, 300)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_batches_and_starts(B, T, dtype):
    """[batch, heads, tokens, D] as a projection's transposed view, positions from starts."""
    g = torch.Generator().manual_seed(B * T)
    D, freqs = 128, prompt.rotary_frequencies(128)[0]
    q, k = (torch.randn(B, T, h, D, generator=g).to(dtype).cuda().transpose(1, 2) for h in (28, 4))
    start = torch.tensor([8192 - 31 * b for b in range(B)], dtype=torch.int32).cuda()
    gq, gk = prompt.rotary_embed(q, k, freqs, start=start)
    at = [8192 - 31 * b + t for b in range(B) for t in range(T)]
    for got, x in ((gq, q), (gk, k)):
        assert got.shape == x.shape and got.stride() == x.stride()
        _check_turned(got.transpose(1, 2).flatten(0, 1), x.transpose(1, 2).flatten(0, 1), at, freqs)
    positions = (start.view(-1, 1) + torch.arange(T, device="cuda")).long()
    assert torch.equal(prompt.rotary_embed(q, k, freqs, positions=positions)[0], gq)
    assert torch.equal(prompt.rotary_embed(q.contiguous(), None, freqs, positions=positions)[0], gq)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,part,tokens,n_q,n_kv,dtype", [
    (128, 128, 300, 28, 4, BF16), (128, 128, 1101, 40, 8, F16), (256, 256, 333, 17, 1, F32), (64, 32, 1500, 9, 0, BF16),
    (80, 48, 999, 31, 2, F16), (256, 2, 200, 3, 1, BF16), (128, 64, 2049, 1, 3, F32)])
def test_calls_that_fill_the_gpu(interleaved, D, part, tokens, n_q, n_kv, dtype):
    """Blocks of both sizes, several heads to a thread, heads that are no multiple of those."""
    g = torch.Generator().manual_seed(tokens)
    q, k = (torch.randn(tokens, h, D, generator=g).to(dtype).cuda() for h in (n_q, n_kv))
    at = torch.randint(0, 70000, (tokens,), generator=g)
    freqs, _ = prompt.rotary_frequencies(part)
    gq, gk = prompt.rotary_embed(q, k, freqs, positions=at.cuda(), interleaved=interleaved)
    _check_turned(gq, q, at.tolist(), freqs, 1.0, interleaved)
    _check_turned(gk, k, at.tolist(), freqs, 1.0, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,part,shift", [(128, 128, 0), (64, 32, 0), (128, 128, 1), (96, 40, 3)])
def test_in_place_and_unaligned(interleaved, D, part, shift):
    """Queries and Keys of one projection's buffer, at any element offset, turned where they lie."""
    g = torch.Generator().manual_seed(D + shift)
    tokens, n_q, n_kv = 70, 5, 2
    room = torch.randn(tokens * (n_q + 2 * n_kv) * D + shift, generator=g).to(BF16).cuda()
    both = room[shift:].view(tokens, n_q + 2 * n_kv, D)
    q, k = both[:, :n_q], both[:, n_q:n_q + n_kv]
    before = room.clone()
    freqs, _ = prompt.rotary_frequencies(part)
    at = torch.arange(tokens).cuda() + 100
    want = prompt.rotary_embed(q.clone(), k.clone(), freqs, positions=at, interleaved=interleaved)
    got = prompt.rotary_embed(q, k, freqs, positions=at, interleaved=interleaved, out=(q, k))
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])
    rest = before[shift:].view(tokens, n_q + 2 * n_kv, D)
    assert torch.equal(both[:, n_q + n_kv:], rest[:, n_q + n_kv:]) and torch.equal(room[:shift], before[:shift])


def test_transposed_takes_it_back():
    g = torch.Generator().manual_seed(5)
    q = torch.randn(50, 4, 64, generator=g).cuda()
    at = (torch.arange(50) * 1013).cuda()
    freqs, _ = prompt.rotary_frequencies(64)
    turned = prompt.rotary_embed(q, None, freqs, positions=at, magnitude=2.0)[0]
    back = prompt.rotary_embed(turned, None, freqs, positions=at, magnitude=0.5, transposed=True)[0]
    _check_turned(prompt.rotary_embed(q, None, freqs, positions=at, magnitude=2.0, transposed=True)[0], q, at.tolist(), freqs, 2.0, sign=-1)
    # two rotations, each within 2^-20 and a rounding of a pair's length
    size = (q[..., :32] ** 2 + q[..., 32:] ** 2).sqrt().repeat(1, 1, 2)
    assert bool(((back - q).abs() <= 4 * 2.0 ** -20 * size).all())


def test_gradient_by_differences():
    """The transposed call is the gradient: sum(g * (f(x + d) - f(x))) = sum(f'(g) * d), f being linear."""
    g = torch.Generator().manual_seed(6)
    x, d, up = (torch.randn(9, 3, 32, generator=g).cuda() for _ in range(3))
    freqs, _ = prompt.rotary_frequencies(16)
    at = torch.arange(9).cuda() * 77
    f = lambda y, **kw: prompt.rotary_embed(y, None, freqs, positions=at, magnitude=1.5, **kw)[0]  # noqa: E731
    left = (up.double() * (f(x + d).double() - f(x).double())).sum()
    grad = f(up, transposed=True).double()
    grad[..., 16:] = up.double()[..., 16:]
    right = (grad * ((x + d).double() - x.double())).sum()
    # 9 * 3 * 32 products of a few units, each factor within 2^-19
    assert abs(float(left - right)) <= 2.0 ** -19 * float((up.abs() * (x.abs() + d.abs()) * 4).double().sum())


def test_non_finite_channels_stay_in_their_pair():
    q = torch.ones(2, 2, 64, dtype=BF16, device="cuda")
    q[0, 1, 3] = float("nan")
    q[1, 0, 40] = float("inf")
    freqs, _ = prompt.rotary_frequencies(64)
    got = prompt.rotary_embed(q, None, freqs, positions=torch.tensor([5, 0], device="cuda"))[0]
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, 1, [3, 35]] = True
    want[1, 0, [8, 40]] = True      # inf * sin(0) is NaN
    assert torch.equal(bad, want)


def test_rotary_streams_graphs_and_empty_calls():
    g = torch.Generator().manual_seed(8)
    q, k = torch.randn(2, 8, 3, 64, generator=g).cuda(), torch.randn(2, 2, 3, 64, generator=g).cuda()
    freqs, _ = prompt.rotary_frequencies(64)
    start = torch.tensor([7, 900], dtype=torch.int32, device="cuda")
    want = prompt.rotary_embed(q, k, freqs, start=start)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = prompt.rotary_embed(q, k, freqs, start=start)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = (torch.zeros_like(q), torch.zeros_like(k))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompt.rotary_embed(q, k, freqs, start=start, out=out)
    graph.replay()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    start += 1
    graph.replay()
    assert torch.equal(out[0], prompt.rotary_embed(q, k, freqs, start=start)[0]) and not torch.equal(out[0], want[0])
    for empty in (q[:, :, :0], q[:0], q[:, :0]):
        s = start[:empty.shape[0]]
        assert prompt.rotary_embed(empty, None, freqs, start=s)[0].shape == empty.shape


def test_rotary_offsets_past_32_bits():
    """Rows more than 2^31 elements apart in one buffer."""
    room = torch.zeros(3 * (1 << 30) + 4096, dtype=BF16, device="cuda")
    q = room.as_strided((3, 2, 64), (1 << 30, 64 * 3, 1), 7 * 8)
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 2, 64, generator=g).to(BF16).cuda()
    q.copy_(x)
    freqs, _ = prompt.rotary_frequencies(64)
    at = torch.arange(3).cuda() + 17
    prompt.rotary_embed(q, None, freqs, positions=at, out=(q, None))
    assert torch.equal(q, prompt.rotary_embed(x, None, freqs, positions=at)[0])
    del room


def test_rotary_refusals():
    q = torch.zeros(2, 8, 3, 64, dtype=BF16, device="cuda")
    k = torch.zeros(2, 2, 3, 64, dtype=BF16, device="cuda")
    freqs, _ = prompt.rotary_frequencies(64)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    ok = dict(start=start)
    for error, args, kw in [
            (ValueError, (q, k, freqs), {}), (ValueError, (q, k, freqs), dict(start=start, positions=start.view(2, 1))),
            (ValueError, (q, k[:1], freqs), ok), (ValueError, (q, k.float(), freqs), ok), (ValueError, (q, k[..., :32], freqs), ok),
            (ValueError, (q, k, freqs.int()), ok), (ValueError, (q, k, freqs.repeat(2)), ok), (ValueError, (q, k, freqs[:0]), ok),
            (ValueError, (q, k, freqs), dict(start=start.long())), (ValueError, (q, k, freqs), dict(start=start[:1])),
            (ValueError, (q, k, freqs), dict(positions=torch.zeros(2, 4, dtype=torch.int32, device="cuda"))),
            (ValueError, (q[0, 0], None, freqs), ok), (TypeError, (q, k, freqs), dict(start=start, out=q)),
            (ValueError, (q, k, freqs), dict(start=start, out=(q[:, :4], k))), (ValueError, (q, k, freqs), dict(start=start, magnitude=float("inf"))),
            (ValueError, (q, q, freqs), dict(start=start, out=(q, q))), (TypeError, (q, 3, freqs), ok),
            (ValueError, (q, k, freqs), dict(start=start, out=(torch.zeros(1, 8, 3, 64, dtype=BF16, device="cuda").expand(2, -1, -1, -1), k))),
            (NotImplementedError, (q.double(), None, freqs), ok), (RuntimeError, (q, k.cpu(), freqs), ok),
            (TypeError, (q, k, freqs), dict(start=start, interleaved=start)), (TypeError, (q, k, freqs), dict(start=start, transposed=start)),
            (NotImplementedError, (q.float().requires_grad_(), None, freqs), ok)]:
        with pytest.raises(error):
            prompt.rotary_embed(*args, **kw)
    with torch.no_grad():
        prompt.rotary_embed(q.float().requires_grad_(), None, freqs, start=start)
    room = torch.zeros(200, 2, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        prompt.rotary_embed(room[:100], None, freqs, positions=torch.arange(100, device="cuda"), out=(room[50:150], None))


# ------------------------------------------------------------ prompt attention
#
# Element by element within  u |out| + (u + 2 e + 2^-16) sum p |v| + n 2^-30 max |v|:
# u is half a step of the type, for the output and for the weights that enter the
# product with Value; e, the fp32 sums of a score: 128 products of 2^-24 each, scaled,
# of the row's largest sum |q k|, in a weight and in the sum of weights; 2^-16 the
# exponential, the running sums and their rescalings; the last term what fp16 weights
# lose below their smallest step (2^-25 of weights whose largest is at 2^7, or 2^-1
# where the running maximum lags by its slack of 2^8).

def _prompts(seed, counts, n_q, n_kv, D, dtype=BF16, keys=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = max(sum(counts), 0)
    q, k, v = (torch.randn(n, h, D, generator=g, device="cuda") for h in (n_q, n_kv, n_kv))
    k[..., ::19] *= keys
    return q.to(dtype), k.to(dtype), v.to(dtype)


def _one(q, k, v, scaling, dtype):
    """(out, bound) of one sequence: q [n, n_q, D], k and v [n, n_kv, D], in 64 bits."""
    n, n_q, D = q.shape
    group = n_q // k.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    later = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
    u = HALF_STEP[dtype]
    for h in range(n_q):
        a, b, c = q[:, h].double(), k[:, h // group].double(), v[:, h // group].double()
        logits = (a @ b.T * scaling).masked_fill(later, -math.inf)
        p = torch.softmax(logits, -1)
        e = (a.abs() @ b.abs().T * abs(scaling)).masked_fill(later, 0).amax(-1, keepdim=True) * 128 * 2.0 ** -24
        out[:, h] = p @ c
        bound[:, h] = u * out[:, h].abs() + (u + 2 * e + 2.0 ** -16) * (p @ c.abs()) + n * 2.0 ** -30 * c.abs().max() + 2.0 ** -24
    return out, bound


def _check_prompts(got, q, k, v, counts, scaling, dtype):
    at = 0
    for c in counts:
        if c:
            want, bound = _one(q[at:at + c], k[at:at + c], v[at:at + c], scaling, dtype)
            off = (got[at:at + c].double() - want).abs() - bound
            assert bool((off <= 0).all()), f"{c} tokens: outside by {float(off.max()):.3g} in {int((off > 0).sum())} places, {int(off.isnan().sum())} NaN"
        at += c


def _starts(counts, device="cuda"):
    return torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32, device=device)


HEADS = [(28, 4), (8, 8), (16, 1), (40, 8), (9, 3)]


@pytest.mark.parametrize("n_q,n_kv", HEADS)
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F16, 128), (BF16, 64)])
def test_prompts_of_every_length(n_q, n_kv, dtype, D):
    counts = [1, 2, 17, 0, 18, 19, 36, 37, 64, 127, 128, 129, 0, 255, 256, 257, 300]
    q, k, v = _prompts(n_q + D, counts, n_q, n_kv, D, dtype)
    got = prompt.prompt_attention(q, k, v, D ** -0.5, starts=_starts(counts))
    assert got.shape == q.shape and got.dtype == dtype
    _check_prompts(got, q, k, v, counts, D ** -0.5, dtype)
    # a sequence's result does not depend on its neighbours
    at = sum(counts[:11])
    alone = prompt.prompt_attention(q[at:at + 129], k[at:at + 129], v[at:at + 129], D ** -0.5)
    assert torch.equal(alone, got[at:at + 129])


@pytest.mark.parametrize("n_q,n_kv,D,dtype,counts", [(28, 4, 128, BF16, [2500]), (4, 2, 128, BF16, [1, 4097, 3]), (128, 1, 64, F16, [333]),
                                                     (100, 1, 128, BF16, [70, 5]), (65, 1, 64, BF16, [40]), (12, 3, 64, F16, [1700, 900])])
def test_longer_prompts_and_wide_groups(n_q, n_kv, D, dtype, counts):
    q, k, v = _prompts(n_q, counts, n_q, n_kv, D, dtype)
    _check_prompts(prompt.prompt_attention(q, k, v, D ** -0.5, starts=_starts(counts)), q, k, v, counts, D ** -0.5, dtype)


def test_many_short_sequences():
    counts = [1 + b * 7 % 23 for b in range(700)]
    q, k, v = _prompts(1, counts, 6, 2, 64, F16)
    _check_prompts(prompt.prompt_attention(q, k, v, 0.125, starts=_starts(counts)), q, k, v, counts, 0.125, F16)


@pytest.mark.parametrize("dtype,D,B,T,n_q,n_kv", [(BF16, 128, 3, 200, 14, 2), (F16, 64, 5, 37, 8, 8), (BF16, 64, 2, 513, 6, 1)])
def test_padded_batches(dtype, D, B, T, n_q, n_kv):
    """Padding holds NaN: it is not read into anything, and comes out as 0."""
    counts = [T, 0, 1, T - 1, 20][:B] if B > 2 else [T - 130, T]
    q, k, v = _prompts(T, [T] * B, n_q, n_kv, D, dtype)
    q, k, v = (x.view(B, T, -1, D) for x in (q, k, v))
    for x in (q, k, v):
        for b, c in enumerate(counts):
            x[b, c:] = float("nan")
    device = torch.tensor(counts, dtype=torch.int32, device="cuda")
    for contiguous in (False, True):
        a, b_, c_ = ((x.transpose(1, 2).contiguous() if contiguous else x.transpose(1, 2)) for x in (q, k, v))
        got = prompt.prompt_attention(a, b_, c_, D ** -0.5, counts=device)
        assert got.shape == (B, n_q, T, D)
        for b, c in enumerate(counts):
            assert not bool(got[b, :, c:].any())
            if c:
                _check_prompts(got[b].transpose(0, 1), q[b], k[b], v[b], [c], D ** -0.5, dtype)
    full = [torch.nan_to_num(x.transpose(1, 2)) for x in (q, k, v)]
    every = prompt.prompt_attention(*full, D ** -0.5)
    for b in range(B):
        _check_prompts(every[b].transpose(0, 1), *(x[b].transpose(0, 1) for x in full), [T], D ** -0.5, dtype)


def test_padding_alone_between_prompts():
    """Many tiles of nothing but padding before, between and after those with tokens."""
    counts, T, D = [0, 3, 0, 0, 1500, 0], 1500, 128
    q, k, v = _prompts(21, [T] * 6, 4, 2, D)
    q, k, v = (x.view(6, T, -1, D).transpose(1, 2) for x in (q, k, v))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = prompt.prompt_attention(q, k, v, 0.09, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"), status=status)
    assert int(status) == 0
    for b, c in enumerate(counts):
        assert not bool(got[b, :, c:].any())
        if c:
            _check_prompts(got[b].transpose(0, 1), *(x[b].transpose(0, 1) for x in (q, k, v)), [c], 0.09, BF16)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64)])
def test_rows_of_no_sequence_stay_as_they_were(dtype, D):
    """Rows before, between and behind the sequences, NaN in all of them."""
    q, k, v = _prompts(2, [400], 10, 2, D, dtype)
    starts = torch.tensor([30, 95, 95, 300], dtype=torch.int32, device="cuda")
    for x in (q, k, v):
        x[:30], x[300:] = float("nan"), float("inf")
    out = torch.full_like(q, 7.0)
    got = prompt.prompt_attention(q, k, v, D ** -0.5, starts=starts, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((out[:30] == 7).all()) and bool((out[300:] == 7).all())
    _check_prompts(out[30:300], q[30:300], k[30:300], v[30:300], [65, 0, 205], D ** -0.5, dtype)
    # starts that leave the rows, or run backwards, are cut to what there is
    for bad, spans in [((-50, 95, 90, 1 << 30), [(0, 95), (90, 400)]), ((300, 30, 2000000000, -5), [(30, 400)]), ((-9, -3), [])]:
        out.fill_(7.0)
        prompt.prompt_attention(*(torch.nan_to_num(x, 1.0, 1.0, 1.0) for x in (q, k, v)), D ** -0.5,
                                starts=torch.tensor(bad, dtype=torch.int32, device="cuda"), out=out)
        covered = torch.zeros(400, dtype=torch.bool)
        for low, high in spans:
            covered[low:high] = True
        written = ~(out == 7).all(-1).all(-1).cpu()
        assert torch.equal(written, covered)


@pytest.mark.parametrize("scaling", [0.0, -0.09, 1e-30, 40.0, -700.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scalings_of_any_sign_and_size(scaling, dtype):
    q, k, v = _prompts(4, [200, 77], 4, 2, 128, dtype, keys=1.0)
    got = prompt.prompt_attention(q, k, v, scaling, starts=_starts([200, 77]))
    if abs(scaling) < 1:
        _check_prompts(got, q, k, v, [200, 77], scaling, dtype)
    else:
        # One token takes nearly all: where the best leads by more than the scores' error, it is the result.
        # (First asked for to the last bit, which is wrong: its weight w, any number near the running maximum's,
        # enters the product with Value as w (1 + d), |d| <= u, half a step of the type, and the sum in fp32 as
        # w; the quotient v (1 + d) is then rounded once more: u |v| + u |v| (1 + u) in all.)
        u = HALF_STEP[dtype]
        at = 0
        for c in (200, 77):
            for h in range(4):
                a, b = q[at:at + c, h].double(), k[at:at + c, h // 2].double()
                later = torch.ones(c, c, dtype=torch.bool, device="cuda").triu(1)
                logits = (a @ b.T * scaling).masked_fill(later, -math.inf)
                e = float((a.abs() @ b.abs().T).max()) * abs(scaling) * 128 * 2.0 ** -24
                best = logits.topk(2, -1)
                sure = best.values[:, 0] - best.values[:, 1] > 30 + 2 * e
                assert int(sure.sum()) > c // 3
                want = v[at:at + c, h // 2][best.indices[:, 0]].double()
                assert bool(((got[at:at + c, h].double() - want).abs() <= (2 * u + 2 * u * u) * want.abs() + 2.0 ** -24)[sure].all())
            at += c


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("size", [3e2, 1e4, 2.0 ** 60])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_magnitude(dtype, D, size, sign):
    """Scores up to 1e5 and 1e19, all above or all below zero, over several tiles: a weight is what the difference
    of two scores says.  Keys are whole multiples of one direction, so that the scores are exact in fp32."""
    n = 600
    g = torch.Generator(device="cuda").manual_seed(7)
    step = torch.randint(1, 60, (n, 1, 1), generator=g, device="cuda").float()
    k = (step * torch.ones(n, 1, D, device="cuda")).to(dtype)
    q = torch.full((n, 3, D), float(sign), dtype=dtype, device="cuda")
    v = torch.randn(n, 1, D, generator=g, device="cuda").to(dtype)
    scaling = size / 60 / D
    got = prompt.prompt_attention(q, k, v, scaling)
    # exact scores D * step * sign, whole numbers: the only error is fp32's in the difference's product with the scaling
    logits = (sign * D * step[:, 0, 0].double() * float(torch.tensor(scaling, dtype=torch.float32))).view(1, n).expand(n, n)
    p = torch.softmax(logits.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf), -1)
    vv, u = v[:, 0].double(), HALF_STEP[dtype]
    want = p @ vv
    # in an exponent of size x (at most 25 where a weight counts) 3 roundings of 2^-24 x; kLargeTop 2^10 leaves 2^-14
    bound = u * want.abs() + (u + 2.0 ** -13) * (p @ vv.abs()) + 2.0 ** -24
    for h in range(3):
        off = (got[:, h].double() - want).abs() - bound
        assert bool((off <= 0).all()), float(off.max())


def test_a_dominant_token_keeps_the_others():
    """An attention sink with a small Value, others 10 to 16 below it: in fp16 weights their share would drop out
    if the largest weight stood at 1."""
    n, D = 500, 128
    g = torch.Generator(device="cuda").manual_seed(5)
    for gap in (10.0, 16.0):
        q = torch.ones(n, 2, D, dtype=F16, device="cuda")
        k = torch.zeros(n, 1, D, dtype=F16, device="cuda")
        k[0] = gap / D
        v = (torch.randn(n, 1, D, generator=g, device="cuda").abs() + 1).to(F16)
        v[0] = 0.0
        got = prompt.prompt_attention(q, k, v, 1.0)
        _check_prompts(got, q, k, v, [n], 1.0, F16)


@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_rise_and_fall(rising):
    """The running maximum moves at every tile, or only at the first."""
    n, D = 1500, 128
    q = torch.ones(n, 7, D, dtype=BF16, device="cuda")
    ramp = torch.linspace(0, 120, n, device="cuda") / D
    k = (ramp if rising else ramp.flip(0)).to(BF16).view(n, 1, 1).expand(n, 1, D).contiguous()
    g = torch.Generator(device="cuda").manual_seed(6)
    v = torch.randn(n, 1, D, generator=g, device="cuda").to(BF16)
    _check_prompts(prompt.prompt_attention(q, k, v, 1.0), q, k, v, [n], 1.0, BF16)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["key", "value", "query"])
def test_non_finite_rows_reach_only_who_sees_them(dtype, D, value, where):
    counts = [300, 140]
    q, k, v = _prompts(7, counts, 6, 2, D, dtype)
    want = [torch.cat(x) for x in zip(*(_one(q[a:b], k[a:b], v[a:b], D ** -0.5, dtype) for a, b in ((0, 300), (300, 440))))]
    at = 133                      # inside a tile, of the first sequence, KV head 1
    dict(key=k, value=v, query=q)[where][at, 1, 5] = value
    got = prompt.prompt_attention(q, k, v, D ** -0.5, starts=_starts(counts))
    touched = torch.zeros(440, 6, D, dtype=torch.bool, device="cuda")
    if where == "query":
        touched[at, 1] = True
    elif where == "key":
        touched[at:300, 3:] = True
    else:
        touched[at:300, 3:, 5] = True
    off = (got.double() - want[0]).abs() - want[1]     # tiles with such a row may be summed in another way: not bit for bit
    assert bool((off[~touched] <= 0).all())
    if where == "value":
        assert not bool(torch.isfinite(got[touched]).any())
    elif math.isnan(value):
        assert bool(torch.isnan(got[touched]).all())


def test_prompt_strides_and_unaligned_rows():
    """Views of one projection's buffer, broadcast Keys, rows at odd offsets (copied first)."""
    counts, D = [90, 41], 64
    g = torch.Generator(device="cuda").manual_seed(8)
    room = torch.randn(131 * (6 + 2 + 2) * D + 1, generator=g, device="cuda").to(BF16)
    for shift in (0, 1):
        both = room[shift:shift + 131 * 10 * D].view(131, 10, D)
        q, k, v = both[:, :6], both[:, 6:8], both[:, 8:]
        got = prompt.prompt_attention(q, k, v, 0.125, starts=_starts(counts))
        _check_prompts(got, q, k, v, counts, 0.125, BF16)
        want = prompt.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), 0.125, starts=_starts(counts))
        assert torch.equal(got, want)
    one = k[:, :1].expand(-1, 2, -1)
    assert torch.equal(prompt.prompt_attention(q, one, v, 0.125), prompt.prompt_attention(q, one.contiguous(), v, 0.125))
    # heads first in memory, an out of other strides
    turned = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    out = torch.zeros(131, 8, D, dtype=BF16, device="cuda")[:, 1:7]
    assert torch.equal(prompt.prompt_attention(*turned, 0.125, starts=_starts(counts), out=out), got)


def test_prompt_streams_graphs_and_empty_calls():
    counts, D = [300, 29, 171], 128
    q, k, v = _prompts(9, counts, 8, 2, D)
    starts = _starts(counts)
    want = prompt.prompt_attention(q, k, v, 0.09, starts=starts)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [prompt.prompt_attention(q, k, v, 0.09, starts=starts) for _ in range(3)]
    both = [prompt.prompt_attention(q, k, v, 0.09, starts=starts) for _ in range(3)]     # two streams at once
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, want) for x in got + both)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompt.prompt_attention(q, k, v, 0.09, starts=starts, out=out)
    graph.replay()
    assert torch.equal(out, want)
    starts.copy_(_starts([100, 350, 50]))     # the lengths are read when it runs
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(out, prompt.prompt_attention(q, k, v, 0.09, starts=starts)) and not torch.equal(out, want)
    assert prompt.prompt_attention(q[:0], k[:0], v[:0], 1.0).shape == (0, 8, D)
    assert prompt.prompt_attention(q[:0], k[:0], v[:0], 1.0, starts=starts).shape == (0, 8, D)
    padded = [x.view(2, 250, -1, D).transpose(1, 2) for x in (q, k, v)]
    assert prompt.prompt_attention(*(x[:0] for x in padded), 1.0).shape == (0, 8, 250, D)
    assert not bool(prompt.prompt_attention(*padded, 1.0, counts=torch.tensor([0, -3], dtype=torch.int32, device="cuda")).any())


def test_prompt_offsets_past_32_bits():
    """Rows more than 2^31 elements apart."""
    n, D, tok = 40, 64, 1 << 26
    room = torch.empty(n * tok, dtype=BF16, device="cuda")
    q = room.as_strided((n, 2, D), (tok, D, 1), 0)
    k, v = room.as_strided((n, 1, D), (tok, D, 1), 1024), room.as_strided((n, 1, D), (tok, D, 1), 2048)
    out = room.as_strided((n, 2, D), (tok, D, 1), 4096)
    made = _prompts(10, [n], 2, 1, D)
    for x, y in zip((q, k, v), made):
        x.copy_(y)
    prompt.prompt_attention(q, k, v, 0.125, out=out)
    assert torch.equal(out, prompt.prompt_attention(*made, 0.125))
    del room


def test_prompt_refusals():
    q, k, v = _prompts(11, [32], 8, 2, 64)
    starts = _starts([20, 12])
    p4 = [x.view(2, 16, -1, 64).transpose(1, 2) for x in (q, k, v)]
    counts = torch.tensor([16, 3], dtype=torch.int32, device="cuda")
    for error, args, kw in [
            (ValueError, (q, k[:31], v, 1.0), {}), (ValueError, (q, k, v[:, :1], 1.0), {}), (ValueError, (q, k.half(), v, 1.0), {}),
            (ValueError, (q[:, :7], k, v, 1.0), {}), (ValueError, (q[:, :0], k, v, 1.0), {}), (ValueError, (q[0], k[0], v[0], 1.0), {}),
            (ValueError, (q, k, v, float("nan")), {}), (ValueError, (q, k, v, float("inf")), {}), (TypeError, (q, k, v, "1"), {}),
            (ValueError, (q, k, v, 1.0), dict(counts=counts)), (ValueError, (*p4, 1.0), dict(starts=starts)),
            (ValueError, (q, k, v, 1.0), dict(starts=starts.long())), (ValueError, (q, k, v, 1.0), dict(starts=starts[:0])),
            (ValueError, (q, k, v, 1.0), dict(starts=starts.cpu())), (ValueError, (*p4, 1.0), dict(counts=counts[:1])),
            (ValueError, (q, k, v, 1.0), dict(out=q)), (ValueError, (q, k, v, 1.0), dict(out=q.float())),
            (ValueError, (q, k, v, 1.0), dict(out=torch.zeros(1, 8, 64, dtype=BF16, device="cuda").expand(32, 8, 64))),
            (NotImplementedError, (q.float(), k.float(), v.float(), 1.0), {}), (RuntimeError, (q.cpu(), k, v, 1.0), {}),
            (RuntimeError, (q, k.cpu(), v, 1.0), {}), (NotImplementedError, tuple(x[..., :32] for x in (q, k, v)) + (1.0,), {}),
            (NotImplementedError, (q.repeat(1, 17, 1), k[:, :1], v[:, :1], 1.0), {}),
            (NotImplementedError, (q.clone().requires_grad_(), k, v, 1.0), {}), (TypeError, (q, None, v, 1.0), {})]:
        with pytest.raises(error):
            prompt.prompt_attention(*args, **kw)
