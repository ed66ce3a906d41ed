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
            (NotImplementedError, (q.float().requires_grad_(), None, freqs), ok)]:
        with pytest.raises(error):
            prompt.rotary_embed(*args, **kw)
    with torch.no_grad():
        prompt.rotary_embed(q.float().requires_grad_(), None, freqs, start=start)
    room = torch.zeros(200, 2, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        prompt.rotary_embed(room[:100], None, freqs, positions=torch.arange(100, device="cuda"), out=(room[50:150], None))
