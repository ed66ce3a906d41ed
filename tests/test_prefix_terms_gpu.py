"""GPU tests of what attention over shared 4-bit pages holds in two fp16 numbers for an fp16
output: Keys, and softmax weights.

Every sequence ends with the shared pages, so nothing but those is read.  Values are whole
numbers (exact in fp16).  Element by element within
  u |out| + sum p e |v| + (sum p e + 2^-16) sum p |v| + n 2^-32 max |v| + 2^-24:
u, half a step of fp16, for the output; e what a score is off by: a Key code * s + z as two
numbers, where the product and the sum are rounded to 2^-11 and what is left over again, to
2^-22 of both (|code * s| is at most twice the token's largest Key) or half of fp16's smallest step,
and the fp32 sums of both numbers' products; 2^-16 the exponential and the sums of weights,
whose second number leaves 2^-22 of them or 2^-32 of the largest (which stands at 2^7).
Each test plants the mistake of a single number in the definition, and sees it outside.
"""
from __future__ import annotations

import math

import pytest
import torch

from logitfill_b200 import int4

F16 = torch.float16
U = 2.0 ** -11


def made(which, seed, D, tokens, rows):
    """(query [rows, D], Key and Value [tokens, D], scaling) in fp32."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randint(-8, 8, (tokens, D), generator=g).float()
    if which == "keys":      # scores of some 8 either way: a score's error is its weight's
        q = (torch.randn(rows, D, generator=g) * 8 / 1.3).to(F16).float()
        k = torch.randn(tokens, D, generator=g)
        k[:, ::19] *= 3.0
    else:                    # four pairs of tokens of nearly equal weights and opposite Values, all others far below: results near 0
        q = torch.randn(rows, D, generator=g).to(F16).float()
        k = torch.randn(tokens // 2, D, generator=g).repeat_interleave(2, 0) * 0.1
        at = torch.randint(3, D, (tokens // 2,), generator=g)
        k[1::2].scatter_add_(1, at.view(-1, 1), torch.full((tokens // 2, 1), 0.1))
        near = torch.randperm(tokens // 2, generator=g)[:4]
        q[:, 2] = D ** 0.5
        k[:, 2] = -30.0
        k[2 * near, 2] = k[2 * near + 1, 2] = 0.0
        v = torch.where(torch.randint(0, 2, (tokens // 2, D), generator=g) == 0, -7.0, 7.0).repeat_interleave(2, 0)
        v[1::2] *= -1
    v[:, 0::32], v[:, 1::32] = -8.0, 7.0     # each group of 32 channels: minimum -8, steps of 1
    return q, k, v, D ** -0.5


def checked(q, k, v, scaling):
    """(out, bound, out with single Keys, out with single weights) over what the pages hold, in 64 bits."""
    logits = q @ k.T * scaling
    top = logits.amax(-1, keepdim=True)
    w = (logits - top).exp()
    p = w / w.sum(-1, keepdim=True)
    out, size = p @ v, p @ v.abs()
    largest, n, D = k.abs().amax(-1), k.shape[0], k.shape[1]
    e = scaling * (q.abs().sum(-1, keepdim=True) * (2.0 ** -22 * 3 * largest + 2.0 ** -25) + q.abs() @ k.abs().T * 2 * D * 2.0 ** -24)
    off = (p * e) @ v.abs() + (p * e).sum(-1, keepdim=True) * size      # of each score in its weight, and in the sum of weights
    bound = U * out.abs() + off + 2.0 ** -16 * size + n * 2.0 ** -32 * float(v.abs().max()) + 2.0 ** -24
    keys = torch.softmax(q @ k.to(F16).double().T * scaling, -1) @ v
    weights = (w * 2.0 ** 7).to(F16).double() @ v / (w * 2.0 ** 7).sum(-1, keepdim=True)
    return out, bound, keys, weights


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["keys", "weights"])
@pytest.mark.parametrize("D,pages,n_q,sequences", [(64, 2, 6, 5), (128, 3, 14, 20), (64, 9, 1, 40)])
def test_an_fp16_output_has_keys_and_weights_in_two_numbers(which, D, pages, n_q, sequences):
    tokens = 64 * pages
    q, k, v, scaling = made(which, D + pages, D, tokens, sequences * n_q)
    pool = int4.alloc_pages(pages + 1, 1, D)
    table = torch.arange(1, pages + 1, dtype=torch.int32, device="cuda").repeat(sequences, 1)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    int4.int4_write(k.cuda().view(1, 1, tokens, D), v.cuda().view(1, 1, tokens, D), pool, table[:1], zero)
    hk, hv = (x[0, 0].double() for x in int4.int4_read(pool, table[:1], zero, tokens))
    assert torch.equal(hv.cpu(), v.double())
    query = q.cuda().to(F16).view(sequences, n_q, D)
    got = int4.int4_prefix_attention(query, pool, table, zero.repeat(sequences) + tokens, scaling, zero.repeat(sequences),
                                     torch.full((1,), pages, dtype=torch.int32, device="cuda"), always=True)
    out, bound, keys, weights = checked(query.view(-1, D).double(), hk, hv, scaling)
    off = (got.view(-1, D).double() - out).abs() - bound
    assert bool((off <= 0).all()), f"outside by {float(off.max()):.3g} in {int((off > 0).sum())} places"
    planted = keys if which == "keys" else weights
    assert int(((planted.to(F16).double() - out).abs() > bound).sum()) > 20


@pytest.mark.parametrize("which", ["keys", "weights"])
@pytest.mark.parametrize("D,pages,n_q,sequences", [(64, 2, 6, 5), (128, 3, 14, 20), (64, 9, 1, 40)])
def test_the_bound_tells_one_number_from_two(which, D, pages, n_q, sequences):
    """The same on the CPU, by the format's definition: what a single number gives is outside, a result that is off
    by a rounding is not."""
    from tests.int4_reference import stored

    q, k, v, scaling = made(which, D + pages, D, 64 * pages, sequences * n_q)
    hk, hv = (torch.from_numpy(stored(x.numpy())).double() for x in (k, v))
    assert torch.equal(hv, v.double())
    out, bound, keys, weights = checked(q.double(), hk, hv, scaling)
    planted = keys if which == "keys" else weights
    assert int(((planted.to(F16).double() - out).abs() > bound).sum()) > 20
    assert bool(((out.to(F16).double() - out).abs() <= bound).all()) and not bool(bound.isnan().any())
    assert math.isfinite(scaling)
