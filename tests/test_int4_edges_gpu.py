"""GPU tests of the 4-bit cache at the edges of its values and arguments.  The
reference and the helpers are those of :mod:`tests.test_int4_gpu`."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from logitfill_b200 import int4
from tests import int4_reference as ref
from tests.test_int4_gpu import BF16, F16, ROUND, _dense_reference, _filled, _garbage, _i32, _kv, _picks, _table

pytestmark = pytest.mark.gpu


def _queries(seed, B, nq, q_len, D, dtype=BF16):
    return torch.randn(B, nq, q_len, D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _check(got, want, weight, dtype, extra=0.0):
    """NaN where the definition has NaN, and elsewhere within ``u |out| + 2^-10 sum p |v|
    + extra``, the bound of :mod:`tests.test_int4_gpu`."""
    got = got.double().cpu().numpy()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    over = np.abs(got - want) - (ROUND[dtype] * np.abs(want) + 2.0 ** -10 * weight + extra)
    assert nan.all() or over[~nan].max() <= 0, f"outside the bound by {over[~nan].max():.3g}"


# ------------------------------------------------------------ NaN among drafts

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,nq", [(64, 4), (64, 12), (128, 4), (128, 14)])
def test_draft_nan_value_stays_in_its_channels(dtype, D, nq):
    """Drafted tokens whose Value groups do not fit (a NaN; a range past 15 * 65504):
    the queries that see one are NaN in that group's 32 channels and nowhere else, in
    sequences with all and with some of the query tokens."""
    lengths, L, H = [70, 97, 66, 130], 4, 2
    pages, table, _, sk, sv = _filled(1, lengths, H, D, dtype=dtype)
    value = torch.randn(4, H, 3, D, generator=torch.Generator().manual_seed(5))
    value[0, :, 1, 40] = float("nan")     # the last but one token, group 1, both KV heads
    value[1, 0, 2, 3] = float("nan")      # the last token, group 0, KV head 0
    value[1, 1, 0, 63] = float("-inf")
    value[2, 1, 1, 33] = 3e6
    key = torch.randn(4, H, 3, D, generator=torch.Generator().manual_seed(6))
    int4.int4_write(key.cuda(), value.cuda(), pages, table, _i32([n - 3 for n in lengths]))
    rows = [np.arange(n - 3, n) for n in lengths]
    wk, wv = ref.stored(key.double().numpy()), ref.stored(value.double().numpy())
    for b in range(4):
        sk[b][:, rows[b]], sv[b][:, rows[b]] = wk[b], wv[b]
    assert np.isnan(sv).any()
    q = _queries(2, 4, nq, L, D, dtype)
    for counts in ([L] * 4, [3, L, 2, 1]):
        got = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5, counts=_i32(counts))
        want, weight = _dense_reference(q, lengths, counts, sk, sv, D ** -0.5)
        assert np.isnan(want).any() and np.isfinite(want).any()
        _check(got, want, np.nan_to_num(weight), dtype, 2.0 ** -24)


def test_sparse_over_every_page_has_the_dense_result_with_nan_drafts():
    lengths, L, D = [70, 200], 3, 64
    pages, table, bounds, _, _ = _filled(1, lengths, 1, D)
    value = torch.zeros(2, 1, 2, D, device="cuda")
    value[..., 1, 7] = float("nan")
    int4.int4_write(torch.zeros_like(value), value, pages, table, _i32([n - 2 for n in lengths]), bounds=bounds)
    q = _queries(0, 2, 4, L, D)
    dense = int4.int4_attention(q, pages, table, _i32(lengths), 0.125)
    sparse, _ = int4.int4_sparse_attention(q, pages, bounds, table, _i32(lengths), 0.125, top_pages=4)
    assert torch.equal(torch.isnan(dense), torch.isnan(sparse))
    assert bool(torch.isnan(dense[:, :, 2, :32]).all()) and bool(torch.isfinite(dense[..., 32:]).all())


# ---------------------------------------------------------------- small weights

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,H,nq,D", [(1, 2, 8, 128), (96, 4, 4, 64), (80, 4, 48, 128)])
@pytest.mark.parametrize("gap", [9.0, 12.0, 15.0, 18.0])
def test_weights_far_below_a_dominant_token(dtype, B, H, nq, D, gap):
    """A first token with a score ``gap`` above the mean of the others' and a Value of
    zero, so that the output is the sum of small weights; in units split over many CTAs
    and in units that one CTA takes whole.

    A weight is held in fp16 with its warp's largest at 2^7 at least: to 2^-11 of itself,
    or to 2^-25 where it is subnormal, which is 2^-32 of the largest weight.  The
    second is bounded by T 2^-32 max p max |v|."""
    T = 700
    g = torch.Generator().manual_seed(int(gap))
    key, value = torch.randn(B, H, T, D, generator=g), 100.0 * (2.0 + torch.randn(B, H, T, D, generator=g))
    q = torch.randn(B, nq, 1, D, generator=g)
    key[..., 0], q[..., 0] = 0.0, 4.0
    key[:, :, 0], value[:, :, 0] = 0.0, 0.0
    key[:, :, 0, 0] = gap * D ** 0.5 / 4.0
    key, value, q = key.to(dtype).cuda(), value.to(dtype).cuda(), q.to(dtype).cuda()
    table, n = _table(3, B, 11)
    pages = _garbage(n, H, D)
    int4.int4_write(key, value, pages, table, _i32([0] * B))
    sk, sv = ref.stored(key.double().cpu().numpy()), ref.stored(value.double().cpu().numpy())
    got = int4.int4_attention(q, pages, table, _i32([T] * B), D ** -0.5)
    some = list(range(0, B, 7))   # of a large batch, sequences enough
    want, weight = _dense_reference(q[some], [T] * len(some), [1] * len(some), sk[some], sv[some], D ** -0.5)
    _check(got[some], want, weight, dtype, T * 2.0 ** -32 * np.abs(sv).max())


# ----------------------------------------------------------------- large Values

@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,nq,L", [(64, 4, 1), (64, 12, 3), (128, 4, 1), (128, 14, 3)])
@pytest.mark.parametrize("first", [0, 400])
def test_values_past_the_fp16_range_beside_small_ones(dtype, D, nq, L, first):
    """Value groups of magnitude 4e4 (and, for bf16 outputs, 6e5) from token ``first`` on,
    in some channels of some tokens, beside groups of magnitude 2e-4."""
    T, H = 600, 2
    g = torch.Generator().manual_seed(D + nq)
    key, value = torch.randn(1, H, T, D, generator=g), torch.randn(1, H, T, D, generator=g) * 2e-4
    low, high = (-4e4, 4e4) if dtype == F16 else (-6e4, 6e5)   # the minimum has to fit fp16, the range 15 times that
    value[:, 0, first::5, 32:64] = low + torch.rand(1, len(range(first, T, 5)), 32, generator=g) * (high - low)
    value[:, 1, first + 1::64, :32] = 3.5e4 + torch.rand(1, len(range(first + 1, T, 64)), 32, generator=g)
    value[:, :, T - 2, :32] = -4e4   # among the drafts
    key, value = key.cuda(), value.cuda()
    table, n = _table(1, 1, 10)
    pages, bounds = _garbage(n, H, D), int4.alloc_bounds(n, H, D)
    int4.int4_write(key, value, pages, table, _i32([0]), bounds=bounds)
    sk, sv = ref.stored(key.double().cpu().numpy()), ref.stored(value.double().cpu().numpy())
    assert np.abs(sv).max() > 32768
    q = 3 * _queries(1, 1, nq, L, D, dtype)
    got = int4.int4_attention(q, pages, table, _i32([T]), D ** -0.5)
    _check(got, *_dense_reference(q, [T], [L], sk, sv, D ** -0.5), dtype, 2.0 ** -24)
    got, picked = int4.int4_sparse_attention(q, pages, bounds, table, _i32([T]), D ** -0.5, top_pages=2, sink_pages=1, recent_pages=1)
    _check(got, *_dense_reference(q, [T], [L], sk, sv, D ** -0.5, picked.cpu().numpy()), dtype, 2.0 ** -24)


@pytest.mark.parametrize("D", [64, 128])
def test_a_masked_large_value_changes_nothing(D):
    """The slots past the length hold Values of 5e4, the seen ones 2e-4."""
    T, H = 100, 1
    g = torch.Generator().manual_seed(1)
    key, value = torch.randn(1, H, 128, D, generator=g).cuda(), (torch.randn(1, H, 128, D, generator=g) * 2e-4).cuda()
    value[:, :, T:] = 5e4
    table, n = _table(1, 1, 2)
    pages = _garbage(n, H, D)
    int4.int4_write(key, value, pages, table, _i32([0]))
    sk, sv = ref.stored(key.double().cpu().numpy()), ref.stored(value.double().cpu().numpy())
    q = _queries(1, 1, 5, 2, D)
    got = int4.int4_attention(q, pages, table, _i32([T]), D ** -0.5)
    _check(got, *_dense_reference(q, [T], [2], sk, sv, D ** -0.5), BF16, 2.0 ** -24)


# ------------------------------------------------------------ negative scalings

@pytest.mark.parametrize("D,nq,H", [(128, 28, 4), (64, 8, 8)])
def test_sparse_with_a_negative_scaling(D, nq, H):
    """The pages with the largest bound on scaling * q . K: those of the negated query."""
    lengths, L = [1500, 64 * 9, 130], 2
    pages, table, bounds, sk, sv = _filled(7, lengths, H, D)
    q = _queries(1, 3, nq, L, D)
    got, picked = int4.int4_sparse_attention(q, pages, bounds, table, _i32(lengths), -D ** -0.5, 4, 1, 2)
    want = _picks(-q, sk, lengths, [L] * 3, 4, 1, 2)
    assert np.array_equal(picked.cpu().numpy(), want)
    _check(got, *_dense_reference(q, lengths, [L] * 3, sk, sv, -D ** -0.5, want), BF16, 2.0 ** -24)
    flipped, same = int4.int4_sparse_attention(-q, pages, bounds, table, _i32(lengths), D ** -0.5, 4, 1, 2)
    assert torch.equal(same, picked) and torch.equal(flipped, got)


# ------------------------------------------------------------ empty pools

def test_pools_without_pages_heads_or_sequences_are_refused():
    pages, bounds = int4.alloc_pages(4, 2, 64), int4.alloc_bounds(4, 2, 64)
    table, n = _i32([[0, 1], [2, 3]]), _i32([5, 5])
    q = torch.zeros(2, 4, 64, dtype=BF16, device="cuda")
    for p, b, t, m, x in ((pages[:, :0], bounds[:, :0], table, n, q), (pages[:0], bounds[:0], table, n, q),
                          (pages[..., :0], bounds, table, n, q), (pages, bounds, table[:, :0], n, q),
                          (pages, bounds, table[:0], n[:0], q[:0])):
        for call in (lambda: int4.int4_attention(x, p, t, m, 1.0), lambda: int4.int4_select(x, p, b, t, m, 4),
                     lambda: int4.int4_sparse_attention(x, p, b, t, m, 1.0, 4), lambda: int4.int4_read(p, t, m, 3)):
            with pytest.raises(ValueError):
                call()


# ------------------------------------------------------------ negative positions

@pytest.mark.parametrize("start", [-10, -64, -70, -300])
def test_read_from_a_negative_position(start):
    """Positions below 0 are zeros and reported; those from 0 on are read."""
    D, T = 64, 150
    pages, table, _, sk, sv = _filled(1, [T], 2, D)
    status = _i32([0])
    k, v = int4.int4_read(pages, table, _i32([start]), T - start, status=status)
    assert int(status) != 0
    assert not k[:, :, :-start].any() and not v[:, :, :-start].any()
    assert np.array_equal(k[:, :, -start:].cpu().numpy(), sk) and np.array_equal(v[:, :, -start:].cpu().numpy(), sv)


# ------------------------------------------------------------ magnitudes of queries

@pytest.mark.parametrize("D,nq", [(64, 3), (128, 14)])
def test_queries_of_any_magnitude(D, nq):
    """bf16 queries near both ends of their range."""
    lengths = [300]
    pages, table, _, sk, sv = _filled(1, lengths, 1, D)
    for scale in (2.0 ** 118, 2.0 ** 100, 2.0 ** -60, 2.0 ** -120):
        q = (_queries(1, 1, nq, 1, D).float() * scale).to(BF16)
        got = int4.int4_attention(q, pages, table, _i32(lengths), 0.125 / scale)
        want, weight = _dense_reference(q, lengths, [1], sk, sv, 0.125 / scale)
        S = float(np.abs(q.double().cpu().numpy()).sum(-1).max() * np.abs(sk).max() * 0.125 / scale)
        _check(got, want, weight * (1.0 + S * 2.0 ** -10), BF16, 2.0 ** -24)


@pytest.mark.parametrize("D,nq", [(64, 3), (128, 14)])
def test_scores_that_are_all_far_below_zero(D, nq):
    """Every score near -1e34: the nearest to zero takes all the weight."""
    T = 300
    g = torch.Generator().manual_seed(D)
    key, value = torch.rand(1, 1, T, D, generator=g).cuda() + 0.5, torch.randn(1, 1, T, D, generator=g).cuda()
    table, n = _table(1, 1, 5)
    pages = _garbage(n, 1, D)
    int4.int4_write(key, value, pages, table, _i32([0]))
    sk, sv = ref.stored(key.double().cpu().numpy()), ref.stored(value.double().cpu().numpy())
    q = (-(torch.rand(1, nq, 1, D, generator=g) + 0.5) * 2.0 ** 110).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32([T]), 0.125)
    _check(got, *_dense_reference(q, [T], [1], sk, sv, 0.125), BF16, 2.0 ** -24)


# ------------------------------------------------------------ shared pages

@pytest.mark.parametrize("q_len", [1, 3])
def test_sequences_that_share_a_prefix(q_len):
    """Two sequences whose first pages are the same pool pages, each with its own tail."""
    D, H, nq, shared, lengths = 128, 2, 14, 5, [5 * 64 + 70, 5 * 64 + 9]
    table, n = _table(2, 2, 7)
    table[1, :shared] = table[0, :shared]
    pages, bounds = _garbage(n, H, D), int4.alloc_bounds(n, H, D)
    k, v = _kv(3, 2, H, max(lengths), D)
    k[1, :, :shared * 64], v[1, :, :shared * 64] = k[0, :, :shared * 64], v[0, :, :shared * 64]
    # the prefix through one of its owners, then both tails
    int4.int4_write(k[:1, :, :shared * 64], v[:1, :, :shared * 64], pages, table[:1], _i32([0]), bounds=bounds)
    int4.int4_write(k[:, :, shared * 64:], v[:, :, shared * 64:], pages, table, _i32([shared * 64] * 2),
                    _i32([m - shared * 64 for m in lengths]), bounds=bounds)
    sk, sv = ref.stored(k.double().cpu().numpy()), ref.stored(v.double().cpu().numpy())
    gk, gv = int4.int4_read(pages, table, _i32([0, 0]), min(lengths))
    assert np.array_equal(gk.cpu().numpy(), sk[:, :, :min(lengths)]) and np.array_equal(gv.cpu().numpy(), sv[:, :, :min(lengths)])
    q = _queries(1, 2, nq, q_len, D)
    got = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5)
    _check(got, *_dense_reference(q, lengths, [q_len] * 2, sk, sv, D ** -0.5), BF16, 2.0 ** -24)
    got, picked = int4.int4_sparse_attention(q, pages, bounds, table, _i32(lengths), D ** -0.5, 2, 1, 1)
    want = _picks(q, sk, lengths, [q_len] * 2, 2, 1, 1)
    assert np.array_equal(picked.cpu().numpy(), want)
    _check(got, *_dense_reference(q, lengths, [q_len] * 2, sk, sv, D ** -0.5, want), BF16, 2.0 ** -24)
