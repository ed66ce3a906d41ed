"""GPU tests of the 4-bit paged cache against its definition in 64 bits
(:mod:`tests.int4_reference`).

What is written is compared bit for bit.  Attention outputs are compared
element by element within ``u |out| + 2^-10 sum p |v|``: u is the output
type's rounding (2^-8 bf16, 2^-11 fp16), and the second term covers the
softmax weights' rounding to fp16 (2^-11 each), the exponential's 2^-22 and the
scores' fp32 sums.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from logitfill_b200 import int4
from tests import int4_reference as ref

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _kv(seed, *shape, dtype=BF16, outliers=True):
    g = torch.Generator().manual_seed(seed)
    k, v = torch.randn(*shape, generator=g), torch.randn(*shape, generator=g)
    if outliers:
        k[..., ::19] *= 8.0
        k += torch.randn(*shape[:-2], shape[-2] // 100 + 1, shape[-1], generator=g).repeat_interleave(100, -2)[..., :shape[-2], :]
    return k.to(dtype).cuda(), v.to(dtype).cuda()


def _table(seed, batch, width, extra=3):
    """A shuffled page table over a pool with some pages nobody owns."""
    g = torch.Generator().manual_seed(seed)
    n = batch * width + extra
    return torch.randperm(n, generator=g)[:batch * width].to(torch.int32).view(batch, width).cuda(), n


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _garbage(n, H, D):
    """A pool whose every bit is set: codes 15, parameters NaN."""
    return torch.full((n, H, 20 * D), -1, dtype=torch.int32, device="cuda")


def _filled(seed, lengths, H, D, dtype=BF16, bounds=True):
    """A pool holding random sequences, and the stored Key/Value per sequence."""
    B, T = len(lengths), max(max(lengths), 1)
    table, n = _table(seed, B, -(-T // 64))
    pages = _garbage(n, H, D)
    bnd = int4.alloc_bounds(n, H, D) if bounds else None
    k, v = _kv(seed, B, H, T, D, dtype=dtype)
    int4.int4_write(k, v, pages, table, _i32([0] * B), _i32(lengths), bnd)
    sk, sv = ref.stored(k.double().cpu().numpy()), ref.stored(v.double().cpu().numpy())
    return pages, table, bnd, sk, sv


def _check_out(got, want, weight, dtype):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    bound = ROUND[dtype] * np.abs(want) + 2.0 ** -10 * weight + 2.0 ** -24
    worst = float((np.abs(got - want) - bound).max())
    assert worst <= 0, f"outside the bound by {worst:.3g} (largest error {np.abs(got - want).max():.3g})"


# ------------------------------------------------------------ write and read

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,start", [(1, 0), (1, 63), (5, 61), (64, 0), (64, 1), (191, 130), (300, 7)])
def test_write_then_read_is_the_definition(D, dtype, T, start):
    B, H = 2, 3
    starts = [start, start + 11]
    table, n = _table(T, B, -(-(max(starts) + T) // 64))
    pages, bounds = _garbage(n, H, D), int4.alloc_bounds(n, H, D)
    k, v = _kv(T + start, B, H, T, D, dtype=dtype)
    int4.int4_write(k, v, pages, table, _i32(starts), bounds=bounds)
    gk, gv = int4.int4_read(pages, table, _i32(starts), T)
    wk, wv = ref.stored(k.double().cpu().numpy()), ref.stored(v.double().cpu().numpy())
    assert np.array_equal(gk.cpu().numpy(), wk) and np.array_equal(gv.cpu().numpy(), wv)
    for out in (BF16, F16):
        rk, rv = int4.int4_read(pages, table, _i32(starts), T, dtype=out)
        assert torch.equal(rk, gk.to(out)) and torch.equal(rv, gv.to(out))
    # nothing else in the pool was touched
    used = {int(table[b, p]) for b in range(B) for p in range(starts[b] // 64, (starts[b] + T - 1) // 64 + 1)}
    idle = [p for p in range(n) if p not in used]
    assert bool((pages[idle] == -1).all())


@pytest.mark.parametrize("D", [64, 128])
def test_record_layout_and_bounds(D):
    H, T = 2, 130
    pages, table, bounds, sk, sv = _filled(5, [T], H, D)
    rec = pages.cpu().numpy()
    vals = int4.int4_read_bounds(bounds).cpu().numpy()
    raw = bounds.cpu().numpy()
    for h in range(H):
        for p in range(3):
            at, rows = int(table[0, p]), min(64, T - 64 * p)
            k, v = ref.record_values(rec[at, h], D)
            assert np.array_equal(k[:rows], sk[0, h, 64 * p:64 * p + rows])
            assert np.array_equal(v[:rows], sv[0, h, 64 * p:64 * p + rows])
            if rows < 64:
                assert not raw[at, h].any()   # an incomplete page has no record
                continue
            up, low, e = ref.page_bounds(k)
            assert np.array_equal(raw[at, h, :D], up) and np.array_equal(raw[at, h, D:2 * D], low)
            assert raw[at, h, 2 * D] == e
            assert np.array_equal(vals[at, h, 0], up * 2.0 ** e) and np.array_equal(vals[at, h, 1], low * 2.0 ** e)
            assert (vals[at, h, 0] >= k.max(0)).all() and (vals[at, h, 1] <= k.min(0)).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("parts", [[40, 24], [1] * 64, [63, 1, 70], [130, 3, 59]])
def test_pieces_give_the_pages_of_one_write(D, parts):
    """Tokens written in pieces, as decode steps do, leave the same records and
    bounds as one write."""
    B, H, T = 2, 2, sum(parts)
    k, v = _kv(9, B, H, T, D)
    table, n = _table(1, B, -(-T // 64))
    whole, wb = _garbage(n, H, D), int4.alloc_bounds(n, H, D)
    int4.int4_write(k, v, whole, table, _i32([0, 0]), bounds=wb)
    pages, bounds = _garbage(n, H, D), int4.alloc_bounds(n, H, D)
    at = 0
    for m in parts:
        int4.int4_write(k[:, :, at:at + m], v[:, :, at:at + m], pages, table, _i32([at, at]), bounds=bounds)
        at += m
    assert torch.equal(pages, whole) and torch.equal(bounds, wb)


def test_special_values():
    """Constant groups, zeros, tiny and large magnitudes, and groups that hold a
    NaN, an infinity or a range past 15 fp16 steps (which read back as NaN)."""
    D, H = 128, 1
    rows = torch.zeros(11, D, dtype=F32)
    rows[0] = 3.25
    rows[2] = torch.linspace(-1, 1, D) * 1e-7
    rows[3] = torch.linspace(-6e4, 6e4, D)
    rows[4] = torch.randn(D, generator=torch.Generator().manual_seed(0))
    rows[4, 7] = float("nan")
    rows[5] = 1.0
    rows[5, 40] = float("inf")
    rows[6] = 1.0
    rows[6, 70] = -float("inf")
    rows[7, 100] = 7e5
    rows[8] = -0.0
    rows[9] = torch.linspace(1.0, 1.0 + 1e-6, D)
    rows[10, 100] = 2e6
    x = rows.view(1, 1, 11, D).cuda()
    table, n = _table(0, 1, 1)
    pages, bounds = _garbage(n, H, D), int4.alloc_bounds(n, H, D)
    int4.int4_write(x, x, pages, table, _i32([0]), bounds=bounds)
    k, v = int4.int4_read(pages, table, _i32([0]), 11)
    want = ref.stored(rows.double().numpy())[None, None]
    assert np.array_equal(k.cpu().numpy(), want, equal_nan=True) and np.array_equal(v.cpu().numpy(), want, equal_nan=True)
    nan = np.isnan(want[0, 0]).reshape(11, 4, 32).all(-1)
    assert nan.sum() == 4 and nan[4, 0] and nan[5, 1] and nan[6, 2] and nan[10, 3]


@pytest.mark.parametrize("dtype", [F16, F32])
def test_groups_of_nearly_equal_values(dtype):
    """Ranges of a few fp16 roundings of the minimum: x - z is then far from x - min,
    codes pass 15 before the clamp and fall below 0."""
    D, T = 64, 128
    g = torch.Generator().manual_seed(0)
    base = torch.rand(T, 2, generator=g).repeat_interleave(32, 1) * 200 - 100
    x = (base + torch.rand(T, D, generator=g) * torch.logspace(-4, 0.5, T).view(T, 1)).to(dtype).view(1, 1, T, D).cuda()
    table, n = _table(0, 1, 2)
    pages, bounds = _garbage(n, 1, D), int4.alloc_bounds(n, 1, D)
    int4.int4_write(x, -x, pages, table, _i32([0]), bounds=bounds)
    k, v = int4.int4_read(pages, table, _i32([0]), T)
    assert np.array_equal(k.cpu().numpy(), ref.stored(x.double().cpu().numpy()))
    assert np.array_equal(v.cpu().numpy(), ref.stored(-x.double().cpu().numpy()))


def test_bounds_of_pages_with_nan_and_zeros():
    D, H = 64, 1
    k = torch.randn(1, H, 128, D, generator=torch.Generator().manual_seed(3)).cuda()
    k[:, :, :64, 32:] = 0.0
    k[0, 0, 5, 3] = float("nan")
    k[:, :, 64:] = 0.0
    table, n = _table(0, 1, 2)
    pages, bounds = _garbage(n, H, D), int4.alloc_bounds(n, H, D)
    int4.int4_write(k, k, pages, table, _i32([0]), bounds=bounds)
    stored = ref.stored(k.double().cpu().numpy())[0, 0]
    for p in range(2):
        up, low, e = ref.page_bounds(stored[64 * p:64 * p + 64])
        raw = bounds[int(table[0, p]), 0].cpu().numpy()
        assert np.array_equal(raw[:D], up) and np.array_equal(raw[D:2 * D], low) and raw[2 * D] == e


@pytest.mark.parametrize("layout", ["token major", "channel strided", "misaligned", "broadcast", "separate"])
def test_write_takes_any_strides(layout):
    B, H, T, D = 2, 4, 70, 64
    k, v = _kv(2, B, H, T, D)
    if layout == "token major":
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    elif layout == "channel strided":
        k, v = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    elif layout == "misaligned":
        k, v = (torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape) for x in (k, v))
        assert k.data_ptr() % 16
    elif layout == "broadcast":
        k, v = (x[:1, :1].expand(B, H, T, D) for x in (k, v))
    else:
        v = v.transpose(1, 2).contiguous().transpose(1, 2)
    table, n = _table(4, B, 2)
    pages = _garbage(n, H, D)
    int4.int4_write(k, v, pages, table, _i32([3, 50]))
    gk, gv = int4.int4_read(pages, table, _i32([3, 50]), T)
    assert np.array_equal(gk.cpu().numpy(), ref.stored(k.double().cpu().numpy()))
    assert np.array_equal(gv.cpu().numpy(), ref.stored(v.double().cpu().numpy()))


def test_ragged_counts_and_out_of_range_pages():
    B, H, T, D = 4, 2, 100, 128
    k, v = _kv(8, B, H, T, D)
    table, n = _table(8, B, 2)
    table[3, 1] = n + 5                     # not a page of the pool
    table[2, 0] = -1
    pages = _garbage(n, H, D)
    counts, status = [100, 0, 37, 100], _i32([0])
    int4.int4_write(k, v, pages, table, _i32([0, 0, 0, 0]), _i32(counts), status=status)
    assert int(status) != 0                 # sequences 2 and 3 met pages outside the pool
    status.zero_()
    gk, _ = int4.int4_read(pages, table, _i32([0] * B), T, _i32(counts), status=status)
    assert int(status) != 0
    want = ref.stored(k.double().cpu().numpy())
    want[1] = 0
    want[2] = 0
    want[3, :, 64:] = 0
    assert np.array_equal(gk.cpu().numpy(), want)
    assert bool((pages[table[1].long()] == -1).all())
    status.zero_()
    int4.int4_write(k, v, pages, table, _i32([100, 100, 100, -7]), _i32([100, 0, 0, 100]), status=status)
    assert int(status) != 0                 # past the table, before position 0
    status.zero_()
    int4.int4_write(k[:, :, :0], v[:, :, :0], pages, table, _i32([0] * B), status=status)
    assert int(status) == 0
    assert int4.int4_read(pages, table, _i32([0] * B), 0)[0].shape == (B, H, 0, D)


# ------------------------------------------------------------------ attention

def _dense_reference(q, lengths, counts, sk, sv, scaling, picks=None):
    B, nq, L, D = q.shape
    H = sk.shape[1]
    q = q.double().cpu().numpy()
    out, weight = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        for i in range(L):
            seen = max(0, lengths[b] - counts[b] + 1 + i) if i < counts[b] else 0
            for h in range(H):
                rows = slice(h * (nq // H), (h + 1) * (nq // H))
                keep = np.arange(sk.shape[2]) < seen
                if picks is not None:
                    keep &= np.isin(np.arange(sk.shape[2]) // 64, [p for p in picks[b, i, h] if p >= 0])
                out[b, rows, i], weight[b, rows, i] = attention_of(q[b, rows, i], sk[b, h], sv[b, h], scaling, keep)
    return out, weight


attention_of = ref.attention


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq,H", [(28, 4), (40, 8), (1, 1), (16, 1), (9, 3), (34, 2)])
@pytest.mark.parametrize("q_len", [1, 4])
def test_attention_heads(D, nq, H, q_len):
    lengths = [1, 64, 65, 700, 3]
    pages, table, _, sk, sv = _filled(nq, lengths, H, D)
    q = torch.randn(5, nq, q_len, D, generator=torch.Generator().manual_seed(q_len)).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5)
    _check_out(got, *_dense_reference(q, lengths, [q_len] * 5, sk, sv, D ** -0.5), BF16)
    if q_len == 1:
        assert torch.equal(int4.int4_attention(q[:, :, 0], pages, table, _i32(lengths), D ** -0.5), got[:, :, 0])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths", [[0], [2], [63, 64, 65, 127, 128, 129], [5000, 0, 1], [20000], [4097] * 3])
def test_attention_lengths(dtype, lengths):
    B, D, nq, H, L = len(lengths), 128, 14, 2, 2
    pages, table, _, sk, sv = _filled(B, lengths, H, D, dtype=dtype)
    q = torch.randn(B, nq, L, D, generator=torch.Generator().manual_seed(0)).to(dtype).cuda()
    got = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5)
    _check_out(got, *_dense_reference(q, lengths, [L] * B, sk, sv, D ** -0.5), dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("nq", [3, 12])
def test_attention_of_one_long_unit(D, nq):
    # one KV head: its pages lie in more ranges than one round of the merge holds
    lengths = [30001]
    pages, table, _, sk, sv = _filled(D, lengths, 1, D)
    q = torch.randn(1, nq, 1, D, generator=torch.Generator().manual_seed(nq)).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5)
    _check_out(got, *_dense_reference(q, lengths, [1], sk, sv, D ** -0.5), BF16)


def test_attention_long_queries_and_many_sequences():
    lengths, nq, H, D, L = [150, 77, 300], 6, 2, 64, 75
    pages, table, _, sk, sv = _filled(3, lengths, H, D)
    q = torch.randn(3, nq, L, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5)
    _check_out(got, *_dense_reference(q, lengths, [L] * 3, sk, sv, D ** -0.5), BF16)
    lengths = [int(x) for x in np.random.default_rng(0).integers(0, 200, 300)]
    pages, table, _, sk, sv = _filled(4, lengths, 1, 64)
    q = torch.randn(300, 2, 1, 64, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32(lengths), 0.125)
    _check_out(got, *_dense_reference(q, lengths, [1] * 300, sk, sv, 0.125), BF16)


def test_attention_counts_give_each_sequence_its_own_queries():
    lengths, counts = [40, 200, 7, 64], [3, 0, 4, 1]
    pages, table, _, sk, sv = _filled(6, lengths, 2, 128)
    q = torch.randn(4, 8, 4, 128, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32(lengths), 0.1, counts=_i32(counts))
    want, weight = _dense_reference(q, lengths, counts, sk, sv, 0.1)
    _check_out(got, want, weight, BF16)
    assert not got[1].any() and not got[0, :, 3].any()


@pytest.mark.parametrize("scale_v,scale_q", [(1e-4, 1.0), (300.0, 1.0), (1.0, 60.0), (1.0, 1e-6)])
def test_attention_magnitudes(scale_v, scale_q):
    """Values from 1e-4 to 1e4, peaked and flat softmaxes, growing magnitudes."""
    D, nq, H, T = 128, 8, 2, 1000
    table, n = _table(0, 1, 16)
    pages = _garbage(n, H, D)
    k, v = _kv(7, 1, H, T, D, dtype=BF16)
    v = (v.float() * torch.logspace(-1, 1, T).view(1, 1, T, 1).cuda() * scale_v).to(BF16)
    int4.int4_write(k, v, pages, table, _i32([0]))
    sk, sv = ref.stored(k.double().cpu().numpy()), ref.stored(v.double().cpu().numpy())
    q = (torch.randn(1, nq, 1, D, generator=torch.Generator().manual_seed(0)) * scale_q).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32([T]), D ** -0.5)
    want, weight = _dense_reference(q, [T], [1], sk, sv, D ** -0.5)
    # a score of magnitude S carries fp32 sums' error of about S 2^-20
    S = float(np.abs(q.double().cpu().numpy()).sum(-1).max() * np.abs(sk).max() * D ** -0.5)
    got = got.double().cpu().numpy()
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -10 + S * 2.0 ** -20) * weight
    assert (np.abs(got - want) <= bound).all()


def test_attention_ignores_what_is_not_seen_and_spreads_what_is_nan():
    """Slots past the length hold NaN parameters (the pool starts as all ones);
    a NaN Value group makes its 32 channels NaN, a NaN Key the whole row."""
    D, T = 64, 100
    pages, table, _, sk, sv = _filled(1, [T], 1, D)
    q = torch.randn(1, 4, 1, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    clean = int4.int4_attention(q, pages, table, _i32([T]), 0.125)
    assert bool(torch.isfinite(clean).all())
    one = torch.zeros(1, 1, 1, D, dtype=BF16, device="cuda")
    bad = one.clone()
    bad[..., 40] = float("nan")
    int4.int4_write(one, bad, pages, table, _i32([T]))
    got = int4.int4_attention(q, pages, table, _i32([T + 1]), 0.125)
    assert bool(torch.isnan(got[..., 32:]).all()) and bool(torch.isfinite(got[..., :32]).all())
    assert torch.equal(int4.int4_attention(q, pages, table, _i32([T]), 0.125), clean)
    int4.int4_write(bad, one, pages, table, _i32([T]))
    assert bool(torch.isnan(int4.int4_attention(q, pages, table, _i32([T + 1]), 0.125)).all())


@pytest.mark.parametrize("scaling", [-0.125, 0.0, 1e-30, 5.0])
def test_attention_scaling_of_any_sign(scaling):
    lengths, D = [130, 500], 64
    pages, table, _, sk, sv = _filled(4, lengths, 2, D, dtype=F16)
    q = torch.randn(2, 4, 3, D, generator=torch.Generator().manual_seed(0)).to(F16).cuda()
    got = int4.int4_attention(q, pages, table, _i32(lengths), scaling).double().cpu().numpy()
    want, weight = _dense_reference(q, lengths, [3, 3], sk, sv, scaling)
    # a score of magnitude S carries fp32 sums' error of about S 2^-20
    S = float(np.abs(q.double().cpu().numpy()).sum(-1).max() * np.abs(sk).max() * abs(scaling))
    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + (2.0 ** -10 + S * 2.0 ** -20) * weight + 2.0 ** -24).all()


def test_attention_draft_nan_reaches_only_the_queries_that_see_it():
    """Drafted tokens 2 and 3 of 4 hold NaN (in Value, in Key): queries 0 and 1 stay
    clean, the others are NaN in every channel that sees it."""
    D, T, L = 128, 70, 4
    for which in ("value", "key"):
        pages, table, _, sk, sv = _filled(1, [T], 2, D)
        q = torch.randn(1, 6, L, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
        clean = int4.int4_attention(q, pages, table, _i32([T]), 0.1)
        ok = torch.zeros(1, 2, 2, D, dtype=BF16, device="cuda")
        bad = ok.clone()
        bad[..., 40] = float("nan")
        int4.int4_write(bad if which == "key" else ok, bad if which == "value" else ok, pages, table, _i32([T - 2]))
        got = int4.int4_attention(q, pages, table, _i32([T]), 0.1)
        assert torch.equal(got[:, :, :2], clean[:, :, :2])
        assert bool(torch.isnan(got[:, :, 2:, 32:64]).all())
        if which == "key":
            assert bool(torch.isnan(got[:, :, 2:]).all())


def test_attention_is_repeatable_and_takes_strides_and_outputs():
    lengths, D = [3000, 129], 128
    pages, table, _, sk, sv = _filled(2, lengths, 4, D)
    q = torch.randn(2, 28, 2, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    first = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5)
    for _ in range(5):
        assert torch.equal(int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5), first)
    strided = q.transpose(1, 2).contiguous().transpose(1, 2)
    buf = torch.zeros(2, 2, 28, D, dtype=BF16, device="cuda").transpose(1, 2)
    assert torch.equal(int4.int4_attention(strided, pages, table, _i32(lengths), D ** -0.5, out=buf), first)
    other = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(int4.int4_attention(other, pages, table, _i32(lengths), D ** -0.5), first)
    # a pool that is a slice of a larger one, per layer
    big = torch.zeros(pages.shape[0], 2, *pages.shape[1:], dtype=torch.int32, device="cuda")
    big[:, 1] = pages
    assert torch.equal(int4.int4_attention(q, big[:, 1], table, _i32(lengths), D ** -0.5), first)


def test_attention_out_of_range_pages_are_skipped():
    D, lengths = 64, [200, 300]
    pages, table, _, sk, sv = _filled(2, lengths, 1, D)
    table[0, 1] = 10 ** 6
    q = torch.randn(2, 4, 1, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    status = _i32([0])
    got = int4.int4_attention(q, pages, table, _i32([200, 2000]), 0.125, status=status)
    assert int(status) != 0
    keep = np.zeros((2, 1, 1, 5), np.int64)
    keep[0] = [0, 2, 3, -1, -1]
    keep[1] = [0, 1, 2, 3, 4]
    picks = keep
    # sequence 1 claims more tokens than its table has pages: the pages it has are
    # attended in full, slots past its 300 tokens included
    got = int4.int4_attention(q[:1], pages, table[:1], _i32([200]), 0.125, status=status)
    want, weight = _dense_reference(q[:1], [200], [1], sk[:1], sv[:1], 0.125, picks[:1])
    _check_out(got, want, weight, BF16)


def test_streams_and_graph_replay():
    """On a side stream next to work on the default one, and replayed from a
    CUDA graph with new inputs in place."""
    lengths, D = [2500, 700], 128
    pages, table, bounds, sk, sv = _filled(11, lengths, 4, D)
    q = torch.randn(2, 28, 1, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    n = _i32(lengths)
    want = int4.int4_attention(q, pages, table, n, D ** -0.5)
    ws, wp = int4.int4_sparse_attention(q, pages, bounds, table, n, D ** -0.5, top_pages=5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = [int4.int4_attention(q, pages, table, n, D ** -0.5) for _ in range(3)]
    b = [int4.int4_attention(q, pages, table, n, D ** -0.5) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in a + b)
    graph = torch.cuda.CUDAGraph()
    static = torch.zeros_like(q)
    with torch.cuda.graph(graph):
        out = int4.int4_attention(static, pages, table, n, D ** -0.5)
        sparse, picked = int4.int4_sparse_attention(static, pages, bounds, table, n, D ** -0.5, top_pages=5)
    for _ in range(2):
        static.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(sparse, ws) and torch.equal(picked, wp)


def test_pool_past_32_bit_offsets():
    """Records whose word offset passes 2^31."""
    D, H = 128, 1
    n = 2 ** 31 // (20 * D) + 40
    pages = torch.empty(n, H, 20 * D, dtype=torch.int32, device="cuda")
    bounds = int4.alloc_bounds(n, H, D)
    table = _i32([[n - 1, 3, n - 2, n - 7, n - 9]])
    k, v = _kv(1, 1, H, 300, D)
    int4.int4_write(k, v, pages, table, _i32([0]), bounds=bounds)
    gk, gv = int4.int4_read(pages, table, _i32([0]), 300)
    sk, sv = ref.stored(k.double().cpu().numpy()), ref.stored(v.double().cpu().numpy())
    assert np.array_equal(gk.cpu().numpy(), sk) and np.array_equal(gv.cpu().numpy(), sv)
    q = torch.randn(1, 7, 1, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    got = int4.int4_attention(q, pages, table, _i32([300]), D ** -0.5)
    _check_out(got, *_dense_reference(q, [300], [1], sk, sv, D ** -0.5), BF16)
    _, picked = int4.int4_sparse_attention(q, pages, bounds, table, _i32([300]), D ** -0.5, 1, 1, 1)
    assert picked[0, 0, 0].tolist() == ref.choose(q[0, :, 0].double().cpu().numpy(), sk[0, 0], 300, 1, 1, 1)


# --------------------------------------------------------------------- sparse

def _picks(q, sk, lengths, counts, top, sink, recent):
    B, nq, L, _ = q.shape
    H = sk.shape[1]
    q = q.double().cpu().numpy()
    out = np.zeros((B, L, H, top + sink + recent), np.int64)
    for b in range(B):
        for i in range(L):
            seen = max(0, lengths[b] - counts[b] + 1 + i) if i < counts[b] else 0
            for h in range(H):
                rows = slice(h * (nq // H), (h + 1) * (nq // H))
                out[b, i, h] = ref.choose(q[b, rows, i], sk[b, h], seen, top, sink, recent)
    return out


@pytest.mark.parametrize("D,nq,H", [(128, 28, 4), (64, 8, 8), (128, 16, 1)])
@pytest.mark.parametrize("top,sink,recent", [(4, 1, 2), (1, 0, 1), (0, 2, 1), (13, 0, 4)])
def test_sparse_pages_and_output(D, nq, H, top, sink, recent):
    lengths, L = [1500, 64 * 9, 130, 0, 1217], 2
    pages, table, bounds, sk, sv = _filled(top, lengths, H, D)
    q = torch.randn(5, nq, L, D, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    got, picked = int4.int4_sparse_attention(q, pages, bounds, table, _i32(lengths), D ** -0.5, top, sink, recent)
    want = _picks(q, sk, lengths, [L] * 5, top, sink, recent)
    assert np.array_equal(picked.cpu().numpy(), want)
    _check_out(got, *_dense_reference(q, lengths, [L] * 5, sk, sv, D ** -0.5, want), BF16)


def test_sparse_ties_go_to_the_lower_page():
    """Pages with the same Key have the same score; a query of zeros ties all."""
    D, T = 64, 64 * 40
    k, v = _kv(3, 1, 1, 64, D)
    k2, _ = _kv(4, 1, 1, 64, D)
    key = torch.cat([k2 if p % 3 == 1 else k for p in range(40)], 2)
    value = v.repeat(1, 1, 40, 1)
    table, n = _table(0, 1, 40)
    pages, bounds = _garbage(n, 1, D), int4.alloc_bounds(n, 1, D)
    int4.int4_write(key, value, pages, table, _i32([0]), bounds=bounds)
    sk = ref.stored(key.double().cpu().numpy())
    for q in (torch.zeros(1, 4, 1, D), torch.randn(1, 4, 1, D, generator=torch.Generator().manual_seed(0))):
        q = q.to(BF16).cuda()
        for top in (1, 5, 16, 30):
            picked = int4.int4_select(q, pages, bounds, table, _i32([T]), top, 1, 2)
            assert picked[0, 0, 0].tolist() == ref.choose(q[0, :, 0].double().cpu().numpy(), sk[0, 0], T, top, 1, 2)


@pytest.mark.parametrize("top", [1, 37, 600, 1500])
def test_sparse_long_sequences(top):
    D, T, H = 64, 64 * 1600 + 5, 1
    g = torch.Generator().manual_seed(2)
    k = torch.randn(1, H, T, D, generator=g).to(F16).cuda()
    table, n = _table(0, 1, 1601)
    pages, bounds = int4.alloc_pages(n, H, D), int4.alloc_bounds(n, H, D)
    int4.int4_write(k, k, pages, table, _i32([0]), bounds=bounds)
    q = torch.randn(1, 2, D, generator=g).to(F16).cuda()
    picked = int4.int4_select(q, pages, bounds, table, _i32([T]), top, 2, 3)
    raw = bounds[table[0].long(), 0].cpu().numpy().astype(np.int64)
    f = ref.exponent(float(q.abs().max()))
    Q = np.rint(q[0].double().cpu().numpy() / 2.0 ** f)
    total = raw[:, :D] @ np.maximum(Q, 0).sum(0).astype(np.int64) + raw[:, D:2 * D] @ np.minimum(Q, 0).sum(0).astype(np.int64)
    score = total.astype(np.float32) * np.exp2(raw[:, 2 * D]).astype(np.float32)
    order = np.argsort(-score[2:1598].astype(np.float64), kind="stable")[:top] + 2
    assert picked[0, 0, 0].tolist() == sorted([0, 1, *order.tolist(), 1598, 1599, 1600])


def test_sparse_with_a_large_budget_is_the_dense_result():
    lengths, D = [1000, 90, 5], 128
    pages, table, bounds, sk, sv = _filled(2, lengths, 2, D)
    q = torch.randn(3, 14, 3, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    dense = int4.int4_attention(q, pages, table, _i32(lengths), D ** -0.5)
    sparse, picked = int4.int4_sparse_attention(q, pages, bounds, table, _i32(lengths), D ** -0.5, top_pages=20)
    want, weight = _dense_reference(q, lengths, [3] * 3, sk, sv, D ** -0.5)
    _check_out(sparse, want, weight, BF16)
    _check_out(dense, want, weight, BF16)
    assert picked[0, 2, 0].tolist() == list(range(16)) + [-1] * 7


def test_sparse_query_with_nan_still_picks_pages():
    D, T = 64, 64 * 20
    pages, table, bounds, sk, sv = _filled(2, [T], 1, D)
    q = torch.randn(1, 2, 1, D, generator=torch.Generator().manual_seed(0)).to(BF16)
    q[0, 0, 0, 3], q[0, 1, 0, 9] = float("nan"), float("inf")
    picked = int4.int4_select(q.cuda(), pages, bounds, table, _i32([T]), 4)
    assert picked[0, 0, 0].tolist() == ref.choose(q[0, :, 0].double().numpy(), sk[0, 0], T, 4, 1, 2)


# ------------------------------------------------------------------ the cache

def test_cache_steps_match_plain_attention():
    """Prompts of unequal length, drafts, a rejected draft, a paused sequence and
    decode steps through the cache object, on two layers."""
    B, nq, H, D, layers = 3, 8, 2, 64, 2
    cache = int4.Int4KVCache(layers, B, nq, H, D, n_pages=40, max_tokens=64 * 12)
    g = torch.Generator().manual_seed(0)
    held = [[(np.zeros((H, 0, D), np.float32),) * 2 for _ in range(B)] for _ in range(layers)]

    def step(counts):
        T = max(counts)
        cache.extend(counts if len(set(counts)) > 1 else counts[0])
        for layer in range(layers):
            k, v = (torch.randn(B, T, H, D, generator=g).to(BF16).cuda().transpose(1, 2) for _ in range(2))
            cache.write(layer, k, v)
            for b in range(B):
                hk, hv = held[layer][b]
                held[layer][b] = (np.concatenate([hk, ref.stored(k[b, :, :counts[b]].double().cpu().numpy())], 1),
                                  np.concatenate([hv, ref.stored(v[b, :, :counts[b]].double().cpu().numpy())], 1))
            q = torch.randn(B, nq, T, D, generator=g).to(BF16).cuda()
            out = cache.attend(layer, q, D ** -0.5)
            sparse, picked = cache.attend_sparse(layer, q, D ** -0.5, top_pages=2, sink_pages=1, recent_pages=1)
            for b in range(B):
                hk, hv = held[layer][b]
                n = [hk.shape[1]]
                args = (n, [counts[b]], hk[None], hv[None], D ** -0.5)
                _check_out(out[b:b + 1], *_dense_reference(q[b:b + 1], *args), BF16)
                picks = _picks(q[b:b + 1], hk[None], n, [counts[b]], 2, 1, 1)
                assert np.array_equal(picked[b].cpu().numpy(), picks[0])
                _check_out(sparse[b:b + 1], *_dense_reference(q[b:b + 1], *args, picks), BF16)

    step([130, 700, 1])
    step([4, 4, 4])
    lengths = cache.lengths - [2, 0, 4]
    cache.truncate(lengths)
    for layer in range(layers):
        held[layer] = [(k[:, :lengths[b]], v[:, :lengths[b]]) for b, (k, v) in enumerate(held[layer])]
    for counts in ([1, 1, 1], [1, 0, 1], [1, 1, 1]):
        step(counts)
    gk, gv = cache.read(1)
    for b in range(B):
        n = int(cache.lengths[b])
        assert np.array_equal(gk[b, :, :n].cpu().numpy(), held[1][b][0]) and not gk[b, :, n:].any()
        assert np.array_equal(gv[b, :, :n].cpu().numpy(), held[1][b][1])
    cache.check_status()
    free = cache.free_pages
    cache.release([1])
    assert cache.free_pages == free + 12 and cache.lengths.tolist()[1] == 0
    held = [[(k[:, :0], v[:, :0]) if b == 1 else (k, v) for b, (k, v) in enumerate(layer)] for layer in held]
    step([1, 30, 1])
    cache.check_status()


def test_cache_step_in_a_graph():
    B, nq, H, D, T = 2, 4, 2, 128, 60
    caches = [int4.Int4KVCache(1, B, nq, H, D, n_pages=8, max_tokens=256) for _ in range(2)]
    k, v = _kv(0, B, H, T + 10, D)
    q = torch.randn(B, nq, 10, D, generator=torch.Generator().manual_seed(0)).to(BF16).cuda()
    for c in caches:
        c.extend(T)
        c.write(0, k[:, :, :T], v[:, :, :T])
        c.reserve(T + 10)
    eager, graphed = caches
    want = []
    for i in range(10):
        eager.extend(1)
        eager.write(0, k[:, :, T + i:T + i + 1], v[:, :, T + i:T + i + 1])
        want.append(eager.attend(0, q[:, :, i], 0.1))
    sk, sv, sq = torch.zeros_like(k[:, :, :1]), torch.zeros_like(k[:, :, :1]), torch.zeros_like(q[:, :, 0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.extend(1)
        graphed.write(0, sk, sv)
        out = graphed.attend(0, sq, 0.1)
    for i in range(10):
        sk.copy_(k[:, :, T + i:T + i + 1])
        sv.copy_(v[:, :, T + i:T + i + 1])
        sq.copy_(q[:, :, i])
        graph.replay()
        graphed.advance_host(1)
        assert torch.equal(out, want[i])
    assert torch.equal(graphed.pages[0][graphed.page_table.clamp(min=0).long()],
                       eager.pages[0][eager.page_table.clamp(min=0).long()])
    assert graphed.lengths.tolist() == [T + 10] * B
    graphed.check_status()


# ------------------------------------------------------------------- refusals

def test_refusals():
    D, H = 64, 2
    pages, bounds = int4.alloc_pages(4, H, D), int4.alloc_bounds(4, H, D)
    table, n = _i32([[0, 1], [2, 3]]), _i32([5, 5])
    k = torch.zeros(2, H, 5, D, dtype=BF16, device="cuda")
    q = torch.zeros(2, 4, D, dtype=BF16, device="cuda")

    def refuses(error, fn, *args, **kwargs):
        with pytest.raises(error):
            fn(*args, **kwargs)

    refuses(ValueError, int4.int4_write, k[:1], k[:1], pages, table, n)
    refuses(ValueError, int4.int4_write, k, k[:, :, :4], pages, table, n)
    refuses(ValueError, int4.int4_write, k, k.to(F16), pages, table, n)
    refuses(ValueError, int4.int4_write, k, k, pages.to(torch.int64), table, n)
    refuses(ValueError, int4.int4_write, k, k, pages, table.to(torch.int64), n)
    refuses(ValueError, int4.int4_write, k, k, pages, table, n.to(torch.int64))
    refuses(ValueError, int4.int4_write, k, k, pages, table, n, n[:1])
    refuses(ValueError, int4.int4_write, k, k, pages, table, n, bounds=bounds[:3])
    refuses(ValueError, int4.int4_write, k, k, pages, table, n, bounds=bounds.to(torch.int32))
    refuses(NotImplementedError, int4.int4_write, k.double(), k.double(), pages, table, n)
    refuses(RuntimeError, int4.int4_write, k.cpu(), k.cpu(), pages, table, n)
    refuses(RuntimeError, int4.int4_write, k, k, pages.cpu(), table, n)
    refuses(ValueError, int4.int4_write, k, k, pages[..., :-1], table, n)
    odd = torch.zeros(4, H, 20 * 96, dtype=torch.int32, device="cuda")
    k96 = torch.zeros(2, H, 5, 96, dtype=BF16, device="cuda")
    refuses(NotImplementedError, int4.int4_write, k96, k96, odd, table, n)
    refuses(NotImplementedError, int4.int4_read, odd, table, n, 3)
    refuses(ValueError, int4.int4_read, pages, table, n, -1)
    refuses(NotImplementedError, int4.int4_read, pages, table, n, 3, dtype=torch.int32)
    refuses(ValueError, int4.int4_attention, q[:, :3], pages, table, n, 1.0)
    refuses(ValueError, int4.int4_attention, q[:1], pages, table, n, 1.0)
    refuses(ValueError, int4.int4_attention, q[..., :32], pages, table, n, 1.0)
    refuses(NotImplementedError, int4.int4_attention, q.float(), pages, table, n, 1.0)
    refuses(RuntimeError, int4.int4_attention, q.cpu(), pages, table, n, 1.0)
    refuses(ValueError, int4.int4_attention, q, pages, table, n, 1.0, out=q.float())
    refuses(ValueError, int4.int4_attention, q, pages, table, n, 1.0, status=n.float())
    refuses(ValueError, int4.int4_attention, q, pages, table, n, float("nan"))
    refuses(ValueError, int4.int4_attention, q, pages, table, n, 1.0, out=torch.empty(2, 4, 66, dtype=BF16, device="cuda")[..., 1:65])
    refuses(ValueError, int4.int4_select, q, pages, bounds, table, n, 4, recent_pages=0)
    refuses(ValueError, int4.int4_select, q, pages, bounds, table, n, -1)
    refuses(ValueError, int4.int4_read_bounds, pages)
    refuses(NotImplementedError, int4.Int4KVCache, 1, 1, 4, 2, 96, 4, 64)
    refuses(ValueError, int4.Int4KVCache, 1, 1, 5, 2, 64, 4, 64)
    cache = int4.Int4KVCache(1, 2, 4, 2, 64, n_pages=3, max_tokens=128, bounds=False)
    refuses(ValueError, cache.extend, 129)
    refuses(RuntimeError, cache.extend, 65)       # four pages of three
    assert cache.free_pages == 3 and cache.lengths.tolist() == [0, 0]
    cache.extend([65, 3])
    refuses(ValueError, cache.extend, [-1, 0])
    refuses(ValueError, cache.truncate, 66)
    refuses(RuntimeError, cache.attend_sparse, 0, q, 1.0, 4)
    refuses(ValueError, cache.attend, 0, q[:, :2], 1.0)


def test_example_serves_dense_sparse_and_drafts():
    """The example's batch, decoded from the 4-bit cache and from uncompressed
    Key and Value side by side."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "int4_decode.py"
    spec = importlib.util.spec_from_file_location("int4_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for kwargs in (dict(), dict(draft=3), dict(top=40), dict(top=4)):
        apart, same, cache = example.serve([300, 1, 129, 64], steps=6, **kwargs)
        # every Key and Value element is within half a step (1/30 of its group's range, about 4
        # standard deviations): 8 % of an element's magnitude at most in root mean square
        assert apart < 0.16 and same > 0.5
        assert cache.lengths.tolist() == [n + 6 * kwargs.get("draft", 1) for n in (300, 1, 129, 64)]
