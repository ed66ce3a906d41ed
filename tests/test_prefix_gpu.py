"""GPU tests of attention over shared 4-bit pages (int4_prefix_attention) against its
formula in 64 bits, over the values that the pages hold (int4_read).

Element by element within  u |out| + (2^-10 + 2 e + 2^-16) sum p |v| + 2^-24: u is half a
step of the output's type; 2^-10 the weights and the Values, each rounded to fp16 (2^-11);
e what a score is off by: its Keys rounded to fp16, 2^-11 sum |q k| |scaling|, in a weight
and in the sum of weights; 2^-16 the exponential and the fp32 sums.
"""
from __future__ import annotations

import math

import pytest
import torch

from logitfill_b200 import int4

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Batch:
    """Sequences over one pool: `group[b]` (-1: none), `shared[g]` pages that a group has in
    common, `tails[b]` tokens of each behind them."""

    def __init__(self, seed, group, shared, tails, H, D, dtype=BF16, spare=2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.group, self.shared, self.H, self.D, self.dtype = group, shared, H, D, dtype
        B = len(group)
        self.lengths = [64 * (shared[x] if 0 <= x < len(shared) else 0) + t for x, t in zip(group, tails)]
        width = max(1, -(-max(self.lengths) // 64)) + spare
        n = sum(shared) + sum(-(-t // 64) for t in tails) + 3
        order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()
        self.pages = torch.full((n, H, 20 * D), -1, dtype=torch.int32, device="cuda")   # every bit set: NaN
        table = torch.full((B, width), -7, dtype=torch.int32)
        fronts = [[order.pop() for _ in range(s)] for s in shared]
        for b in range(B):
            front = fronts[group[b]] if 0 <= group[b] < len(shared) else []
            row = front + [order.pop() for _ in range(-(-tails[b] // 64))]
            table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
        self.table = table.cuda()
        for x, front in enumerate(fronts):
            self._fill(g, 64 * len(front), torch.tensor([front], dtype=torch.int32).cuda(), 0)
        for b in range(B):
            self._fill(g, tails[b], self.table[b:b + 1], self.lengths[b] - tails[b])

    def _fill(self, g, tokens, table, start):
        if not tokens:
            return
        k, v = (torch.randn(1, self.H, tokens, self.D, generator=g, device="cuda") for _ in range(2))
        k[..., ::19] *= 3.0
        int4.int4_write(k, v, self.pages, table, _i32([start]))

    def query(self, seed, n_q, q_len, dtype=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return torch.randn(len(self.group), n_q, q_len, self.D, generator=g, device="cuda").to(dtype or self.dtype)

    def run(self, q, scaling, counts=None, **kw):
        """The shared pages read once, whatever the sizes (where it does not pay, a call leaves them to int4_attention)."""
        return int4.int4_prefix_attention(q, self.pages, self.table, _i32(self.lengths), scaling, _i32(self.group), _i32(self.shared),
                                          counts=None if counts is None else _i32(counts), **dict(dict(always=True), **kw))

    def values(self):
        """Key and Value [B, H, tokens, D] that the pages hold, in 64 bits."""
        most = max(max(self.lengths), 1)
        k, v = int4.int4_read(self.pages, self.table, _i32([0] * len(self.group)), most, _i32(self.lengths))
        return k.double(), v.double()

    def want(self, q, scaling, counts=None, lengths=None):
        k, v = self.values()
        B, n_q, q_len, D = q.shape
        heads = n_q // self.H
        lengths = lengths or self.lengths
        out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        for b in range(B):
            c = q_len if counts is None else min(counts[b], q_len)
            for i in range(c):
                see = max(0, lengths[b] - (q_len if counts is None else counts[b]) + 1 + i)
                if not see:
                    continue
                x = q[b, :, i].double().view(self.H, heads, D)
                ks, vs = k[b, :, :see], v[b, :, :see]
                p = torch.softmax(x @ ks.transpose(1, 2) * scaling, -1)
                e = (x.abs() @ ks.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scaling) * 2.0 ** -11
                o = p @ vs
                out[b, :, i] = o.view(n_q, D)
                bound[b, :, i] = (HALF_STEP[q.dtype] * o.abs() + (2.0 ** -10 + 2 * e + 2.0 ** -16) * (p @ vs.abs()) + 2.0 ** -24).view(n_q, D)
        return out, bound

    def check(self, got, q, scaling, counts=None):
        want, bound = self.want(q, scaling, counts)
        off = (got.double() - want).abs() - bound
        assert bool((off <= 0).all()), f"outside by {float(off.max()):.3g} in {int((off > 0).sum())} places, {int(off.isnan().sum())} NaN"


@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16), (64, BF16), (128, F16)])
@pytest.mark.parametrize("pages", [1, 2, 3, 9])
def test_one_group(D, dtype, pages):
    batch = Batch(pages, [0] * 5, [pages], [1, 64, 65, 130, 17], 2, D, dtype)
    q = batch.query(1, 14, 1)
    batch.check(batch.run(q, D ** -0.5), q, D ** -0.5)


@pytest.mark.parametrize("n_q,H", [(28, 4), (40, 8), (8, 8), (16, 1), (6, 2), (130, 1)])
@pytest.mark.parametrize("q_len", [1, 3])
def test_heads_and_drafts(n_q, H, q_len):
    batch = Batch(n_q, [0, 1, 0, 1, -1, 0], [5, 12], [9, 70, 3, 200, 150, 64], H, 128)
    q = batch.query(2, n_q, q_len)
    batch.check(batch.run(q, 0.09), q, 0.09)
    flat = q[:, :, :1]
    got = batch.run(flat.squeeze(2), 0.09)           # [batch, n_q, D]
    assert got.shape == (6, n_q, 128) and torch.equal(got, batch.run(flat, 0.09).squeeze(2))


@pytest.mark.parametrize("members", [1, 2, 18, 19, 37, 64, 150])
def test_rows_of_several_tiles(members):
    """7 query heads on a KV head: 128 and 256 rows end inside a sequence's."""
    batch = Batch(members, [0] * members, [21], [1 + 5 * b % 90 for b in range(members)], 1, 64, F16)
    q = batch.query(3, 7, 1)
    batch.check(batch.run(q, 0.125), q, 0.125)


@pytest.mark.parametrize("D,dtype,q_len,own", [(128, BF16, 300, 300), (64, F16, 77, 100), (128, F16, 40, 40)])
def test_a_chunk_behind_its_history(D, dtype, q_len, own):
    """One sequence with many query tokens: its own first pages are the shared ones."""
    batch = Batch(q_len, [0], [30], [own], 2, D, dtype)
    q = batch.query(4, 8, q_len)
    batch.check(batch.run(q, D ** -0.5), q, D ** -0.5)


def test_long_prefixes_in_many_ranges():
    batch = Batch(7, [0, 1, 0, 1, 0, 2], [400, 333, 1], [100, 1, 700, 64, 63, 5], 4, 128)
    q = batch.query(5, 28, 1)
    got = batch.run(q, 0.0884)
    batch.check(got, q, 0.0884)
    assert all(torch.equal(batch.run(q, 0.0884), got) for _ in range(3))     # no result depends on timing


def test_where_it_does_not_pay():
    """Few sequences, few pages: the call is int4_attention's, bit for bit; many of both are not, and right too; groups of
    both kinds in one call."""
    batch = Batch(22, [0, 0, 1, -1], [9, 4], [70, 1, 64, 30], 2, 128)
    q = batch.query(19, 8, 1)
    plain = int4.int4_attention(q, batch.pages, batch.table, _i32(batch.lengths), 0.09)
    assert torch.equal(batch.run(q, 0.09, always=False), plain)
    batch = Batch(23, [0] * 40 + [1, 1], [300, 2], [70 - b for b in range(42)], 4, 128)
    q = batch.query(20, 28, 1)
    got = batch.run(q, 0.0884, always=False)
    batch.check(got, q, 0.0884)
    assert torch.equal(got[:40], batch.run(q, 0.0884)[:40])
    # few shared pages in wide tables: planned on the GPU, and left to the sequences there
    batch = Batch(24, [0] * 40, [2], [70 - b for b in range(40)], 4, 64, F16, spare=600)
    q = batch.query(21, 28, 1)
    batch.check(batch.run(q, 0.125, always=False), q, 0.125)


def test_many_groups():
    groups = 70
    group = [b * 29 % (groups + 1) - 1 for b in range(150)]
    batch = Batch(8, group, [1 + x % 5 for x in range(groups)], [1 + b % 70 for b in range(150)], 2, 64, F16)
    q = batch.query(6, 6, 1)
    batch.check(batch.run(q, 0.125), q, 0.125)


def test_counts_and_sequences_that_pause():
    batch = Batch(9, [0, 0, -1, 0, 0], [4], [20, 7, 100, 64, 3], 2, 128)
    q = batch.query(7, 8, 4)
    counts = [4, 0, 2, 1, 3]
    got = batch.run(q, 0.09, counts)
    batch.check(got, q, 0.09, counts)
    for b, c in enumerate(counts):
        assert not bool(got[b, :, c:].any())


def test_sequences_inside_their_shared_pages():
    """Lengths that end before the shared pages do, down to none, with garbage behind them in nobody's sight."""
    batch = Batch(10, [0] * 6, [8], [0, 10, 90, 0, 0, 1], 2, 64, F16)
    batch.lengths = [512, 522, 602, 100, 0, 1]
    q = batch.query(8, 6, 2)
    batch.check(batch.run(q, 0.125), q, 0.125)


def test_more_shared_pages_named_than_are_written():
    """prefix_pages past every member's length: table entries there are out of the pool, pages unwritten (NaN)."""
    batch = Batch(11, [0, 0, 0], [3], [5, 70, 64], 2, 128)
    q = batch.query(9, 8, 1)
    want, bound = batch.want(q, 0.09)
    for named in (4, 1 << 30, -5, 0):
        got = int4.int4_prefix_attention(q, batch.pages, batch.table, _i32([192, 192, 192]), 0.09, _i32([0, 0, 0]), _i32([named]), always=True)
        alike = int4.int4_attention(q, batch.pages, batch.table, _i32([192, 192, 192]), 0.09)
        w, b = batch.want(q, 0.09, lengths=[192, 192, 192])
        assert bool(((got.double() - w).abs() <= b).all()) and bool(((alike.double() - w).abs() <= b).all())


@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("kind", ["nan", "wide"])
def test_groups_out_of_fp16(where, kind):
    """A shared page with a NaN, or numbers past fp16: its group's members read all pages themselves, the other
    group does not."""
    batch = Batch(12, [0, 1, 0, 1, 1], [6, 5], [30, 64, 100, 1, 90], 2, 64, F16)
    q = batch.query(10, 6, 1)
    k, v = (torch.randn(1, 2, 1, 64, device="cuda") for _ in range(2))
    (k if where == "key" else v)[0, 1, 0, 40] = float("nan") if kind == "nan" else 3e4 if where == "key" else 9e5
    if kind == "wide" and where == "key":
        k[0, 1, 0, 41] = -6e4
    int4.int4_write(k, v, batch.pages, batch.table[:1], _i32([70]))
    got = batch.run(q, 0.125)
    alike = int4.int4_attention(q, batch.pages, batch.table, _i32(batch.lengths), 0.125)
    assert torch.equal(got[[0, 2]].isnan(), alike[[0, 2]].isnan())
    if kind == "nan":
        assert bool(got[0, 3:].isnan().any()) and not bool(got[:, :3].isnan().any())
    want, bound = batch.want(q, 0.125)
    fine = ~want.isnan()
    assert torch.equal(got[[0, 2]].isnan(), want[[0, 2]].isnan())
    assert bool(((got.double() - want).abs() <= bound)[fine].all())
    others = [1, 3, 4]
    assert bool(((got.double() - want).abs() <= bound)[others].all())


@pytest.mark.parametrize("scaling", [0.0, -0.1, 1e-20])
def test_scalings(scaling):
    batch = Batch(13, [0] * 4, [9], [70, 1, 64, 30], 2, 128)
    q = batch.query(11, 8, 1)
    batch.check(batch.run(q, scaling), q, scaling)


@pytest.mark.parametrize("size", [1e-30, 1e-5, 3e4])
def test_queries_of_any_size(size):
    batch = Batch(14, [0] * 3, [5], [70, 1, 64], 1, 128)
    q = (batch.query(12, 4, 1, F32) * size).to(BF16)
    batch.check(batch.run(q, 0.09 / size), q, 0.09 / size)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_scores_that_are_all_far_below_zero(D, dtype):
    """Every score far below zero, down to -1e34: the nearest to zero takes all the weight, wherever it lies."""
    batch = Batch(21, [0] * 4, [7], [70, 1, 64, 300], 1, D, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    for table, start, tokens in ([batch.table[:1], 0, 448], *[(batch.table[b:b + 1], 448, t) for b, t in enumerate([70, 1, 64, 300])]):
        key, value = torch.rand(1, 1, tokens, D, generator=g, device="cuda") + 0.5, torch.randn(1, 1, tokens, D, generator=g, device="cuda")
        int4.int4_write(key, value, batch.pages, table, _i32([start]))
    for size in ((1e3, 6e4) if dtype == F16 else (1e3, 1e9, 2.0 ** 110)):
        q = (-(torch.rand(4, 6, 1, D, generator=g, device="cuda") + 0.5) * size).to(dtype)
        got = batch.run(q, 0.125)
        k, v = batch.values()
        for b in range(4):
            n = batch.lengths[b]
            logits = q[b, :, 0].double() @ k[b, 0, :n].T * 0.125
            best = logits.topk(2, -1)
            # a score is off by its Keys' rounding (bf16 queries: 2^-11) and its fp32 sums
            e = (q[b, :, 0].double().abs() @ k[b, 0, :n].abs().T).amax(-1) * 0.125 * (2.0 ** -11 + 128 * 2.0 ** -24)
            sure = best.values[:, 0] - best.values[:, 1] > 30 + 2 * e
            want = v[b, 0][best.indices[:, 0]]
            off = (got[b, :, 0].double() - want).abs()
            # weight and Value rounded to fp16, the output to its type
            fine = torch.isfinite(q[b, :, 0]).all(-1)         # (fp16 ends at 65504: some queries of 6e4 * 1.5 are infinite)
            assert bool((off <= (HALF_STEP[dtype] + 2.0 ** -10 + 2.0 ** -12) * want.abs() + 2.0 ** -20)[sure & fine].all())
            assert bool(torch.isfinite(got[b, fine]).all())
            # and no result leaves what the Values near the best span
            near = logits >= (best.values[:, :1] - 40 - 2 * e.view(-1, 1))
            for h in fine.nonzero()[:, 0].tolist():
                span = v[b, 0, :n][near[h]]
                low, high = span.amin(0), span.amax(0)
                slack = 2.0 ** -7 * torch.maximum(low.abs(), high.abs()) + 2.0 ** -8
                assert bool(((got[b, h, 0].double() >= low - slack) & (got[b, h, 0].double() <= high + slack)).all())


def test_non_finite_queries_stay_in_their_rows():
    batch = Batch(15, [0] * 4, [5], [70, 1, 64, 8], 2, 64, F16)
    q = batch.query(13, 6, 1)
    clean = batch.run(q, 0.125)
    q[1, 2, 0, 5], q[3, 5, 0, 0] = float("nan"), float("inf")
    got = batch.run(q, 0.125)
    touched = torch.zeros(4, 6, dtype=torch.bool, device="cuda")
    touched[1, 2] = touched[3, 5] = True
    assert torch.equal(got[~touched.view(4, 6, 1)[..., 0]], clean[~touched]) and not bool(torch.isfinite(got[touched]).all(-1).all())


def test_a_dominant_shared_token():
    """One shared token far above the others, and own tokens far above all shared ones."""
    batch = Batch(16, [0] * 3, [6], [90, 64, 2], 1, 128, F16)
    k, v = torch.full((1, 1, 1, 128), 0.7, device="cuda"), torch.zeros(1, 1, 1, 128, device="cuda")
    int4.int4_write(k, v, batch.pages, batch.table[:1], _i32([100]))
    q = torch.full((3, 2, 1, 128), 1.0, dtype=F16, device="cuda") + batch.query(14, 2, 1) * 0.1
    for scaling in (0.1, 0.17, -0.1):
        batch.check(batch.run(q, scaling), q, scaling)
    int4.int4_write(k * 3, v + 1, batch.pages, batch.table[1:2], _i32([batch.lengths[1] - 1]))
    batch.check(batch.run(q, 0.17), q, 0.17)


def test_strides_streams_and_graphs():
    batch = Batch(17, [0, 0, 1, 0, 1], [7, 11], [70, 1, 64, 30, 200], 2, 128)
    q = batch.query(15, 8, 3)
    want = batch.run(q, 0.09)
    turned = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    out = torch.zeros(5, 3, 8, 128, dtype=BF16, device="cuda").transpose(1, 2)
    assert torch.equal(batch.run(turned, 0.09, out=out), want) and torch.equal(out, want)
    odd = torch.zeros(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(batch.run(odd, 0.09), want)
    room = torch.zeros(batch.pages.shape[0], 3, 20 * 128 + 4, dtype=torch.int32, device="cuda")
    spread = room[:, 1:, 4:]
    spread.copy_(batch.pages)
    kept, batch.pages = batch.pages, spread
    assert torch.equal(batch.run(q, 0.09), want)
    batch.pages = kept
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = [batch.run(q, 0.09) for _ in range(3)]
    here = [batch.run(q, 0.09) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, want) for x in there + here)
    lengths, group, shared = _i32(batch.lengths), _i32(batch.group), _i32(batch.shared)
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    for o in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            int4.int4_prefix_attention(q, batch.pages, batch.table, lengths, 0.09, group, shared, out=o, always=True)
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    assert all(torch.equal(o, want) for o in outs)
    lengths -= 1                                     # read when it runs
    group[1] = -1
    graphs[0].replay()
    direct = int4.int4_prefix_attention(q, batch.pages, batch.table, lengths, 0.09, group, shared, always=True)
    assert torch.equal(outs[0], direct) and not torch.equal(direct, want)


def test_pages_out_of_the_pool_are_reported():
    batch = Batch(18, [0, 0], [6], [70, 10], 2, 64, F16)
    q = batch.query(16, 6, 1)
    status = _i32([0])
    batch.run(q, 0.125, status=status)
    assert int(status) == 0
    batch.table[:, 2] = 1 << 20
    got = batch.run(q, 0.125, status=status)
    assert int(status) != 0
    assert torch.equal(got, int4.int4_attention(q, batch.pages, batch.table, _i32(batch.lengths), 0.125))


def test_no_groups_and_refusals():
    batch = Batch(19, [-1, -1], [2], [70, 10], 2, 64, F16)
    q = batch.query(17, 6, 1)
    plain = int4.int4_attention(q, batch.pages, batch.table, _i32(batch.lengths), 0.125)
    assert torch.equal(batch.run(q, 0.125), plain)
    args = dict(query=q, pages=batch.pages, page_table=batch.table, lengths=_i32(batch.lengths), scaling=0.125, prefix_group=_i32([5, -3]),
                prefix_pages=_i32([2]))
    assert torch.equal(int4.int4_prefix_attention(**args), plain)                                  # groups that are not there
    assert torch.equal(int4.int4_prefix_attention(**dict(args, prefix_pages=_i32([]))), plain)
    for error, change in [(ValueError, dict(prefix_group=_i32([0]))), (ValueError, dict(prefix_group=_i32([0, 0]).long())),
                          (ValueError, dict(prefix_pages=_i32([[1]]))), (ValueError, dict(prefix_pages=_i32([1]).cpu())),
                          (TypeError, dict(prefix_pages=None)), (TypeError, dict(prefix_group=None)), (ValueError, dict(scaling=math.nan)),
                          (ValueError, dict(out=q)), (ValueError, dict(out=q[:, :, :1])), (TypeError, dict(always=_i32([1, 2]))),
                          (ValueError, dict(out=q[:1].expand(2, -1, -1, -1))), (ValueError, dict(query=q[:, :5])), (NotImplementedError, dict(query=q.float())),
                          (NotImplementedError, dict(prefix_pages=_i32([1] * 4097)))]:
        with pytest.raises(error):
            int4.int4_prefix_attention(**dict(args, **change))


def test_offsets_past_32_bits():
    """Pages more than 2^31 words into the pool."""
    D, H, n = 128, 8, 110000
    pages = torch.empty(n, H, 20 * D, dtype=torch.int32, device="cuda")
    batch = Batch(20, [0, 0, 0], [4], [70, 10, 64], H, D)
    far = n - batch.pages.shape[0]
    pages[far:] = batch.pages
    q = batch.query(18, 8, 1)
    want = batch.run(q, 0.09)
    batch.pages, batch.table = pages, torch.where(batch.table >= 0, batch.table + far, batch.table)
    assert torch.equal(batch.run(q, 0.09), want)


def test_workspace_of_many_groups_that_share_little():
    """A group for every sequence, few of which share: no record for each, and none for calls that int4_attention takes."""
    B, H, D = 500, 8, 128
    batch = Batch(25, [b // 2 if b < 20 else b for b in range(B)], [2 if x < 10 else 0 for x in range(B)], [1 + b % 3 for b in range(B)], H, D)
    q = batch.query(22, 16, 1)
    lengths, group, shared = _i32(batch.lengths), _i32(batch.group), _i32(batch.shared)
    wide = torch.full((B, 300), -1, dtype=torch.int32, device="cuda")
    wide[:, :batch.table.shape[1]] = batch.table
    for n, always, most in ((4, False, 0), (B, False, 150 << 20), (B, True, 330 << 20)):
        stream = torch.cuda.Stream()
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            int4.int4_attention(q[:n], batch.pages, wide[:n], lengths[:n], 0.09, out=out[:n])      # its own workspace
            before = torch.cuda.memory_allocated()
            int4.int4_prefix_attention(q[:n], batch.pages, wide[:n], lengths[:n], 0.09, group[:n], shared, out=out[:n], always=always)
            assert torch.cuda.memory_allocated() - before <= most
        torch.cuda.synchronize()
        want, bound = batch.want(q, 0.09)
        assert bool(((out.double() - want).abs() <= bound)[:n].all()) and not bool(out[n:].any())
