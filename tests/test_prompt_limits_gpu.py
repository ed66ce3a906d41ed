"""GPU tests of what ends a call of the tensor-core attention kernels before its time: the
limit of their waits, how it is reported, and what must not reach it.  No test faults or
hangs the GPU: a wait runs out on a flag that nothing sets, and the kernel returns."""
from __future__ import annotations

import time

import pytest
import torch

from logitfill_b200 import _lib, prompt
from logitfill_b200.adapter import DeepSeekQwenKVAdapter
from logitfill_b200.synthetic import synthetic_levels
from tests.qwen_cases import tiny_qwen2

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_the_adapter_reports_a_prefill_that_gave_up(monkeypatch):
    """What a prompt's kernel writes into its status word is raised by the cache's check_status."""
    model = tiny_qwen2(n_q=4, n_kv=2, head_dim=128, layers=2, vocab=64, seed=3, device="cuda", dtype=BF16, attn="sdpa")
    a = DeepSeekQwenKVAdapter(model, prompt="kernel").attach()
    a.set_k_levels(list(synthetic_levels(2, 2, 128, 3.0, seed=3)))
    ids = torch.zeros(1, 40, dtype=torch.long, device="cuda")
    with torch.no_grad():
        model(input_ids=ids, use_cache=True, past_key_values=a.make_cache())
    a.packed_manager().cache.check_status()              # a call that went well leaves it clean
    a.packed_manager().reset()
    real = prompt.prompt_attention

    def gives_up(*args, status=None, **kw):
        out = real(*args, status=status, **kw)
        if status is not None:
            status.fill_(_lib.LF_ERR_DEVICE_TIMEOUT)
        return out

    monkeypatch.setattr(prompt, "prompt_attention", gives_up)
    with torch.no_grad():
        model(input_ids=ids, use_cache=True, past_key_values=a.make_cache())
    with pytest.raises(RuntimeError, match="timed out"):
        a.packed_manager().cache.check_status()
    a.detach()


MS = 1_000_000


def _tile_wait(limit_ns, busy_ns, arrive):
    status = torch.full((1,), 77, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    since = time.perf_counter()
    _lib.check(_lib.lib().lf_selftest_tile_wait(_lib.ptr(status), limit_ns, busy_ns, int(arrive), _lib.stream_handle(status.device)),
               "lf_selftest_tile_wait")
    torch.cuda.synchronize()
    return int(status), time.perf_counter() - since


@pytest.mark.parametrize("limit,busy,arrive,want", [(50 * MS, 0, True, "LF_OK"), (20 * MS, 0, False, "LF_ERR_DEVICE_TIMEOUT"),
                                                    (10 * MS, 200 * MS, True, "LF_OK"), (10 * MS, 100 * MS, False, "LF_ERR_DEVICE_TIMEOUT")])
def test_the_limit_is_on_a_time_in_which_nothing_moves(limit, busy, arrive, want):
    status, took = _tile_wait(limit, busy, arrive)
    assert status == getattr(_lib, want)
    assert took >= (busy if arrive else busy + limit) * 1e-9 and took < 3.0
    # the context is as good as before
    assert float(torch.ones(8, device="cuda").sum()) == 8.0


def test_rows_that_take_longer_than_the_limit():
    """A Value that not all rows of a tile may see is NaN: its rows are done one by one, 16 to a warp over all Keys,
    which takes seconds here.  The roles that wait meanwhile do not give up."""
    n, D = 3 << 18, 64
    g = torch.Generator(device="cuda").manual_seed(12)
    q, k, v = (torch.randn(n, 1, D, generator=g, device="cuda").to(BF16) for _ in range(3))
    v += 2.0                                             # (results of 2, not of the small mean of many signs)
    v[n - 1] = float("nan")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    prompt.prompt_attention(q, k, v, 0.125, out=out, status=status)
    assert int(status) == _lib.LF_OK
    assert bool(out[n - 1].isnan().all()) and bool(torch.isfinite(out[:n - 1]).all())
    assert not bool((out == 7.0).all(-1).any())          # every row was written
    u = 2.0 ** -8
    for i in (0, 129, 200001, n - 257, n - 256, n - 129, n - 128, n - 2):
        a, b, c = q[i, 0].double(), k[:i + 1, 0].double(), v[:i + 1, 0].double()
        p = torch.softmax(b @ a * 0.125, 0)
        # the bound of the operator's own tests; n 2^-30 for fp32 sums of n terms, whose roundings go both ways
        # (some sqrt(n) 2^-24 of the sum, far less)
        e = float((b.abs() @ a.abs()).max()) * 0.125 * D * 2.0 ** -24
        bound = u * (p @ c).abs() + (u + 2 * e + 2.0 ** -16 + n * 2.0 ** -30) * (p @ c.abs()) + 2.0 ** -24
        assert bool(((out[i, 0].double() - p @ c).abs() <= bound).all()), i


def test_very_many_sequences():
    """The plan's time goes with the number of sequences, not with its square (3 s for these, were each item searched
    among all sequences), and deals every one of them out."""
    n, H, D = 100000, 8, 64
    g = torch.Generator(device="cuda").manual_seed(13)
    counts = torch.tensor([1, 0, 2, 1, 1], device="cuda").repeat(n // 5)
    counts[77] = 700                                     # and one with several items, in levels of its own
    starts = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    starts[1:] = counts.cumsum(0)
    rows = int(starts[-1])
    q, k, v = (torch.randn(rows, H, D, generator=g, device="cuda").to(BF16) for _ in range(3))
    out = torch.full_like(q, 7.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    prompt.prompt_attention(q[:9], k[:9], v[:9], 0.125)   # (the first call of a process loads the kernel)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    prompt.prompt_attention(q, k, v, 0.125, starts=starts, out=out, status=status)
    end.record()
    torch.cuda.synchronize()
    assert int(status) == _lib.LF_OK and begin.elapsed_time(end) < 500
    first = starts[:-1].long()[counts == 1]
    assert torch.equal(out[first], v[first])             # a token that sees itself alone
    first = starts[:-1].long()[counts == 2]
    assert torch.equal(out[first], v[first])
    a, u = q[first + 1].double(), 2.0 ** -8
    p = torch.softmax(torch.stack([(a * k[first].double()).sum(-1), (a * k[first + 1].double()).sum(-1)], -1) * 0.125, -1).unsqueeze(-1)
    x, y = v[first].double(), v[first + 1].double()
    want, size = p[..., 0, :] * x + p[..., 1, :] * y, p[..., 0, :] * x.abs() + p[..., 1, :] * y.abs()
    e = (a.abs() * torch.maximum(k[first].abs(), k[first + 1].abs()).double()).sum(-1, keepdim=True) * 0.125 * D * 2.0 ** -24
    assert bool(((out[first + 1].double() - want).abs() <= u * want.abs() + (u + 2 * e + 2.0 ** -16) * size + 2.0 ** -24).all())
    at = int(starts[77])
    alone = prompt.prompt_attention(q[at:at + 700], k[at:at + 700], v[at:at + 700], 0.125)
    assert torch.equal(out[at:at + 700], alone)
