"""GPU tests of what ends a call of the tensor-core attention kernels before its time: the
limit of their waits, how it is reported, and what must not reach it.  No test faults or
hangs the GPU: a wait runs out on a flag that nothing sets, and the kernel returns."""
from __future__ import annotations

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
