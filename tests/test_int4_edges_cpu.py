"""CPU tests of the 4-bit cache's refusals and bookkeeping at the edges."""
from __future__ import annotations

import pytest
import torch

from logitfill_b200 import int4


def test_pools_without_pages_heads_or_sequences_are_refused():
    """Before anything divides by an extent: ValueError, wherever the tensors are."""
    pages, table = torch.zeros(4, 2, 1280, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    q, n = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for p, t, m, x in ((pages[:, :0], table, n, q), (pages[:0], table, n, q), (pages[..., :0], table, n, q),
                       (pages, table[:, :0], n, q), (pages, table[:0], n[:0], q[:0])):
        with pytest.raises(ValueError):
            int4.int4_attention(x, p, t, m, 1.0)
        with pytest.raises(ValueError):
            int4.int4_read(p, t, m, 3)
