"""B200-native LogitFill packed KV-cache hot path.

Drop-in for the ``packed`` backend of GASSFY/Logitfill (``logitfill.packed``):
page quantize+pack (K1), split-K GQA decode attention over packed pages plus
the residual page (K2) and the split merge (K3), hand-written for sm_100a and
called through the C ABI in ``include/logitfill_b200.h``.  Beside it,
:mod:`logitfill_b200.int4`: a 4-bit paged cache that needs no policy, attention
over it, and attention over selected pages.
"""
from logitfill_b200.int4 import Int4KVCache, int4_attention, int4_sparse_attention
from logitfill_b200.packed import LogitFillCache, PackedKVCache, PackedKVManager
from logitfill_b200.packed.attention import packed_attention, packed_attention_batched

__all__ = ["Int4KVCache", "LogitFillCache", "PackedKVCache", "PackedKVManager", "int4_attention",
           "int4_sparse_attention", "packed_attention", "packed_attention_batched"]
