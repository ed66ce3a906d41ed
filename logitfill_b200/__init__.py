"""B200-native LogitFill packed KV-cache hot path.

Drop-in for the ``packed`` backend of GASSFY/Logitfill (``logitfill.packed``):
page quantize+pack (K1), split-K GQA decode attention over packed pages plus
the residual page (K2) and the split merge (K3), hand-written for sm_100a and
called through the C ABI in ``include/logitfill_b200.h``.  Beside it,
:mod:`logitfill_b200.int4`: a 4-bit paged cache that needs no policy, attention
over it, over selected pages, and over pages that sequences share; and
:mod:`logitfill_b200.prompt`: rotary positions and the attention of whole prompts.
"""
from logitfill_b200.int4 import Int4KVCache, int4_attention, int4_prefix_attention, int4_sparse_attention
from logitfill_b200.packed import LogitFillCache, PackedKVCache, PackedKVManager
from logitfill_b200.packed.attention import packed_attention, packed_attention_batched
from logitfill_b200.prompt import prompt_attention, rotary_embed, rotary_frequencies

__all__ = ["Int4KVCache", "LogitFillCache", "PackedKVCache", "PackedKVManager", "int4_attention",
           "int4_prefix_attention", "int4_sparse_attention", "packed_attention", "packed_attention_batched",
           "prompt_attention", "rotary_embed", "rotary_frequencies"]
