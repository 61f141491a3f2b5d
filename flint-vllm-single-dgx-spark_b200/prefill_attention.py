"""Causal attention of whole prompts over the paged KV cache (the decode attention's counterpart for many query tokens).

``flint_prefill_attention(q, kv_cache, block_tables, cu_seqlens, seq_lens, sinks, window, scale, out) -> out``:
q bf16 [tokens, heads, 128], the query tokens of all sequences packed one behind the other; cu_seqlens int32 [batch + 1],
where each sequence's queries begin (a sequence may have none); kv_cache FlashInfer HND bf16 [blocks, kv_heads, 16, 256]
(K | V); block_tables int32 [batch, max_blocks]; seq_lens int32 [batch], the cached tokens of each sequence, its queries'
own keys and values included (write them first); sinks fp32 [heads] or None; window None for full attention;
out bf16 [tokens, heads, 128].

The queries are the last tokens of their sequence: a whole prompt, a chunk behind what is cached, or drafted tokens.
Slots of the cache that no query sees may hold anything; a value that is not finite in a slot that some queries see may
also reach queries of the same sequence that do not.
CUDA-graph safe: the launch depends on the shapes only; lengths and tables are read on the device.
"""
from __future__ import annotations

from . import ops as _ops


def flint_prefill_attention(q, kv_cache, block_tables, cu_seqlens, seq_lens, sinks, window, scale, out):
    _ops.run("prefill_attention", q, kv_cache, block_tables, cu_seqlens, seq_lens, sinks, int(window or 0), float(scale), out)
    return out
