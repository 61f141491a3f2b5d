"""Decode attention of streams that share a prompt: the shared pages of the paged cache are read once for all of them.

``flint_shared_prefix_attention(q, kv_cache, block_tables, seq_lens, group_starts, prefix_lens, sinks, window, scale, out)
-> out`` gives what ``flint_decode_attention(q, kv_cache, block_tables, seq_lens, sinks, window, scale, out)`` gives, for
streams that come in groups: group g is the streams group_starts[g] .. group_starts[g + 1] - 1 (int32 [groups + 1], rising
from 0 to the batch size), whose tables begin with the same pages for prefix_lens[g] tokens (int32 [groups]; 0: nothing
shared, and a page that is not full is read per stream).  A stream with seq_lens 0 (a padded slot) gives zeros.
CUDA-graph safe: the launch depends on the shapes only; lengths, groups and tables are read on the device.
"""
from __future__ import annotations

from . import ops as _ops


def flint_shared_prefix_attention(q, kv_cache, block_tables, seq_lens, group_starts, prefix_lens, sinks, window, scale,
                                  out):
    _ops.run("shared_prefix_attention", q, kv_cache, block_tables, seq_lens, group_starts, prefix_lens, sinks,
             int(window or 0), float(scale), out)
    return out
