"""Prompts, shared prompts and page operations over the paged KV cache on the CPU -- test infrastructure only.

Attention straight from its definition in float64: query i of a sequence's n, at position p = len - n + i, over the keys
max(0, p - window + 1) .. p: o = sum e^(s_j - m) v_j / (sum e^(s_j - m) + e^(sink - m)), s = scale q . k.  Beside o comes
spread = sum e^(s_j - m) |v_j| / (..), what the rounding of the probabilities is measured against.
"""
from __future__ import annotations

import numpy as np

PAGE = 16


def attention_rows(q, keys, values, first_pos, sinks, window, scale):
    """q [n, Hq, D] at positions first_pos ..; keys / values [L, Hkv, D] -> (o, spread) [n, Hq, D] float64."""
    n, Hq, D = q.shape
    G = Hq // keys.shape[1] if keys.shape[1] else 1
    o, spread = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    for i in range(n):
        p = first_pos + i
        lo = max(0, p - window + 1) if window else 0
        if p < 0:
            continue
        k, v = keys[lo:p + 1].astype(np.float64), values[lo:p + 1].astype(np.float64)
        for h in range(Hq):
            s = scale * (k[:, h // G] @ q[i, h].astype(np.float64))
            m = s.max()
            e = np.exp(s - m)
            den = e.sum() + (np.exp(float(sinks[h]) - m) if sinks is not None else 0.0)
            o[i, h] = e @ v[:, h // G] / den
            spread[i, h] = e @ np.abs(v[:, h // G]) / den
    return o, spread


def cached(kv, table, length):
    """Keys and values [length, Hkv, D] of one stream (kv [blocks, Hkv, 16, 2D])."""
    D = kv.shape[3] // 2
    rows = np.concatenate([kv[table[i]].transpose(1, 0, 2) for i in range((length + PAGE - 1) // PAGE)] +
                          [np.zeros((0, kv.shape[1], 2 * D), kv.dtype)])[:length]
    return rows[..., :D], rows[..., D:]


def prefill_attention(q, kv, tables, q_lens, seq_lens, sinks, window, scale):
    out, spread, at = np.zeros(q.shape), np.zeros(q.shape), 0
    for b, n in enumerate(q_lens):
        k, v = cached(kv, tables[b], int(seq_lens[b]))
        out[at:at + n], spread[at:at + n] = attention_rows(q[at:at + n], k, v, int(seq_lens[b]) - n, sinks, window, scale)
        at += n
    return out, spread


class Pool:
    """The page pool in plain Python; `bad` collects the status bits."""

    def __init__(self, kv, streams, max_blocks):
        self.kv = kv.copy()                                   # [layers, blocks, ...]
        self.ref = [0] * kv.shape[1]
        self.tables = [[] for _ in range(streams)]
        self.lens, self.max_blocks, self.bad = [0] * streams, max_blocks, 0

    def _take(self):
        p = self.ref.index(0)
        self.ref[p] = 1
        return p

    def _first(self, ids):
        """Places of `ids` that name a stream for the first time; the others are recorded."""
        seen = set()
        for i, s in enumerate(ids):
            if 0 <= s < len(self.tables) and s not in seen:
                seen.add(s)
                yield i
            else:
                self.bad |= 4

    def reserve(self, streams, lens):
        left, asked = self.ref.count(0), 0
        for i in self._first(streams):
            want = -(-lens[i] // PAGE)
            if lens[i] < 0 or want > self.max_blocks:
                self.bad |= 4
                continue
            need = max(0, want - len(self.tables[streams[i]]))
            asked += need
            if need and asked > left:
                self.bad |= 8
                continue
            self.tables[streams[i]] += [self._take() for _ in range(need)]

    def fork(self, src, dst):
        todo = []
        for i in self._first(dst):
            s, d = src[i], dst[i]
            if not 0 <= s < len(self.tables) or s == d or self.tables[d]:
                self.bad |= 4
            elif -(-self.lens[s] // PAGE) > len(self.tables[s]):
                self.bad |= 4
            else:
                todo.append((s, d, self.lens[s]))
        sources = {s: list(self.tables[s]) for s, _, _ in todo}
        for s, d, n in todo:
            if n % PAGE and 0 not in self.ref:
                self.bad |= 8
                continue
            self.tables[d] = sources[s][:n // PAGE]
            for p in self.tables[d]:
                self.ref[p] += 1
            if n % PAGE:
                p = self._take()
                self.kv[:, p] = self.kv[:, sources[s][n // PAGE]]
                self.tables[d].append(p)
            self.lens[d] = n

    def free(self, streams):
        for s in streams:
            if not 0 <= s < len(self.tables):
                self.bad |= 4
                continue
            for p in self.tables[s]:
                self.ref[p] -= 1
            self.tables[s], self.lens[s] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.ref)
        holes = [p for p in range(live) if not self.ref[p]]
        remap = [p if r else -1 for p, r in enumerate(self.ref)]
        for p in range(live, len(self.ref)):
            if self.ref[p]:
                to = holes.pop(0)
                remap[p] = to
                self.kv[:, to] = self.kv[:, p]
                self.ref[to], self.ref[p] = self.ref[p], 0
        self.tables = [[remap[p] for p in t] for t in self.tables]
        return remap, live
