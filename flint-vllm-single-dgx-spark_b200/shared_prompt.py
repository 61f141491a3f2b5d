"""Several continuations of one prompt: the prompt is read once and whole, its pages are shared, decode reads them once.

    dec = SharedPromptDecoder(model, streams=8, sampling={...})
    dec.reserve_history(n); dec.capture()
    dec.read_prompt(prompt, room=n)     # prompt attention over all its tokens; stream 0 forked into the others
    tokens = dec.decode(n)              # one CUDA graph per step; the shared pages are read once per layer and step
                                        # (steps beyond the room, counted wherever they are run, are refused)
    dec.branch([3, 5], [0, 0])          # streams 3 and 5 go on from where stream 0 is
    dec.compact()                       # used pages to the front of the cache

The prompt runs layer by layer: add + RMSNorm, QKV and O as plain matrix products on the dequantised weights (exact in
bf16; the library's GEMM), q/k norm and RoPE, the K/V rows written to their pages, flint_prefill_attention, the router and
the grouped prompt MoE; with the decode kernels' rounding points.  Decode is the Decoder's chain with
flint_shared_prefix_attention in the place of the per-stream attention.  One GPU; any layer structure of FlintConfig.
"""
from __future__ import annotations

import numpy as np
import torch

from .fp4moe_decode import grouped_moe
from .kv_pages import PagePool
from .model import PAGE, Decoder
from .prefill_attention import flint_prefill_attention
from .shared_prefix_attention import flint_shared_prefix_attention


class _CountedSteps:
    """The step graph of `dec`, whose every replay takes one of the steps that read_prompt left room for."""

    def __init__(self, graph, dec):
        self.graph, self.dec = graph, dec

    def replay(self):
        self.dec._check_room(1)
        self.dec.steps_left -= 1
        self.dec.steps_done += 1
        self.graph.replay()


class SharedPromptDecoder(Decoder):
    def __init__(self, model, streams: int, moe: str | None = None, sampling: dict | None = None):
        if model.world != 1:
            raise ValueError("SharedPromptDecoder runs on one GPU")
        super().__init__(model, batch=streams, moe=moe or ("block" if streams == 1 else "fused"), attn="chain",
                         sampling=sampling)
        self.pool = PagePool(model.kv_all, streams, model.blocks_per_stream)
        self.bt = self.pool.block_tables
        i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=model.dev)
        self.group_starts, self.prefix_lens = i32(0, streams), i32(0)
        self.all_streams = torch.arange(streams, dtype=torch.int32, device=model.dev)
        self.lens_to_come = torch.zeros_like(self.all_streams)   # tokens each stream has pages for
        self.steps_left = None                               # steps that have pages; None: no prompt has been read
        self.steps_done = 0                                  # since the prompt was read: the column of the next tokens

    # ---- decode ----
    def layer_ops(self, l):
        c, m, L = self.c, self.m, self.m.layers[l]
        attention = lambda: flint_shared_prefix_attention(
            self.q.view(self.M, c.num_heads, c.head_dim), m.kv[l], self.bt, self.seq_lens, self.group_starts,
            self.prefix_lens, L["sinks"], c.window(l), self.scale, self.attn)
        return [(name, attention if name == "attention" else fn) for name, fn in super().layer_ops(l)]

    def capture(self):
        self.steps_left = None
        self.pool.free(self.all_streams)
        self.pool.reserve(self.all_streams, torch.ones_like(self.all_streams))
        super().capture()                                    # runs one step, at the first position
        self.pool.free(self.all_streams)
        self.graphs["step"] = _CountedSteps(self.graphs["step"], self)

    def _check_room(self, n):
        """Behind the reserved pages a step would drop its K and V and attend to keys that are not there."""
        if n > (self.steps_left or 0):
            raise ValueError(f"{n} steps: the room of read_prompt holds {self.steps_left or 0} more")

    def decode(self, n: int):
        """n steps -> their tokens [streams, n] (int32, on the device, a view of the history)."""
        self._check_room(n)
        first = self.steps_done
        if first + n > self.history.shape[1]:
            raise ValueError(f"the history holds {self.history.shape[1]} steps, {first} are done: reserve_history() for all")
        super().decode(n)
        return self.history[:, first:first + n]

    def _set_state(self, tokens, positions):
        dev = self.m.dev
        self.tokens.copy_(torch.as_tensor(np.asarray(tokens, np.int32), device=dev))
        self.positions.copy_(torch.as_tensor(np.asarray(positions, np.int64), device=dev))
        self._follow_tables()

    def _follow_tables(self):
        """seq_lens and slots from positions and the tables (a stream without a page there writes nothing)."""
        self.seq_lens.copy_(self.positions + 1)
        column, width = self.positions // PAGE, self.bt.shape[1]
        page = self.bt.gather(1, column.clamp(max=width - 1)[:, None])[:, 0].long()
        self.slots.copy_(torch.where((page >= 0) & (column < width), page * PAGE + self.positions % PAGE, -1))

    def prefill(self, prompts):
        raise NotImplementedError("SharedPromptDecoder reads one prompt for all streams: read_prompt()")

    def fill_kv_random(self, prompts, seed: int = 0):
        raise NotImplementedError("the streams' pages come from read_prompt()")

    def generate_host_driven(self, n, pinned):
        raise NotImplementedError("slots follow the pool's tables on the device: decode()")

    # ---- the prompt ----
    @staticmethod
    def _norm(x, res, w, eps):
        s = x.float() if res is None else x.float() + res.float()
        return (s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * w.float()).bfloat16(), s.bfloat16()

    @staticmethod
    def _project(x, weight):
        P, S, gs = weight
        w = torch.empty((P.shape[0], 2 * P.shape[1]), dtype=torch.bfloat16, device=P.device)
        torch.ops.flint_b200.nvfp4_dequant(P, S, None, w)
        return (torch.mm(x, w.t(), out_dtype=torch.float32) * gs).bfloat16()

    def _heads(self, y, w, cos_sin):
        n = (y.float() * torch.rsqrt(y.float().square().mean(-1, keepdim=True) + self.c.rms_eps) * w.float())
        if cos_sin is None:
            return n.bfloat16()
        a, b = n.bfloat16().float().chunk(2, -1)
        cos, sin = cos_sin[:, None].chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).bfloat16()

    @staticmethod
    def _router_logits(xn, gate):
        return torch.mm(xn, gate.t(), out_dtype=torch.float32).bfloat16().float()

    @staticmethod
    def _choose(logits, ew):
        """-> (experts, weights) [tokens, topk]: the largest logits, ties to the lower id, their scores over their sum."""
        value, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
        value, ids = value[:, :ew.topk], ids[:, :ew.topk].to(torch.int32).contiguous()
        weight = torch.softmax(value, -1) if ew.score_fn == 0 else torch.sigmoid(value)
        return ids, weight / weight.sum(-1, keepdim=True)

    def _experts(self, xn, L):
        T, ew = xn.shape[0], L["experts"]
        one = lambda w: grouped_moe(xn, torch.zeros((T, 1), dtype=torch.int32, device=xn.device),
                                    torch.ones((T, 1), device=xn.device), w)
        if L["gate"] is None:
            return one(ew)
        out = grouped_moe(xn, *self._choose(self._router_logits(xn, L["gate"]), ew), ew)
        return out if ew.shared is None else out + one(ew.shared)

    def read_prompt(self, prompt, room: int):
        """Every stream goes on from `prompt` (token ids), with pages for `room` more tokens.  Leaves the state at the
        last prompt token, as Decoder.prefill does: the first step reads it and draws each stream's first token."""
        m, prompt = self.m, np.asarray(prompt, np.int64)
        n = prompt.size - 1                                   # tokens whose K and V the cache takes now
        # (the last page may reach behind the rotary table, which has a row for each position)
        most = min(m.blocks_per_stream * PAGE, m.cos_sin.shape[0])
        if n < 0 or room < 0 or n + 1 + room > most:
            raise ValueError(f"a prompt of {n + 1} tokens and {room} more do not fit {most}")
        if prompt.min() < 0 or prompt.max() >= m.embed.shape[0]:
            raise ValueError(f"token ids must lie in 0 .. {m.embed.shape[0] - 1}, got {prompt.min()} .. {prompt.max()}")
        if not self.graphs:
            self.capture()
        c, pool, dev = self.c, self.pool, m.dev
        ids = torch.as_tensor(prompt, device=dev)
        self.steps_left = None
        pool.free(self.all_streams)
        if n:
            pool.reserve([0], [n])
            pos = torch.arange(n, device=dev)
            page, row = self.bt[0, pos // PAGE].long(), pos % PAGE
            cu, lens = (torch.tensor(v, dtype=torch.int32, device=dev) for v in ([0, n], [n]))
            x, res = m.embed[ids[:n]], None
            for l, L in enumerate(m.layers):
                xn, res = self._norm(x, res, L["ln1"], c.rms_eps)
                qkv = self._project(xn, L["qkv"]).view(n, -1, c.head_dim)
                q, k, v = qkv.split([c.num_heads, c.num_kv_heads, c.num_kv_heads], 1)
                cs = m.cos_sin[:n] if c.uses_rope(l) else None
                m.kv[l][page, :, row] = torch.cat([self._heads(k, L["k_norm"], cs), v], -1)
                if l + 1 == c.layers:
                    break                                     # nothing reads the last layer's output for these tokens
                a = torch.empty((n, c.num_heads, c.head_dim), dtype=torch.bfloat16, device=dev)
                flint_prefill_attention(self._heads(q, L["q_norm"], cs), m.kv[l], self.bt[:1], cu, lens, L["sinks"],
                                        c.window(l), self.scale, a)
                xn, res = self._norm(self._project(a.view(n, -1), L["o"]), res, L["ln2"], c.rms_eps)
                x = self._experts(xn, L)
        pool.seq_lens[0] = n
        if self.M > 1:
            pool.fork([0] * (self.M - 1), self.all_streams[1:])
        self.lens_to_come.fill_(n + 1 + room)
        pool.reserve(self.all_streams, self.lens_to_come)
        self.prefix_lens.fill_(n // PAGE * PAGE)
        self._set_state(np.full(self.M, int(ids[-1])), np.full(self.M, n))
        self.step_ctr.zero_()
        torch.cuda.synchronize()
        self.check_status()
        self.steps_done = 0
        self.steps_left = room + 1                            # the first one writes the last prompt token's K and V

    def branch(self, dst, src):
        """Streams dst[i] (host ints) give up their own continuation and go on from where stream src[i] is."""
        pool, dev = self.pool, self.m.dev
        if self.steps_left is None:
            raise ValueError("branch: no prompt yet: read_prompt() first")
        if (len(src) != len(dst) or len(set(dst)) != len(dst) or set(src) & set(dst)
                or any(not 0 <= b < self.M for b in (*src, *dst))):
            raise ValueError(f"branch: {dst} from {src} among {self.M} streams")
        if not dst:
            return
        src, dst = (torch.as_tensor(v, dtype=torch.int32, device=dev) for v in (src, dst))
        pool.seq_lens.copy_(self.positions)                   # cached tokens; the current one is not yet among them
        pool.free(dst)
        pool.fork(src, dst)
        for state in (self.tokens, self.positions, self.out_tok):
            state[dst.long()] = state[src.long()]
        if self.history.shape[1] > 1:
            self.history[dst.long()] = self.history[src.long()]
        pool.reserve(self.all_streams, self.lens_to_come)
        self._follow_tables()

    def compact(self) -> int:
        """Used pages to the front of the cache; -> how many are in use."""
        self.pool.compact()
        self._follow_tables()
        return int(self.pool.live.item())
