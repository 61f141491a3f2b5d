"""The operators of a paged KV cache whose prompts are read whole and shared: what is measured of them, and their plain forms.

  prefill    causal grouped-query attention of packed prompts (or prompt chunks, or drafted tokens) over the paged cache
  shared     decode attention of streams that share a prompt's pages, the shared pages read once for all of them
  turnover   one step of a search over continuations: finished streams freed, survivors forked, the next pages reserved
  compact    live pages moved to the front of the pool, the block tables rewritten

The cache is bf16 [blocks, kv_heads, 16, 256], K in the first 128 columns and V in the rest.  With `own` false the
operators run in elementary torch operations in 32 bits, with `own` true through the framework's entry points.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

D = 128          # head dimension of the framework's kernels
PAGE = 16        # tokens of a cache page
SCALE = D ** -0.5


def _package():
    """The framework's package (its folder's name is no identifier) as flint_b200."""
    if "flint_b200" not in sys.modules:
        folder = os.path.abspath("flint-vllm-single-dgx-spark_b200")
        spec = importlib.util.spec_from_file_location("flint_b200", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules["flint_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["flint_b200"]


def _ints(text):
    return [int(x) for x in text.split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


# ---------------------------------------------------------------------------------------------------------------
# The cases.  32 query heads on 4 KV heads of 128, 48 layers, a 6,057-token prompt, a window of 513 tokens with a
# learned sink per head and 8 streams are this repository's own configurations.
# ---------------------------------------------------------------------------------------------------------------
def listed():
    layer = dict(heads=32, kv_heads=4)
    return [
        # a chat turn's first tokens: the smallest call, where latency counts
        dict(name="prefill short prompt", op="prefill", q="17", past="0", window=0, sinks=False, **layer),
        # drafted tokens of eight streams looked at in one call: few rows on long contexts
        dict(name="prefill drafted tokens", op="prefill", q="4,5,1,4,4,3,4,2",
             past="6057,513,1200,4000,31,0,2750,5120", window=0, sinks=False, **layer),
        # prompts of a batch packed together, one of them empty, in a layer with a window and sinks
        dict(name="prefill packed, window", op="prefill", q="1,16,513,77,2048,0,300,1111", past="0,0,0,100,0,0,16,0",
             window=513, sinks=True, **layer),
        # the benchmark's prompt in one call
        dict(name="prefill 6057", op="prefill", q="6057", past="0", window=0, sinks=False, **layer),
        # a long document; the largest call
        dict(name="prefill 16421", op="prefill", q="16421", past="0", window=0, sinks=False, **layer),
        # two samples of a short prompt
        dict(name="shared 2 streams", op="shared", groups="2", prefix="256", lens="300,271", window=0, sinks=False,
             **layer),
        # eight samples of the benchmark's prompt (6,048 of its 6,057 tokens fill whole pages)
        dict(name="shared 8 streams", op="shared", groups="8", prefix="6048",
             lens="6058,6070,6101,6066,6209,6160,6084,6131", window=0, sinks=False, **layer),
        # a server's batch: three system prompts, a stream without one, two padded slots, sinks
        dict(name="shared 192 streams", op="shared", groups="100,60,29,1,2", prefix="16384,4096,1008,0,0",
             lens=_text([16384 + 1 + 37 * i % 700 for i in range(100)] + [4096 + 5 + 53 * i % 1100 for i in range(60)]
                        + [1008 + 11 * i % 300 + 1 for i in range(29)] + [777, 0, 0]),
             window=0, sinks=True, **layer),
        # beam search over four beams of a small model: the smallest turnover
        dict(name="turnover 4 streams", op="turnover", layers=2, blocks=96, kv_heads=4, streams=4, prompt=300, grown=21,
             freed=2),
        # a search over 64 continuations of the benchmark's prompt, 48 layers
        dict(name="turnover 64 streams", op="turnover", layers=48, blocks=900, kv_heads=4, streams=64, prompt=6057,
             grown=37, freed=40),
        # a small pool with holes
        dict(name="compact 96 blocks", op="compact", layers=2, blocks=96, kv_heads=4, streams=4, pages=12, live=50),
        # a server's pool half emptied by streams that ended
        dict(name="compact 1536 blocks", op="compact", layers=48, blocks=1536, kv_heads=4, streams=38, pages=40, live=55),
    ]


def _log(rng, lo, hi):
    """A whole number, spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        pool = case.get("layers", 0) * case.get("blocks", 0) * case["kv_heads"]
        if w["flops"] <= 2.2e12 and w["bytes"] <= 3.6e8 and pool <= 48 * 1536 * 4:
            return case


def _draw(rng):
    op = rng.choice(["prefill", "prefill", "shared", "shared", "turnover", "compact"])
    kv_heads = rng.choice([1, 2, 4, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 8])
    window = rng.choice([0, 0, 1, 128, 513, _log(rng, 2, 4000)])
    common = dict(heads=heads, kv_heads=kv_heads, window=window, sinks=rng.random() < 0.5)
    if op == "prefill":
        n, most = _log(rng, 1, 16), _log(rng, 1, 12000)
        q = [_log(rng, 1, most) if rng.random() > 0.06 else 0 for _ in range(n)]
        if not sum(q):
            q[0] = 1
        return dict(op=op, q=_text(q), past=_text([rng.choice([0, _log(rng, 1, 9000)]) for _ in range(n)]), **common)
    if op == "shared":
        groups = [_log(rng, 1, 96) for _ in range(rng.choice([1, 1, 2, 3]))]
        prefix = [rng.choice([0, 1, 1, 1]) * PAGE * _log(rng, 1, 1024) for _ in groups]
        most = _log(rng, 1, 1500)
        lens = [p + _log(rng, 1, most) for g, p in zip(groups, prefix) for _ in range(g)]
        lens = [0 if rng.random() < 0.04 else x for x in lens]
        return dict(op=op, groups=_text(groups), prefix=_text(prefix), lens=_text(lens), **common)
    layers, streams = _log(rng, 1, 48), _log(rng, 2, 128)
    if op == "turnover":
        freed = rng.randint(1, streams - 1)
        prompt, grown = _log(rng, 1, 6000), _log(rng, 1, 100)
        pages = -(-prompt // PAGE) + streams * (grown // PAGE + 4)
        return dict(op=op, layers=layers, blocks=pages + _log(rng, 1, 64), kv_heads=kv_heads, streams=streams,
                    prompt=prompt, grown=grown, freed=freed)
    pages = _log(rng, 1, 24)
    return dict(op=op, layers=layers, blocks=streams * pages + _log(rng, 1, 64), kv_heads=kv_heads, streams=streams,
                pages=pages, live=rng.randint(0, 100))


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------
def _pages(tokens):
    return -(-tokens // PAGE)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] in ("turnover", "compact"):
        return _prepare_pages(case, g, ints)
    hq, hkv = case["heads"], case["kv_heads"]
    if case["op"] == "prefill":
        q_lens = _ints(case["q"])
        lens = [q + p for q, p in zip(q_lens, _ints(case["past"]))]
        owned, rows = [_pages(n) for n in lens], sum(q_lens)
    else:
        groups, prefix, lens = _ints(case["groups"]), _ints(case["prefix"]), _ints(case["lens"])
        of = [k for k, n in enumerate(groups) for _ in range(n)]
        owned = [max(0, _pages(n) - prefix[k] // PAGE) for k, n in zip(of, lens)]
        rows = len(lens)
    # every stream's pages lie scattered over the pool, as they do after some time of serving
    own_pages = sum(owned) + (sum(p // PAGE for p in prefix) if case["op"] == "shared" else 0)
    ids = torch.randperm(own_pages + 3, generator=torch.Generator().manual_seed(seed)).tolist()
    take = lambda n: [ids.pop() for _ in range(n)]  # noqa: E731
    if case["op"] == "prefill":
        tables = [take(n) for n in owned]
    else:
        first = [take(p // PAGE) for p in prefix]
        tables = [first[k] + take(n) for k, n in zip(of, owned)]
    width = max(1, max(map(len, tables)))
    s = dict(op=case["op"], lens=lens, window=case["window"], heads=hq)
    s["kv"] = torch.randn(own_pages + 3, hkv, PAGE, 2 * D, generator=g, device="cuda", dtype=torch.bfloat16)
    s["tables"] = ints([t + [0] * (width - len(t)) for t in tables])
    s["seq_lens"] = ints(lens)
    s["q"] = 2 * torch.randn(rows, hq, D, generator=g, device="cuda", dtype=torch.bfloat16)
    s["sinks"] = 2 * torch.randn(hq, generator=g, device="cuda") if case["sinks"] else None
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "prefill":
        s["q_lens"] = q_lens
        s["cu_seqlens"] = ints([sum(q_lens[:i]) for i in range(len(q_lens) + 1)])
    else:
        s["groups"], s["prefix"] = groups, prefix
        s["group_starts"] = ints([sum(groups[:i]) for i in range(len(groups) + 1)])
        s["prefix_lens"] = ints(prefix)
    return s


def _prepare_pages(case, g, ints):
    """A pool in use: reference counts, block tables, lengths and page counts of its streams, in one buffer so that a
    caller can go back to an earlier moment with one copy (as run() does before each pass)."""
    blocks, streams = case["blocks"], case["streams"]
    ids = torch.randperm(blocks, generator=g, device="cuda").tolist()
    ref, lens, tables = [0] * blocks, [0] * streams, [[] for _ in range(streams)]
    if case["op"] == "turnover":
        shared = ids[:case["prompt"] // PAGE]
        del ids[:len(shared)]
        for b in range(streams):
            lens[b] = case["prompt"] + case["grown"] + b % 7
            tables[b] = shared + [ids.pop() for _ in range(_pages(lens[b]) - len(shared))]
        width = _pages(case["prompt"] + case["grown"] + 7 + 2 * PAGE)
        # the worst streams end (every third first); each makes room for a copy of a survivor
        order = sorted(range(streams), key=lambda b: (b % 3 != 1, b))
        ended, alive = order[:case["freed"]], sorted(order[case["freed"]:])
        src = [alive[(i * i) % len(alive)] for i in range(len(ended))]
        grow = [n + PAGE for n in lens]
        for d, b in zip(ended, src):
            grow[d] = lens[b] + PAGE
    else:
        stays = (torch.rand(streams, generator=g, device="cuda") * 100 < case["live"]).tolist()
        for b in range(streams):
            if stays[b]:
                tables[b] = [ids.pop() for _ in range(case["pages"])]
                lens[b] = case["pages"] * PAGE - b % PAGE
        width, src, ended, grow = case["pages"], [], [], []
    for t in tables:
        for p in t:
            ref[p] += 1
    flat = ref + lens + [len(t) for t in tables] + [x for t in tables for x in t + [-1] * (width - len(t))]
    saved = ints(flat)
    meta = saved.clone()
    at = lambda a, n: meta[a:a + n]  # noqa: E731
    return dict(op=case["op"], saved=saved, meta=meta, ref=at(0, blocks), seq_lens=at(blocks, streams),
                num_pages=at(blocks + streams, streams), tables=at(blocks + 2 * streams, streams * width).view(streams, width),
                kv=torch.randn(case["layers"], blocks, case["kv_heads"], PAGE, 2 * D, generator=g, device="cuda",
                               dtype=torch.bfloat16),
                src=ints(src), dst=ints(ended), every=torch.arange(streams, dtype=torch.int32, device="cuda"),
                grow=ints(grow), remap=torch.empty(blocks, dtype=torch.int32, device="cuda"),
                live=torch.empty(1, dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        _package()
        return _own[state["op"]](state)
    return _plain[state["op"]](state)


def _own_prefill(s):
    from flint_b200 import prefill_attention
    return prefill_attention.flint_prefill_attention(s["q"], s["kv"], s["tables"], s["cu_seqlens"], s["seq_lens"],
                                                     s["sinks"], s["window"], SCALE, s["out"])


def _own_shared(s):
    from flint_b200 import shared_prefix_attention
    return shared_prefix_attention.flint_shared_prefix_attention(s["q"], s["kv"], s["tables"], s["seq_lens"],
                                                                 s["group_starts"], s["prefix_lens"], s["sinks"],
                                                                 s["window"], SCALE, s["out"])


def _own_turnover(s):
    from flint_b200 import kv_pages
    s["meta"].copy_(s["saved"])
    pool = s["ref"], s["tables"], s["seq_lens"], s["num_pages"]
    kv_pages.flint_kv_free(*pool, s["dst"])
    kv_pages.flint_kv_fork(s["kv"], *pool, s["src"], s["dst"])
    kv_pages.flint_kv_reserve(*pool, s["every"], s["grow"])
    return [s["meta"], s["kv"]]


def _own_compact(s):
    from flint_b200 import kv_pages
    s["meta"].copy_(s["saved"])
    kv_pages.flint_kv_compact(s["kv"], s["ref"], s["tables"], s["num_pages"], s["remap"], s["live"])
    return [s["meta"], s["kv"], s["remap"], s["live"]]


def _visible(pos, keys, window):
    """Whether the query at position pos [n, 1] sees the keys at positions [k]."""
    ok = keys <= pos
    return ok & (keys > pos - window) if window else ok


def _attend(scores, ok, sinks):
    """Softmax of scores [..., heads, rows, keys] over the keys that ok lets through; a sink takes its share of the sum;
    a row that sees nothing gives zeros."""
    scores = scores.masked_fill(~ok, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks[:, None, None] - top)
    return p / total.masked_fill(top == -math.inf, 1)


def _plain_prefill(s):
    out, hkv = s["out"], s["kv"].shape[1]
    at = 0
    for b, n in enumerate(s["q_lens"]):
        kv = s["kv"][s["tables"][b, :_pages(s["lens"][b])].long()].transpose(0, 1).reshape(hkv, -1, 2 * D).float()
        # rows in blocks, so that the scores of a long prompt fit the memory; a block reads only the keys it may see
        for i in range(0, n, 1024):
            m, past = min(1024, n - i), s["lens"][b] - n + i
            lo = max(0, past - s["window"] + 1) if s["window"] else 0
            k, v = kv[:, lo:past + m, :D], kv[:, lo:past + m, D:]
            q = s["q"][at + i:at + i + m].float().transpose(0, 1).reshape(hkv, -1, D)
            keys = torch.arange(lo, past + m, device="cuda")
            pos = torch.arange(past, past + m, device="cuda")[:, None]
            p = _attend((q @ k.transpose(1, 2) * SCALE).view(s["heads"], m, -1), _visible(pos, keys, s["window"]),
                        s["sinks"])
            o = (p.view(hkv, -1, p.shape[-1]) @ v).view(s["heads"], m, D)
            out[at + i:at + i + m] = o.transpose(0, 1).to(out.dtype)
        at += n
    return out


def _plain_shared(s):
    out, hkv, at = s["out"], s["kv"].shape[1], 0
    g = s["heads"] // hkv
    for n, prefix in zip(s["groups"], s["prefix"]):
        first = prefix // PAGE
        rows = slice(at, at + n)
        tables, lens = s["tables"][rows], s["seq_lens"][rows, None]
        ends = max(first, 1, max(_pages(x) for x in s["lens"][rows]))
        q = s["q"][rows].float().view(n, hkv, g, D)
        shared = s["kv"][tables[0, :first].long()].transpose(0, 1).reshape(hkv, prefix, 2 * D).float()
        each = s["kv"][tables[:, first:ends].long()].transpose(1, 2).reshape(n, hkv, -1, 2 * D).float()
        near = torch.einsum("nhgd,hkd->nhgk", q, shared[..., :D])
        far = q @ each[..., :D].transpose(2, 3)
        keys = torch.arange(near.shape[-1] + far.shape[-1], device="cuda")
        ok = _visible(lens - 1, keys, s["window"])[:, None, None]
        scores = torch.cat([near, far], -1) * SCALE
        p = _attend(scores.view(n, s["heads"], 1, -1), ok, s["sinks"]).view(n, hkv, g, -1)
        # what the mask keeps out has the weight zero; cached values are finite
        o = torch.einsum("nhgk,hkd->nhgd", p[..., :prefix], shared[..., D:]) + p[..., prefix:] @ each[..., D:]
        out[rows] = o.reshape(n, s["heads"], D).to(out.dtype)
        at += n
    return out


def _lowest_free(ref):
    """Page ids, the free ones first, in rising order."""
    return torch.argsort((ref != 0).to(torch.uint8), stable=True)


def _add_refs(ref, pages, ok, by):
    return ref.index_add_(0, pages.clamp(min=0).flatten().long(), (ok * by).flatten().to(ref.dtype))


def _plain_turnover(s):
    s["meta"].copy_(s["saved"])
    ref, tables, lens, num, kv = s["ref"], s["tables"], s["seq_lens"], s["num_pages"], s["kv"]
    column = torch.arange(tables.shape[1], device="cuda")
    src, dst, every = s["src"].long(), s["dst"].long(), s["every"].long()
    # free
    _add_refs(ref, tables[dst], column < num[dst, None], -1)
    tables[dst], num[dst], lens[dst] = -1, 0, 0
    # fork: whole pages are shared, a page that is not full is copied into the lowest free page
    n = lens[src]
    whole, tail = n // PAGE, (n % PAGE != 0)
    fresh = _lowest_free(ref)[(tail.cumsum(0) - 1).clamp(min=0)].to(tables.dtype)
    last = tables[src].gather(1, whole.clamp(max=tables.shape[1] - 1).long()[:, None])[:, 0]
    fresh = torch.where(tail, fresh, last)
    rows = torch.where(column < whole[:, None], tables[src], -1)
    rows = torch.where((column == whole[:, None]) & tail[:, None], fresh[:, None], rows)
    _add_refs(ref, rows, rows >= 0, 1)
    tables[dst], num[dst], lens[dst] = rows, (whole + tail).to(num.dtype), n
    kv[:, fresh[tail].long()] = kv[:, last[tail].long()]
    # reserve: pages for the lengths to come, stream by stream from the lowest free page
    want = ((s["grow"] + PAGE - 1) // PAGE).to(num.dtype)
    missing = (want - num[every]).clamp(min=0)
    rank = (missing.cumsum(0) - missing)[:, None] + (column - num[every, None])
    new = (column >= num[every, None]) & (column < want[:, None])
    free = _lowest_free(ref).to(tables.dtype)
    rows = torch.where(new, free[rank.clamp(0, ref.numel() - 1).long()], tables[every])
    _add_refs(ref, rows, new, 1)
    tables[every], num[every] = rows, torch.maximum(want, num[every])
    return [s["meta"], kv]


def _plain_compact(s):
    s["meta"].copy_(s["saved"])
    ref, tables, kv = s["ref"], s["tables"], s["kv"]
    ids = torch.arange(ref.numel(), device="cuda")
    used = ref != 0
    live = used.sum()
    # the k-th used page behind the first `live` ids moves to the k-th free page among them
    move, hole = (used & (ids >= live)).nonzero()[:, 0], (~used & (ids < live)).nonzero()[:, 0]
    remap = ids.index_copy(0, move, hole)
    kv[:, hole] = kv[:, move]
    new = torch.zeros_like(ref).index_add_(0, remap, ref)
    ref.copy_(new)
    tables.copy_(torch.where(tables >= 0, remap[tables.clamp(min=0).long()].to(tables.dtype), tables))
    s["remap"].copy_(torch.where(used, remap, -1))
    s["live"].copy_(live.view(1))
    return [s["meta"], kv, s["remap"], s["live"]]


_plain = dict(prefill=_plain_prefill, shared=_plain_shared, turnover=_plain_turnover, compact=_plain_compact)


_own = dict(prefill=_own_prefill, shared=_own_shared, turnover=_own_turnover, compact=_own_compact)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def _seen(first, last, window):
    """Number of (query, key) pairs of queries at positions first .. last - 1."""
    if not window:
        return (first + 1 + last) * (last - first) // 2
    ramp = min(max(window - 1, first), last)             # below it a query sees all that is before it
    return (first + 1 + ramp) * (ramp - first) // 2 + (last - ramp) * window


def work(case):
    if case["op"] in ("turnover", "compact"):
        page, table = case["layers"] * case["kv_heads"] * PAGE * 2 * D * 2, 4
        if case["op"] == "turnover":
            # a tail page for each fork (its length decides whether there is one), the rows and counts that change
            width = _pages(case["prompt"] + case["grown"])
            return dict(bytes=2 * page * case["freed"] + table * (4 * width * case["freed"] + 4 * case["streams"]), flops=0)
        used = case["streams"] * case["pages"] * case["live"] / 100
        return dict(bytes=2 * page * used * (1 - used / case["blocks"])
                    + table * (2 * case["blocks"] + 2 * case["streams"] * case["pages"]), flops=0)
    token, row = case["kv_heads"] * 2 * D * 2, case["heads"] * D * 2
    if case["op"] == "prefill":
        bytes_, pairs = 0, 0
        for q, past in zip(_ints(case["q"]), _ints(case["past"])):
            if q:
                lo = max(0, past - case["window"] + 1) if case["window"] else 0
                bytes_ += 2 * q * row + (past + q - lo) * token
                pairs += _seen(past, past + q, case["window"])
        return dict(bytes=bytes_, flops=4 * D * case["heads"] * pairs)
    lens, prefix, at, bytes_, pairs = _ints(case["lens"]), _ints(case["prefix"]), 0, 0, 0
    for n, p in zip(_ints(case["groups"]), prefix):
        mine = [(max(0, x - case["window"]) if case["window"] else 0, x) for x in lens[at:at + n] if x]
        bytes_ += 2 * n * row + sum(max(0, x - max(p, lo)) for lo, x in mine) * token
        if mine:
            bytes_ += max(0, p - min(lo for lo, _ in mine)) * token
        pairs += sum(x - lo for lo, x in mine)
        at += n
    return dict(bytes=bytes_, flops=4 * D * case["heads"] * pairs)


# ---------------------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "turnover":
        return _exact_turnover(s)
    if case["op"] == "compact":
        return _exact_compact(s)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if case["op"] == "prefill":
        first = [sum(s["q_lens"][:b]) for b in range(len(s["q_lens"]))]
        for b, n in enumerate(s["q_lens"]):
            for i in range(0, n, 256):
                m = min(256, n - i)
                rows = slice(first[b] + i, first[b] + i + m)
                out[rows] = _exact_rows(s, b, s["q"][rows], range(s["lens"][b] - n + i, s["lens"][b] - n + i + m))
    else:
        for b, n in enumerate(s["lens"]):
            if n:
                out[b] = _exact_rows(s, b, s["q"][b:b + 1], range(n - 1, n))[0]
    return out


def _exact_rows(s, b, q, positions):
    """Attention of stream b's queries at these consecutive positions, straight from the sum over keys."""
    end = positions[-1] + 1
    slots = torch.arange(end, device="cuda")
    cached = s["kv"][s["tables"][b].long()[slots // PAGE], :, slots % PAGE]        # [keys, kv_heads, 256]
    rows = torch.empty(len(positions), s["heads"], D, dtype=torch.float64, device="cuda")
    group = s["heads"] // cached.shape[1]
    pos = torch.tensor(list(positions), device="cuda")[:, None]
    hidden = slots[None] > pos
    if s["window"]:
        hidden |= slots[None] <= pos - s["window"]
    for h in range(cached.shape[1]):
        k, v = cached[:, h, :D].double(), cached[:, h, D:].double()
        for j in range(h * group, (h + 1) * group):
            x = (q[:, j].double() @ k.T) / math.sqrt(D)
            x[hidden] = -math.inf
            if s["sinks"] is None:
                rows[:, j] = torch.softmax(x, 1) @ v
            else:
                sink = s["sinks"][j].double().expand(len(positions), 1)
                rows[:, j] = torch.softmax(torch.cat([x, sink], 1), 1)[:, :-1] @ v
    return rows


def _exact_turnover(s):
    ref, tables = s["ref"].tolist(), s["tables"].tolist()
    lens, num = s["seq_lens"].tolist(), s["num_pages"].tolist()
    fresh = lambda: ref.index(0)  # noqa: E731
    for d in s["dst"].tolist():
        for p in tables[d][:num[d]]:
            ref[p] -= 1
        tables[d], num[d], lens[d] = [-1] * len(tables[d]), 0, 0
    copies = []
    for b, d in zip(s["src"].tolist(), s["dst"].tolist()):
        lens[d] = lens[b]
        for p in range(lens[b] // PAGE):
            tables[d][p] = tables[b][p]
            ref[tables[b][p]] += 1
        num[d] = lens[b] // PAGE
        if lens[b] % PAGE:
            page = fresh()
            ref[page] = 1
            tables[d][num[d]] = page
            copies.append((tables[b][num[d]], page))
            num[d] += 1
    for b, n in zip(s["every"].tolist(), s["grow"].tolist()):
        while num[b] < _pages(n):
            page = fresh()
            ref[page] = 1
            tables[b][num[b]] = page
            num[b] += 1
    kv = s["kv"].clone()
    for a, b in copies:
        kv[:, b] = s["kv"][:, a]
    return [torch.tensor(ref + lens + num + [x for t in tables for x in t], dtype=torch.int32), kv]


def _exact_compact(s):
    ref, tables = s["ref"].tolist(), s["tables"].tolist()
    live = sum(r > 0 for r in ref)
    holes = [p for p in range(live) if not ref[p]]
    remap = [p if ref[p] else -1 for p in range(len(ref))]
    kv = s["kv"].clone()
    for p in range(live, len(ref)):
        if ref[p]:
            to = holes.pop(0)
            remap[p] = to
            kv[:, to] = s["kv"][:, p]
            ref[to], ref[p] = ref[p], 0
    flat = ref + s["seq_lens"].tolist() + s["num_pages"].tolist() + [remap[x] if x >= 0 else x for t in tables for x in t]
    return [torch.tensor(flat, dtype=torch.int32), kv, torch.tensor(remap, dtype=torch.int32),
            torch.tensor([live], dtype=torch.int32)]
