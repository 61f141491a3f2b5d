"""Prompt and shared-prefix attention and the page operations at their edges: values that are not numbers, tables that end
before their streams do, batches of many sequences, long prompts, and calls that follow one another without a pause."""
import numpy as np
import pytest
import torch

from helpers import bf16, dev_bf16, host, to_dev
from oracle import paged
from test_paged_attention_gpu import D, PAGE, SCALE, close, make_cache, run_prefill, run_shared, scattered

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


# ---- values that are not numbers ----
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("q_lens,lens,window", [([17], [17], 0), ([40, 3], [300, 40], 0), ([2], [9000], 0), ([150], [400], 37),
                                                ([20], [12], 0)])
def test_prefill_query_that_is_not_a_number(fb, q_lens, lens, window, sinks):
    """A row of q with a NaN gives NaN where it sees keys (zeros where it sees none); no other row changes a bit."""
    from flint_b200 import prefill_attention as pa
    args, out = run_prefill(np.random.default_rng(31 + len(lens)), q_lens, lens, 2, 4, window, sinks)
    want = host(out).copy()
    for row, head in ((0, 3), (1, 0), (q_lens[0] - 1, 7)):
        args[0][row, head, 5] = float("nan")
        if lens[0] - q_lens[0] + row >= 0:
            want[row, head] = np.nan
    out.zero_()
    pa.flint_prefill_attention(*args)
    np.testing.assert_array_equal(host(out), want)


@pytest.mark.parametrize("first,last", [(4096, 4097), (4000, 5000), (0, 9000), (8999, 9000), (100, 8900)])
def test_prefill_keys_that_are_not_numbers(fb, first, last):
    """Keys of NaN in a long cache reach every row that sees one of them, wherever the line of items is cut."""
    from flint_b200 import prefill_attention as pa
    n, rows = 9000, 3
    args, out = run_prefill(np.random.default_rng(33), [rows, 5], [n, 40], 2, 8, 0, True)
    want, bt = host(out).copy(), args[2].cpu()
    for j in range(first, last):
        args[1][int(bt[0, j // PAGE]), 1, j % PAGE, 7] = float("nan")
    want[[i for i in range(rows) if n - rows + i >= first], 8:] = np.nan
    out.zero_()
    pa.flint_prefill_attention(*args)
    np.testing.assert_array_equal(host(out), want)


@pytest.mark.parametrize("first,last", [(0, 1024), (300, 301), (1030, 1090)])
def test_shared_keys_and_queries_that_are_not_numbers(fb, first, last):
    from flint_b200 import shared_prefix_attention as sp
    lens = [1030, 1100, 0, 1025, 1200, 1024]
    args, out = run_shared(np.random.default_rng(34), [6], [1024], lens, 2, 8, 0, True)
    want, bt = host(out).copy(), args[2].cpu()
    for j in range(first, last):
        args[1][int(bt[4, j // PAGE]), 0, j % PAGE, 100] = float("nan")
    args[0][:3, 11, 0] = float("nan")
    for b, n in enumerate(lens):
        if n > first and (first < 1024 or b == 4):                # (stream 4's own keys are its alone)
            want[b, :8] = np.nan
        if b < 3 and n:
            want[b, 11] = np.nan
    out.zero_()
    sp.flint_shared_prefix_attention(*args)
    np.testing.assert_array_equal(host(out), want)


# ---- tables that end before their streams do ----
def test_missing_pages_are_reported(fb):
    """A page below a row's length whose table entry is negative is a sequence longer than its table; entries that no row
    looks at are not."""
    from flint_b200 import prefill_attention as pa
    from flint_b200 import shared_prefix_attention as sp
    fb._lib.check_device_status()
    report = lambda: pytest.raises(fb._lib.FlintError, match="longer than its block table")
    for column, window, bad in ((0, 0, True), (18, 0, True), (12, 70, False), (12, 80, True)):
        args, _ = run_prefill(np.random.default_rng(41), [5, 20], [290, 300], 2, 4, window, False)
        fb._lib.check_device_status()
        args[2][1, column] = -1
        pa.flint_prefill_attention(*args)
        if bad:
            with report():
                fb._lib.check_device_status()
        fb._lib.check_device_status()
    for column, streams, window, bad in ((3, [0, 1, 2], 0, True), (17, [1], 0, True), (3, [0, 1, 2], 64, False),
                                         (17, [0], 0, False)):
        args, _ = run_shared(np.random.default_rng(42), [3], [256], [270, 290, 260], 2, 4, window, False)
        fb._lib.check_device_status()
        args[2][streams, column] = -1
        sp.flint_shared_prefix_attention(*args)
        if bad:
            with report():
                fb._lib.check_device_status()
        fb._lib.check_device_status()


def test_pages_between_windows_may_be_gone(fb):
    """Streams that end inside a shared prefix under a window: the shared pages between their keys are seen by no row, and a
    table that has given them away is no fault."""
    from flint_b200 import shared_prefix_attention as sp
    fb._lib.check_device_status()
    for lens, gone in (([300, 1000, 990], range(19, 32)), ([100, 500, 490], range(7, 26))):
        args, out = run_shared(np.random.default_rng(43), [3], [512], lens, 2, 4, 64, True)
        was = host(out).copy()
        args[2][:, list(gone)] = -1
        sp.flint_shared_prefix_attention(*args)
        np.testing.assert_array_equal(host(out), was)
        fb._lib.check_device_status()


# ---- what autograd is told ----
def test_calls_are_seen_by_autograd(fb):
    """Written tensors count a version, as through the registered ops."""
    from flint_b200 import kv_pages
    from flint_b200 import prefill_attention as pa
    from flint_b200 import shared_prefix_attention as sp
    args, out = run_prefill(np.random.default_rng(51), [5], [30], 2, 4, 0, False)
    was = out._version
    pa.flint_prefill_attention(*args)
    assert out._version > was
    saved = torch.ones_like(out, requires_grad=True)
    product = (saved * out).sum()                                 # keeps out for its backward pass
    pa.flint_prefill_attention(*args)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    args, out = run_shared(np.random.default_rng(52), [2], [32], [40, 50], 2, 4, 0, False)
    was = out._version
    sp.flint_shared_prefix_attention(*args)
    assert out._version > was
    pool = kv_pages.PagePool(torch.zeros((1, 9, 1, PAGE, 256), dtype=torch.bfloat16, device="cuda"), 3, 4)
    versions = lambda: [t._version for t in (pool.kv, *pool.state, pool.remap, pool.live)]
    for call, written in ((lambda: pool.reserve([0], [40]), [0, 1, 1, 0, 1, 0, 0]), (lambda: pool.fork([0], [1]), [1, 1, 1, 1, 1, 0, 0]),
                          (lambda: pool.free([0]), [0, 1, 1, 1, 1, 0, 0]), (lambda: pool.compact(), [1, 1, 1, 0, 0, 1, 1])):
        was = versions()
        call()
        assert [int(b > a) for a, b in zip(was, versions())] == written


# ---- page operations on tables that do not fit ----
@pytest.mark.parametrize("column,entry", [(0, -1), (1, 99), (2, -7), (2, 40)])
def test_fork_of_a_bad_table_is_left_out_whole(fb, column, entry):
    """An id outside the pool among the source's full pages (0, 1) or as its started page (2): no child, no page taken, the
    other forks of the call as ever."""
    from flint_b200 import kv_pages
    fb._lib.device_status(clear=True)
    kv = torch.randn((2, 40, 1, PAGE, 256), device="cuda").bfloat16()
    pool = kv_pages.PagePool(kv, 6, 9)
    pool.reserve([2, 4], [45, 20])
    pool.seq_lens.copy_(torch.tensor([0, 0, 45, 0, 20, 0], dtype=torch.int32))
    pool.block_tables[2, column] = entry
    before = [t.clone() for t in pool.state]
    pool.fork([2, 4, 2], [0, 3, 5])
    with pytest.raises(fb._lib.FlintError, match="did not fit"):
        fb._lib.check_device_status()
    ref, tables, lens, num = (t.clone() for t in pool.state)
    for s in (0, 5):
        assert num[s] == 0 and lens[s] == 0 and (tables[s] == -1).all()
    child = int(tables[3, 1])
    assert num[3] == 2 and lens[3] == 20 and tables[3, 0] == before[1][4, 0] and torch.equal(kv[:, child], kv[:, int(tables[4, 1])])
    want = before[0].clone()
    want[int(tables[4, 0])] += 1
    want[child] += 1
    assert torch.equal(ref, want) and (before[0][child] == 0)
    assert all(torch.equal(a[[1, 2, 4]], b[[1, 2, 4]]) for a, b in zip((tables, lens, num), before[1:]))


def test_refusals_keep_their_place_and_repeats_are_freed_once(fb):
    from flint_b200 import kv_pages
    fb._lib.device_status(clear=True)
    pool = kv_pages.PagePool(torch.zeros((1, 6, 1, PAGE, 256), dtype=torch.bfloat16, device="cuda"), 5, 4)
    pool.reserve([0, 1, 2, 3, 4], [40, 64, 16, 0, 10])            # 3 of 6; 4 of 3: refused, and so are 2 and 4
    assert pool.num_pages.tolist() == [3, 0, 0, 0, 0] and pool.ref.tolist() == [1, 1, 1, 0, 0, 0]
    with pytest.raises(fb._lib.FlintError, match="fewer pages were free"):
        fb._lib.check_device_status()
    pool.free([0, 0, 3])
    assert pool.num_pages.tolist() == [0] * 5 and pool.ref.tolist() == [0] * 6
    fb._lib.check_device_status()


# ---- many sequences, long prompts, head groups ----
@pytest.mark.parametrize("batch", [1100, 2100])
def test_prefill_many_sequences(fb, batch):
    """More sequences than are kept in shared memory while the items are cut (2,048), and more than one lane-full of runs."""
    rng = np.random.default_rng(batch)
    q_lens = [int(x) for x in rng.integers(0, 4, size=batch)]
    run_prefill(rng, q_lens, [n + int(x) for n, x in zip(q_lens, rng.integers(0, 50, size=batch))], 1, 2, 0, True)


@pytest.mark.parametrize("groups", [600, 1100])
def test_shared_many_groups(fb, groups):
    rng = np.random.default_rng(groups)
    sizes = [1 if i % 7 else 2 for i in range(groups)]
    prefix = [int(x) * PAGE for x in rng.integers(0, 4, size=groups)]
    lens = [p + int(x) for p, n in zip(prefix, sizes) for x in rng.integers(0, 40, size=n)]
    run_shared(rng, sizes, prefix, lens, 1, 2, 0, False)


@pytest.mark.parametrize("n,past,Hkv,G,window", [(4100, 0, 4, 8, 0), (5003, 0, 1, 3, 0), (2050, 6001, 2, 8, 0),
                                                 (4500, 333, 2, 4, 700)])
def test_prefill_long_prompts(fb, n, past, Hkv, G, window):
    """Prompts of many items to a block, compared at the rows beside every item's ends and at random ones."""
    from flint_b200 import prefill_attention as pa
    rng = np.random.default_rng(n)
    tables = scattered(rng, [-(-(n + past) // PAGE)])
    kv, bt = make_cache(rng, tables, [n + past], Hkv)
    q = bf16(rng, (n, Hkv * G, D), 2.0)
    out = torch.empty((n, Hkv * G, D), dtype=torch.bfloat16, device="cuda")
    pa.flint_prefill_attention(dev_bf16(q), dev_bf16(kv), to_dev(bt), to_dev(np.array([0, n], np.int32)),
                               to_dev(np.array([n + past], np.int32)), None, window or None, SCALE, out)
    got, tile = host(out), 2 * (128 // G)
    assert np.isfinite(got).all()
    rows = sorted({0, n - 1, *rng.integers(0, n, size=40).tolist(),
                   *[r for i in rng.integers(1, n // tile, size=15).tolist() for r in (i * tile - 1, i * tile)]})
    k, v = paged.cached(kv, bt[0], n + past)
    for r in rows:
        want, spread = paged.attention_rows(q[r:r + 1], k, v, past + r, None, window, SCALE)
        close(got[r:r + 1], want, spread, f"row {r} of {n}")


@pytest.mark.parametrize("Hkv", [1, 3])
def test_six_heads_to_a_group(fb, Hkv):
    run_prefill(np.random.default_rng(61), [3, 0, 64, 1, 33], [43, 5, 64, 1, 233], Hkv, 6, 0, True)
    run_shared(np.random.default_rng(62), [2, 1, 4], [64, 0, 320], [70, 81, 9, 321, 322, 400, 336], Hkv, 6, 0, True)


# ---- calls that follow one another without a pause ----
def test_attention_right_behind_page_operations(fb):
    """The decode attention looks at lengths, tables and older pages before its wait on the call before it: what it reads
    right behind a fork, a compaction or a reservation is what it reads after a pause."""
    from flint_b200 import decode_attention as da
    from flint_b200 import kv_pages
    rng = np.random.default_rng(71)
    kv = torch.randn((24, 700, 4, PAGE, 2 * D), device="cuda").bfloat16()
    q = dev_bf16(bf16(rng, (1, 32, D))).expand(8, -1, -1).contiguous()
    n = 1003
    for turn in range(12):
        pool = kv_pages.PagePool(kv, 8, 80)
        pool.reserve([6, 3], [160, n])                            # a stream in front, so that compaction moves pages
        pool.seq_lens[3] = n
        others = torch.tensor([0, 1, 2, 4, 5, 7], dtype=torch.int32, device="cuda")
        source, gone = torch.full_like(others, 3), torch.tensor([6], dtype=torch.int32, device="cuda")
        outs = [torch.empty_like(q) for _ in range(3)]
        torch.cuda.synchronize()
        pool.fork(source, others)
        da.flint_decode_attention(q, kv[turn], pool.block_tables, pool.seq_lens, None, None, SCALE, outs[0])
        pool.free(gone)
        da.flint_decode_attention(q, kv[turn], pool.block_tables, pool.seq_lens, None, None, SCALE, outs[1])
        pool.compact()
        da.flint_decode_attention(q, kv[turn], pool.block_tables, pool.seq_lens, None, None, SCALE, outs[2])
        after = torch.empty_like(q)
        torch.cuda.synchronize()
        da.flint_decode_attention(q, kv[turn], pool.block_tables, pool.seq_lens, None, None, SCALE, after)
        others = others.long().tolist()
        for o in outs + [after]:
            for b in (3, *others):
                np.testing.assert_array_equal(host(o[b]), host(after[3]), err_msg=f"turn {turn}, stream {b}")
            assert (host(o[6]) == 0).all()
