"""Prompt and shared-prefix attention over the paged cache against the definition in float64.

Tolerance, from the roundings the kernels are allowed (bf16 keeps 8 significant bits, so rounding to it moves a value by
up to 2^-8 of it): the probabilities go to bf16 (2^-8 of spread = sum p |v| / l in the result), the result goes to bf16
(2^-8 of it), and the 32-bit scores, exponentials and sums get 2^-11 of spread (scores of the inputs below stay under 64,
2^-17 of a score's units each).
"""
import numpy as np
import pytest
import torch

from helpers import bf16, dev_bf16, host, to_dev
from oracle import paged

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
D, PAGE, SCALE = 128, 16, 128 ** -0.5


def close(got, want, spread, what):
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -11) * spread + 1e-30
    bad = ~(np.abs(np.asarray(got, np.float64) - want) <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}: "
                           f"{np.asarray(got)[bad][0]} for {want[bad][0]}, tolerance {tol[bad][0]}")


def make_cache(rng, tables, owned, Hkv, poison=True):
    """Cache and block tables for streams whose pages `tables` were laid out; slots behind each length are NaN."""
    blocks = 1 + max([p for t in tables for p in t], default=0) + 5
    kv = bf16(rng, (blocks, Hkv, PAGE, 2 * D))
    if poison:
        used = np.zeros((blocks, PAGE), bool)
        for t, n in zip(tables, owned):
            for j in range(n):
                used[t[j // PAGE], j % PAGE] = True
        kv = np.where(used[:, None, :, None], kv, np.float32(np.nan))
    width = max(1, max(len(t) for t in tables))
    bt = np.full((len(tables), width), -1, np.int32)
    for b, t in enumerate(tables):
        bt[b, :len(t)] = t
    return kv, bt


def scattered(rng, counts):
    ids = rng.permutation(sum(counts) + 7).tolist()
    return [[ids.pop() for _ in range(n)] for n in counts]


def run_prefill(rng, q_lens, lens, Hkv, G, window, sinks, spare_rows=0, q_pad=0):
    from flint_b200 import prefill_attention as pa
    Hq, T = Hkv * G, sum(q_lens)
    tables = scattered(rng, [-(-n // PAGE) for n in lens])
    kv, bt = make_cache(rng, tables, lens, Hkv)
    q = bf16(rng, (T + spare_rows, Hq, D), 2.0)
    sk = (rng.standard_normal(Hq) * 2).astype(np.float32) if sinks else None
    qd = dev_bf16(np.concatenate([q.reshape(len(q), -1), np.zeros((len(q), q_pad), np.float32)], 1))
    qd = qd[:, :Hq * D].view(len(q), Hq, D) if not q_pad else qd.as_strided((len(q), Hq, D), (Hq * D + q_pad, D, 1))
    out = torch.full((len(q), Hq * D + q_pad), 7.0, dtype=torch.bfloat16, device="cuda")
    out = out.as_strided((len(q), Hq, D), (Hq * D + q_pad, D, 1))
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    args = (qd, dev_bf16(kv), to_dev(bt), to_dev(cu), to_dev(np.array(lens, np.int32)), to_dev(sk) if sinks else None,
            window or None, SCALE, out)
    assert pa.flint_prefill_attention(*args) is out
    torch.cuda.synchronize()
    got = host(out)
    want, spread = paged.prefill_attention(q[:T], kv, bt, q_lens, lens, sk, window, SCALE)
    close(got[:T], want, spread, f"prefill {q_lens} of {lens}")
    assert (got[T:] == 7.0).all(), "rows behind the last sequence were written"
    return args, out


@pytest.mark.parametrize("Hkv,G", [(1, 1), (4, 8), (2, 3), (1, 5), (2, 7), (3, 2)])
@pytest.mark.parametrize("q_lens,past", [([1], [0]), ([17], [0]), ([130], [0]), ([3, 0, 64, 1, 33], [40, 5, 0, 0, 200])])
def test_prefill_heads(fb, Hkv, G, q_lens, past):
    rng = np.random.default_rng(Hkv * 100 + G + sum(q_lens))
    run_prefill(rng, q_lens, [a + b for a, b in zip(q_lens, past)], Hkv, G, 0, False)


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("window", [1, 16, 100, 513])
def test_prefill_window(fb, window, sinks):
    rng = np.random.default_rng(window)
    run_prefill(rng, [140, 1, 20], [140, 700, 333], 2, 4, window, sinks)


@pytest.mark.parametrize("length", [15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
def test_prefill_page_and_tile_ends(fb, length):
    rng = np.random.default_rng(length)
    run_prefill(rng, [min(9, length), length], [length, length], 1, 8, 0, True)


@pytest.mark.parametrize("q_lens,lens", [([4], [9000]), ([1, 5, 2], [4097, 3000, 20]), ([1], [20011]), ([40], [5000])])
def test_prefill_few_rows_on_a_long_cache(fb, q_lens, lens):
    rng = np.random.default_rng(lens[0])
    run_prefill(rng, q_lens, lens, 2, 8, 0, True)


def test_prefill_rows_before_the_cache(fb):
    """More query tokens than cached ones: the first rows see nothing and give zeros, with and without sinks."""
    for sinks in (False, True):
        _, out = run_prefill(np.random.default_rng(5), [40, 6], [33, 0], 2, 4, 0, sinks)
        assert (host(out)[:7] == 0).all() and (host(out)[40:46] == 0).all()


def test_prefill_strided_rows_and_spare_rows(fb):
    rng = np.random.default_rng(6)
    run_prefill(rng, [50, 3], [50, 90], 2, 2, 0, False, spare_rows=9, q_pad=512)


def test_prefill_strided_cache(fb):
    """One layer of a cache whose pages hold all layers side by side: strides other than the tested ones."""
    from flint_b200 import prefill_attention as pa
    rng = np.random.default_rng(8)
    every = bf16(rng, (9, 3, 2, PAGE, 2 * D))
    bt, q, lens = np.array([[4, 1, 7, 0, 2]], np.int32), bf16(rng, (70, 8, D)), [70]
    out = torch.empty((70, 8, D), dtype=torch.bfloat16, device="cuda")
    pa.flint_prefill_attention(dev_bf16(q), dev_bf16(every)[:, 1], to_dev(bt), to_dev(np.array([0, 70], np.int32)),
                               to_dev(np.array(lens, np.int32)), None, None, SCALE, out)
    want, spread = paged.prefill_attention(q, every[:, 1], bt, lens, lens, None, 0, SCALE)
    close(host(out), want, spread, "strided cache")


@pytest.mark.parametrize("shift", [0.0, 60.0, -60.0])
def test_prefill_rising_scores_and_extreme_sinks(fb, shift):
    """Scores that keep rising along the keys (each step has a new maximum), with sinks far above, far below and absent
    (-inf) for single heads."""
    from flint_b200 import prefill_attention as pa
    rng = np.random.default_rng(9)
    n, Hkv, G = 400, 1, 4
    kv, bt = make_cache(rng, [list(range(25))], [n], Hkv, poison=False)
    ramp = np.linspace(-30, 30, n)
    q = bf16(rng, (n, G, D), 0.05)
    q[..., 0] = 8.0
    kv[:25, 0, :, 0] = ramp.reshape(25, 16) * (1 if shift >= 0 else -1)
    kv, q = kv.astype(np.float32), q.astype(np.float32)
    kv = host(dev_bf16(kv))
    q = host(dev_bf16(q))
    sk = np.array([shift, -np.inf, 2.0, shift], np.float32)
    out = torch.empty((n, G, D), dtype=torch.bfloat16, device="cuda")
    pa.flint_prefill_attention(dev_bf16(q), dev_bf16(kv), to_dev(bt), to_dev(np.array([0, n], np.int32)),
                               to_dev(np.array([n], np.int32)), to_dev(sk), None, SCALE, out)
    want, spread = paged.prefill_attention(q, kv, bt, [n], [n], sk, 0, SCALE)
    close(host(out), want, spread, "rising scores")


def test_prefill_graph_replay_and_streams(fb):
    """Captured calls follow lengths that change between replays; a call on another stream gives the same bits."""
    from flint_b200 import prefill_attention as pa
    rng = np.random.default_rng(10)
    args, out = run_prefill(rng, [5, 90, 1], [3000, 90, 700], 2, 8, 0, True)
    first = host(out).copy()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pa.flint_prefill_attention(*args)
    lens = args[4].clone()
    for step in (0, 1, 0):
        args[4].copy_(lens - step)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(out), first) == (step == 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.zero_()
        pa.flint_prefill_attention(*args)
    side.synchronize()
    np.testing.assert_array_equal(host(out), first)


def test_prefill_bad_lengths_are_reported(fb):
    from flint_b200 import prefill_attention as pa
    fb._lib.check_device_status()
    kv = torch.zeros((4, 1, PAGE, 2 * D), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((4, 2, D), dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    bt = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for cu, lens in ((i32(0, 4), i32(33)), (i32(0, 9), i32(9)), (i32(0, -1), i32(4))):
        pa.flint_prefill_attention(q, kv, bt, cu, lens, None, None, SCALE, out)
        with pytest.raises(fb._lib.FlintError, match="longer than its block table"):
            fb._lib.check_device_status()
    # a block id outside the cache reads as zeros
    bt.fill_(99)
    pa.flint_prefill_attention(q + 1, kv + 1, bt, i32(0, 4), i32(4), None, None, SCALE, out)
    assert (host(out) == 0).all()
    fb._lib.check_device_status()


# ---- shared prefix ----
def run_shared(rng, groups, prefix, lens, Hkv, G, window, sinks, poison=True):
    from flint_b200 import shared_prefix_attention as sp
    Hq, B = Hkv * G, sum(groups)
    of = [g for g, n in enumerate(groups) for _ in range(n)]
    ids = rng.permutation(sum(p // PAGE for p in prefix) + sum(-(-n // PAGE) for n in lens) + 9).tolist()
    first = [[ids.pop() for _ in range(p // PAGE)] for p in prefix]
    tables = [first[g] + [ids.pop() for _ in range(max(0, -(-n // PAGE) - prefix[g] // PAGE))] for g, n in zip(of, lens)]
    owned = [max(n, prefix[g] // PAGE * PAGE) for g, n in zip(of, lens)]
    kv, bt = make_cache(rng, tables, owned, Hkv, poison)
    q = bf16(rng, (B, Hq, D), 2.0)
    sk = (rng.standard_normal(Hq) * 2).astype(np.float32) if sinks else None
    out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device="cuda")
    starts = np.concatenate([[0], np.cumsum(groups)]).astype(np.int32)
    args = (dev_bf16(q), dev_bf16(kv), to_dev(bt), to_dev(np.array(lens, np.int32)), to_dev(starts),
            to_dev(np.array(prefix, np.int32)), to_dev(sk) if sinks else None, window or None, SCALE, out)
    assert sp.flint_shared_prefix_attention(*args) is out
    torch.cuda.synchronize()
    want, spread = paged.prefill_attention(q, kv, bt, [1] * B, lens, sk, window, SCALE)
    close(host(out), want, spread, f"shared {groups} {prefix}")
    return args, out


@pytest.mark.parametrize("Hkv,G", [(1, 1), (4, 8), (2, 3), (1, 5), (2, 7)])
@pytest.mark.parametrize("groups,prefix,lens", [
    ([1], [0], [1]), ([2], [32], [33, 48]), ([3], [256], [300, 271, 257]), ([5], [100], [97, 130, 112, 113, 0]),
    ([2, 1, 4], [64, 0, 320], [70, 81, 9, 321, 322, 400, 336])])
def test_shared_heads(fb, Hkv, G, groups, prefix, lens):
    run_shared(np.random.default_rng(Hkv * 10 + G + len(lens)), groups, prefix, lens, Hkv, G, 0, G % 2 == 1)


@pytest.mark.parametrize("window", [1, 16, 40, 300])
def test_shared_window(fb, window):
    run_shared(np.random.default_rng(window), [4, 2], [512, 48], [513, 530, 700, 600, 49, 200], 2, 4, window, True)


def test_shared_window_forgets_the_prefix(fb):
    """Pages that lie behind every window may have been given away: their ids are not looked at."""
    from flint_b200 import shared_prefix_attention as sp
    args, out = run_shared(np.random.default_rng(3), [3], [640], [900, 870, 800], 2, 4, 64, False)
    args[2][:, :30] = -1
    was = host(out).copy()
    sp.flint_shared_prefix_attention(*args)
    np.testing.assert_array_equal(host(out), was)


@pytest.mark.parametrize("n,prefix", [(16, 4096), (17, 1000), (33, 2048), (70, 528)])
def test_shared_many_streams(fb, n, prefix):
    rng = np.random.default_rng(n)
    run_shared(rng, [n], [prefix], [prefix + 1 + 3 * i % 50 for i in range(n)], 1, 8, 0, True)


def test_shared_long_prefix(fb):
    run_shared(np.random.default_rng(12), [2], [20000], [20003, 20033], 1, 8, 0, False, poison=False)


def test_shared_prefix_longer_than_a_stream(fb):
    """A stream that ends inside the shared prefix sees its own length only."""
    run_shared(np.random.default_rng(13), [4], [256], [256, 100, 17, 300], 2, 4, 0, True)


def test_shared_long_suffixes(fb):
    run_shared(np.random.default_rng(14), [2, 1], [64, 0], [5000, 70, 3000], 2, 8, 0, False)


def test_shared_many_short_suffixes(fb):
    """Several items to a block, of one, two, three and more steps each, in every order."""
    rng = np.random.default_rng(16)
    lens = [64 + int(x) for x in rng.integers(0, 520, size=150)] + [int(x) for x in rng.integers(0, 400, size=90)]
    run_shared(rng, [150, 90], [64, 0], lens, 8, 2, 0, True)


def test_prefill_many_short_sequences(fb):
    rng = np.random.default_rng(17)
    q_lens = [int(x) for x in rng.integers(0, 40, size=60)]
    run_prefill(rng, q_lens, [n + int(x) for n, x in zip(q_lens, rng.integers(0, 500, size=60))], 8, 4, 0, False)


def test_shared_graph_replay(fb):
    from flint_b200 import shared_prefix_attention as sp
    args, out = run_shared(np.random.default_rng(15), [6, 2], [1024, 0], [1030, 1100, 0, 1025, 1200, 1024, 40, 7], 2, 8, 0,
                           True)
    first = host(out).copy()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sp.flint_shared_prefix_attention(*args)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(host(out), first)


def test_shared_bad_groups_are_reported(fb):
    from flint_b200 import shared_prefix_attention as sp
    fb._lib.check_device_status()
    kv = torch.zeros((4, 1, PAGE, 2 * D), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((3, 2, D), dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    bt = i32(0, 1, 0, 2, 0, 3).view(3, 2)
    for lens, starts, prefix in ((i32(20, 20, 40), i32(0, 3), i32(16)), (i32(20, 20, 20), i32(0, 3), i32(64)),
                                 (i32(20, 20, 20), i32(0, 5), i32(16)), (i32(20, 20, 20), i32(2, 3), i32(-4))):
        sp.flint_shared_prefix_attention(q, kv, bt, lens, starts, prefix, None, None, SCALE, out)
        with pytest.raises(fb._lib.FlintError, match="longer than its block table"):
            fb._lib.check_device_status()


# ---- what no query sees ----
def forget(kv, bt, dead):
    """NaN in the first dead[b] tokens of stream b."""
    bt = bt.cpu()
    for b, n in enumerate(dead):
        for j in range(max(0, n)):
            kv[int(bt[b, j // PAGE]), :, j % PAGE] = float("nan")


@pytest.mark.parametrize("window", [1, 3, 5, 37, 100, 131, 300])
@pytest.mark.parametrize("q_lens,lens", [([1, 20, 3, 1, 2], [700, 140, 33, 10, 16]), ([300], [900]), ([1], [5000])])
def test_prefill_window_leaves_anything_behind(fb, window, q_lens, lens):
    from flint_b200 import prefill_attention as pa
    args, out = run_prefill(np.random.default_rng(window + len(lens)), q_lens, lens, 2, 4, window, True)
    was = host(out).copy()
    forget(args[1], args[2], [n - q - window + 1 for q, n in zip(q_lens, lens)])
    out.zero_()
    pa.flint_prefill_attention(*args)
    np.testing.assert_array_equal(host(out), was)


@pytest.mark.parametrize("window", [1, 6, 40, 100, 250])
@pytest.mark.parametrize("groups,prefix,lens", [([3, 2], [512, 64], [513, 530, 521, 75, 190]), ([40], [2048], list(range(2050, 2090))),
                                                ([1, 1], [0, 0], [10, 300])])
def test_shared_window_leaves_anything_behind(fb, window, groups, prefix, lens):
    from flint_b200 import shared_prefix_attention as sp
    args, out = run_shared(np.random.default_rng(window + len(lens)), groups, prefix, lens, 2, 4, window, False)
    was = host(out).copy()
    dead, at = [], 0
    for n, p in zip(groups, prefix):
        first = min(lens[at:at + n]) - window                     # of the shared pages, what the group's shortest stream sees
        dead += [min(first, p) if lens[b] - window < p else lens[b] - window if first >= p else 0 for b in range(at, at + n)]
        at += n
    forget(args[1], args[2], dead)
    out.zero_()
    sp.flint_shared_prefix_attention(*args)
    np.testing.assert_array_equal(host(out), was)


@pytest.mark.parametrize("lens", [[0, 300, 17, 290], [40, 0, 0, 261], [256, 255, 270, 0]])
def test_shared_tables_end_with_their_streams(fb, lens):
    """Padded and short streams, first in their group too, whose tables do not name the whole prefix."""
    from flint_b200 import shared_prefix_attention as sp
    args, out = run_shared(np.random.default_rng(21), [4], [256], lens, 2, 8, 0, True)
    was = host(out).copy()
    for b, n in enumerate(lens):
        args[2][b, -(-n // PAGE):] = -1
    out.zero_()
    sp.flint_shared_prefix_attention(*args)
    np.testing.assert_array_equal(host(out), was)


# ---- refusals on the host ----
def test_refusals(fb):
    from flint_b200 import prefill_attention as pa
    from flint_b200 import shared_prefix_attention as sp
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device="cuda")
    i = lambda *s: z(*s, dt=torch.int32)
    good = dict(q=z(4, 8, D), kv_cache=z(3, 2, PAGE, 2 * D), block_tables=i(2, 3), cu_seqlens=i(3), seq_lens=i(2), sinks=None,
                window=None, scale=SCALE, out=z(4, 8, D))
    pa.flint_prefill_attention(**good)
    bad = [dict(q=z(4, 8, 64)), dict(q=z(4, 8, D, dt=torch.float16)), dict(q=z(4, 8, 2 * D)[..., ::2]),
           dict(q=z(4, 9, D), out=z(4, 9, D)), dict(q=z(4, 18, D), out=z(4, 18, D)), dict(out=z(4, 8, D, dt=torch.float32)),
           dict(out=z(5, 8, D)), dict(kv_cache=z(3, 2, 32, 2 * D)), dict(kv_cache=z(3, 2, PAGE, 2 * D, dt=torch.float16)),
           dict(kv_cache=z(3, PAGE, 2, 2 * D).transpose(1, 2)), dict(block_tables=i(2, 3).long()), dict(block_tables=i(1, 3)),
           dict(cu_seqlens=i(2)), dict(seq_lens=i(2).long()), dict(sinks=z(8)), dict(sinks=z(7, dt=torch.float32)),
           dict(window=-1), dict(out=None), dict(cu_seqlens=i(3).cpu()), dict(seq_lens=i(2).cpu())]
    for change in bad:
        args = {**good, **change}
        if args["out"] is None:
            args["out"] = args["q"]                               # in place
        with pytest.raises(fb._lib.FlintError):
            pa.flint_prefill_attention(**args)
    good = dict(q=z(2, 8, D), kv_cache=z(3, 2, PAGE, 2 * D), block_tables=i(2, 3), seq_lens=i(2),
                group_starts=torch.tensor([0, 2], dtype=torch.int32, device="cuda"), prefix_lens=i(1), sinks=None, window=None,
                scale=SCALE, out=z(2, 8, D))
    sp.flint_shared_prefix_attention(**good)
    for change in [dict(q=z(3, 8, D), out=z(3, 8, D)), dict(group_starts=i(3)), dict(prefix_lens=i(3), group_starts=i(4)),
                   dict(prefix_lens=i(1).long()), dict(out=z(2, 8, D).cpu()), dict(q=z(2, 8 * D + 4)[:, 4:].view(2, 8, D),)]:
        with pytest.raises((fb._lib.FlintError, RuntimeError)):
            sp.flint_shared_prefix_attention(**{**good, **change})
    torch.cuda.synchronize()
    fb._lib.device_status(clear=True)


def test_registered_ops_and_widest_window(fb):
    """torch.ops gives the shim's bits; a window wider than any length is no window; out may lie at 16 bytes."""
    from flint_b200 import prefill_attention as pa
    args, out = run_prefill(np.random.default_rng(20), [40, 70], [40, 300], 2, 4, 0, True)
    first = host(out).copy()
    torch.ops.flint_b200.prefill_attention(*args[:6], 0, SCALE, out.zero_())
    np.testing.assert_array_equal(host(out), first)
    for window in (2 ** 31 - 1, 2 ** 40, 16 * args[2].shape[1]):
        pa.flint_prefill_attention(*args[:6], window, SCALE, out.zero_())
        np.testing.assert_array_equal(host(out), first)
    odd = torch.zeros(out.numel() + 8, dtype=torch.bfloat16, device="cuda")[8:].view(out.shape)
    assert odd.data_ptr() % 32 == 16
    pa.flint_prefill_attention(*args[:8], odd)
    np.testing.assert_array_equal(host(odd), first)


def test_no_rows(fb):
    from flint_b200 import prefill_attention as pa
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device="cuda")
    out = z(0, 8, D)
    assert pa.flint_prefill_attention(z(0, 8, D), z(3, 2, PAGE, 2 * D), z(1, 3, dt=torch.int32), z(2, dt=torch.int32),
                                      z(1, dt=torch.int32), None, None, SCALE, out) is out
