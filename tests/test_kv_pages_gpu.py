"""The page pool on the device against its plain restatement: states and caches have to be equal."""
import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


def make(seed, layers=2, blocks=40, Hkv=1, streams=6, max_blocks=9, spread=False):
    from flint_b200 import kv_pages
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = torch.randn((layers, blocks, Hkv, 16, 256), generator=g, device="cuda", dtype=torch.bfloat16)
    if spread:                                       # a cache whose layers are strides apart
        big = torch.zeros((layers, blocks + 3, Hkv, 16, 256), dtype=torch.bfloat16, device="cuda")
        big[:, :blocks] = kv
        kv = big[:, :blocks]
    pool = kv_pages.PagePool(kv, streams, max_blocks)
    return pool, paged.Pool(kv.float().cpu().numpy(), streams, max_blocks)


def set_lens(pool, plain, lens):
    plain.lens = list(lens)
    pool.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))


def same(fb, pool, plain, what=""):
    torch.cuda.synchronize()
    assert pool.ref.tolist() == plain.ref, what
    assert pool.seq_lens.tolist() == plain.lens, what
    assert pool.num_pages.tolist() == [len(t) for t in plain.tables], what
    width = pool.block_tables.shape[1]
    assert pool.block_tables.tolist() == [t + [-1] * (width - len(t)) for t in plain.tables], what
    np.testing.assert_array_equal(pool.kv.float().cpu().numpy(), plain.kv, err_msg=what)
    bits = fb._lib.device_status(clear=True)
    assert sum(bits.values()) == plain.bad, (what, bits, plain.bad)
    plain.bad = 0


@pytest.mark.parametrize("seed", range(6))
def test_random_walk(fb, seed):
    """Random calls, among them ids out of range, streams named twice, full pools and empty lists of work."""
    fb._lib.device_status(clear=True)
    rng = np.random.default_rng(seed)
    S, width = int(rng.integers(2, 12)), int(rng.integers(1, 12))
    pool, plain = make(seed, layers=int(rng.integers(1, 4)), blocks=int(rng.integers(3, 60)), Hkv=int(rng.integers(1, 4)),
                       streams=S, max_blocks=width, spread=seed % 2 == 1)
    for step in range(40):
        op = rng.choice(["reserve", "reserve", "fork", "fork", "free", "compact"])
        n = int(rng.integers(1, S + 2))
        ids = rng.integers(-1 if rng.random() < 0.2 else 0, S + (rng.random() < 0.2), size=n).tolist()
        if op == "reserve":
            lens = rng.integers(0, 16 * width + (3 if rng.random() < 0.2 else 1), size=n).tolist()
            plain.reserve(ids, lens)
            pool.reserve(ids, lens)
            set_lens(pool, plain, [int(rng.integers(0, 16 * len(t) + 1)) for t in plain.tables])
        elif op == "fork":
            src = rng.integers(0, S, size=n).tolist()
            plain.fork(src, ids)
            pool.fork(src, ids)
        elif op == "free":
            plain.free(ids)
            pool.free(ids)
        else:
            remap, live = plain.compact()
            assert pool.compact().tolist() == remap and pool.live.tolist() == [live]
        same(fb, pool, plain, f"step {step}: {op} {ids}")


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 48])
def test_fork_lengths(fb, length):
    """Whole pages are shared, a started page is the child's own; pages reserved ahead stay the parent's."""
    fb._lib.device_status(clear=True)
    pool, plain = make(length, Hkv=2)
    for p in (pool, plain):
        p.reserve([2], [80])
    set_lens(pool, plain, [0, 0, length, 0, 0, 0])
    for p in (pool, plain):
        p.fork([2, 2, 2], [0, 5, 3])
    same(fb, pool, plain)
    assert plain.ref[0] == (4 if length >= 16 else 1)


def test_many_blocks_and_streams(fb):
    """More pages and streams than the planning block has threads."""
    fb._lib.device_status(clear=True)
    S = 1500
    pool, plain = make(1, layers=1, blocks=5003, streams=S, max_blocks=4)
    rng = np.random.default_rng(2)
    order, lens = rng.permutation(S).tolist(), rng.integers(0, 65, size=S).tolist()
    for p in (pool, plain):
        p.reserve(order, lens)
    gone = rng.permutation(S)[:900].tolist()
    for p in (pool, plain):
        p.free(gone)
    same(fb, pool, plain, "freed")
    set_lens(pool, plain, [max(0, 16 * len(t) - 5) for t in plain.tables])
    alive = [s for s in range(S) if plain.tables[s]]
    src = rng.choice(alive, size=800).tolist()
    for p in (pool, plain):
        p.fork(src, gone[:800])
    same(fb, pool, plain, "forked")
    assert pool.compact().tolist() == plain.compact()[0]
    same(fb, pool, plain, "compacted")


def test_full_pool_refuses_whole_requests(fb):
    fb._lib.device_status(clear=True)
    pool, plain = make(3, blocks=5, streams=4, max_blocks=4)
    for p in (pool, plain):
        p.reserve([1, 0, 2, 3], [40, 33, 0, 16])
    same(fb, pool, plain, "3 pages of 5, then 3 refused, and what follows in order")
    with pytest.raises(fb._lib.FlintError, match="fewer pages were free"):
        pool.reserve([3], [64])
        fb._lib.check_device_status()
    set_lens(pool, plain, [0, 40, 0, 0])
    for p in (pool, plain):
        p.fork([1, 1, 1], [0, 2, 3])
    same(fb, pool, plain, "tails for two of three forks")


def test_compact_full_empty_and_ordered_pools(fb):
    fb._lib.device_status(clear=True)
    pool, plain = make(4, blocks=6, streams=3, max_blocks=4)
    for call in ((lambda p: p.compact()), (lambda p: p.reserve([0, 1], [64, 32])), (lambda p: p.compact()),
                 (lambda p: p.free([0])), (lambda p: p.compact()), (lambda p: p.free([1])), (lambda p: p.compact())):
        call(pool)
        call(plain)
        same(fb, pool, plain)
    assert pool.live.tolist() == [0]


def test_refusals(fb):
    from flint_b200 import kv_pages
    pool, _ = make(5)
    i = lambda *v, dt=torch.int32: torch.tensor(v, dtype=dt, device="cuda")
    with pytest.raises(fb._lib.FlintError):
        pool.free(i(1, dt=torch.int64))
    with pytest.raises(fb._lib.FlintError):
        pool.fork(i(1), i(2, 3))
    with pytest.raises(fb._lib.FlintError):
        pool.reserve(i(1, 2), i(16))
    with pytest.raises(fb._lib.FlintError):
        kv_pages.flint_kv_fork(pool.kv.float(), *pool.state, i(0), i(1))
    with pytest.raises(fb._lib.FlintError):
        kv_pages.flint_kv_fork(pool.kv[:, 1:], *pool.state, i(0), i(1))
    with pytest.raises(fb._lib.FlintError):
        kv_pages.flint_kv_compact(pool.kv, pool.ref, pool.block_tables, pool.num_pages, pool.remap[1:], pool.live)
    with pytest.raises(fb._lib.FlintError):
        kv_pages.flint_kv_free(pool.ref.cpu(), pool.block_tables, pool.seq_lens, pool.num_pages, i(0))
    with pytest.raises(ValueError):
        kv_pages.PagePool(pool.kv, 0, 4)
    pool.free([])
    pool.fork([], [])
    pool.reserve([], [])
