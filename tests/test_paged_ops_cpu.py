"""The prompt, shared-prefix and page operations without a GPU: what they refuse, their sizes, tracing, and their oracle."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import attention as oatt
from oracle import paged

D, PAGE = 128, 16


def test_cpu_tensors_are_refused(fb):
    from flint_b200 import kv_pages, prefill_attention, shared_prefix_attention
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt)
    i = lambda *s: z(*s, dt=torch.int32)
    kv = z(3, 2, PAGE, 2 * D)
    with pytest.raises(fb._lib.FlintError, match="CUDA"):
        prefill_attention.flint_prefill_attention(z(4, 8, D), kv, i(1, 3), i(2), i(1), None, None, 0.1, z(4, 8, D))
    with pytest.raises(fb._lib.FlintError, match="CUDA"):
        shared_prefix_attention.flint_shared_prefix_attention(z(2, 8, D), kv, i(2, 3), i(2), i(2), i(1), None, None, 0.1,
                                                              z(2, 8, D))
    with pytest.raises(fb._lib.FlintError, match="CUDA"):
        kv_pages.flint_kv_free(i(9), i(2, 3), i(2), i(2), i(1))
    with pytest.raises(fb._lib.FlintError, match="CUDA"):
        kv_pages.PagePool(z(1, 9, 2, PAGE, 2 * D), 2, 3)


def test_fake_tensors_reach_the_registered_ops(fb):
    """Under a dispatch mode the shims go through torch.ops, whose fake kernels run."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from flint_b200 import kv_pages, prefill_attention, shared_prefix_attention
    with FakeTensorMode():
        e = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="cuda")
        i = lambda *s: e(*s, dt=torch.int32)
        out = e(4, 8, D)
        assert prefill_attention.flint_prefill_attention(e(4, 8, D), e(3, 2, PAGE, 2 * D), i(1, 3), i(2), i(1), None, None,
                                                         0.1, out) is out
        assert shared_prefix_attention.flint_shared_prefix_attention(e(4, 8, D), e(3, 2, PAGE, 2 * D), i(4, 3), i(4), i(2),
                                                                     i(1), None, 7, 0.1, out) is out
        state = i(9), i(2, 3), i(2), i(2)
        kv = e(1, 9, 2, PAGE, 2 * D)
        kv_pages.flint_kv_reserve(*state, i(1), i(1))
        kv_pages.flint_kv_fork(kv, *state, i(1), i(1))
        kv_pages.flint_kv_free(*state, i(1))
        kv_pages.flint_kv_compact(kv, state[0], state[1], state[3], i(9), i(1))


P = ctypes.c_void_p(256)
PREFILL = dict(q=P, q_stride=4096, kv=P, blocks=8, Hkv=4, sb=16384, sh=4096, bt=P, bts=4, max_blocks=4, cu=P, lens=P,
               sinks=None, window=0, scale=0.1, batch=2, tokens=9, Hq=32, out=ctypes.c_void_p(512), out_stride=4096, ws=P, pdl=0, stream=None)
ARGUMENT, SHAPE, ALIGN = 6, 1, 2


@pytest.mark.parametrize("change,code", [
    (dict(q=None), ARGUMENT), (dict(kv=None), ARGUMENT), (dict(cu=None), ARGUMENT), (dict(lens=None), ARGUMENT),
    (dict(ws=None), ARGUMENT), (dict(window=-1), ARGUMENT), (dict(out=P, q=P), ARGUMENT), (dict(scale=0.0), ARGUMENT), (dict(scale=-0.1), ARGUMENT),
    (dict(scale=float("nan")), ARGUMENT), (dict(scale=float("inf")), ARGUMENT), (dict(batch=0), SHAPE),
    (dict(tokens=0), SHAPE), (dict(tokens=1 << 25), SHAPE), (dict(Hq=30), SHAPE), (dict(Hq=36), SHAPE), (dict(Hkv=0), SHAPE),
    (dict(blocks=0), SHAPE), (dict(max_blocks=0), SHAPE), (dict(max_blocks=1 << 26), SHAPE), (dict(q_stride=4088), SHAPE),
    (dict(out_stride=4088), SHAPE), (dict(sh=4088), SHAPE), (dict(q=ctypes.c_void_p(264)), ALIGN),
    (dict(out=ctypes.c_void_p(264)), ALIGN), (dict(kv=ctypes.c_void_p(264)), ALIGN), (dict(q_stride=4100), ALIGN),
    (dict(sb=16388), ALIGN)])
def test_prefill_arguments_are_checked_on_the_host(fb, change, code):
    assert fb._lib.lib().flint_prefill_attention(*{**PREFILL, **change}.values()) == code


def test_shared_prefix_groups_are_checked_on_the_host(fb):
    L = fb._lib.lib()
    args = [P, 4096, P, 8, 4, 16384, 4096, P, 4, 4, P, P, P, 1, None, 0, 0.1, 2, 32, ctypes.c_void_p(512), 4096, P, 0, None]
    for at, value, code in ((11, None, ARGUMENT), (12, None, ARGUMENT), (13, 0, SHAPE), (13, 3, SHAPE), (17, 0, SHAPE)):
        assert L.flint_shared_prefix_attention(*[value if i == at else v for i, v in enumerate(args)]) == code


def test_page_arguments_are_checked_on_the_host(fb):
    L = fb._lib.lib()
    pool = [P, 40, P, 6, 6]
    for n in (0, 4097):
        assert L.flint_kv_free(*pool, P, P, 5, P, n, P, 0, None) != 0
        assert L.flint_kv_reserve(*pool, P, 5, P, P, n, P, 0, None) != 0
        assert L.flint_kv_fork(P, 1, 4, 1 << 20, 16384, *pool, P, P, 5, P, P, n, P, 0, None) != 0
    assert L.flint_kv_free(P, 40, P, 5, 6, P, P, 5, P, 1, P, 0, None) == SHAPE              # rows overlap
    assert L.flint_kv_free(*pool, P, P, 5000, P, 1, P, 0, None) == SHAPE
    assert L.flint_kv_fork(P, 1, 4, 1 << 20, 16383, *pool, P, P, 5, P, P, 1, P, 0, None) == SHAPE
    assert L.flint_kv_fork(ctypes.c_void_p(264), 1, 4, 1 << 20, 16384, *pool, P, P, 5, P, P, 1, P, 0, None) == ALIGN
    assert L.flint_kv_compact(P, 1, 4, 1 << 20, 16388, *pool, P, 5, P, P, P, 0, None) == ALIGN
    assert L.flint_kv_compact(P, 1, 4, 1 << 20, 16384, *pool, P, 5, None, P, P, 0, None) == ARGUMENT


def test_workspace_sizes(fb):
    L = fb._lib.lib()
    a = L.flint_prefill_attention_workspace_bytes
    assert a(1, 1, 32, 4) == a(9, 100000, 32, 4) > 0 and a(0, 1, 32, 4) == -1
    b = L.flint_shared_prefix_attention_workspace_bytes
    assert b(8, 1, 32, 4) - a(1, 1, 32, 4) >= 2 * 8 * 32 * (128 + 2) * 4 and b(8, 0, 32, 4) == -1
    c = L.flint_kv_pages_workspace_bytes
    assert c(0) == -1 and c(1 << 20) >= 8 << 20
    assert L.flint_workspace_status_offset(16) == 0 and L.flint_workspace_status_offset(17) == 0


def test_status_names(fb):
    L = fb._lib
    assert L._status_kind("prefill_attention") == L._status_kind("shared_prefix_attention") == 16
    assert L._status_kind("kv_pages") == 17
    assert "fewer pages" in L.describe_status("kv_pages", 8) and "block table" in L.describe_status("prefill_attention", 4)


def test_oracle_agrees_with_the_decode_oracle(fb):
    """One query token per sequence: the decode attention's oracle, but for its rounding of the probabilities."""
    rng = np.random.default_rng(0)
    kv = rng.standard_normal((9, 2, PAGE, 2 * D)).astype(np.float32)
    bt, lens = np.array([[4, 1, 7], [0, 2, 5]]), [37, 20]
    q = rng.standard_normal((2, 6, D)).astype(np.float32)
    sinks = rng.standard_normal(6).astype(np.float32)
    for window in (0, 9):
        want = oatt.decode_attention(q, kv, bt, lens, sinks, window, D ** -0.5)
        got, spread = paged.prefill_attention(q, kv, bt, [1, 1], lens, sinks, window, D ** -0.5)
        assert (np.abs(got - want) <= 2.0 ** -8 * (np.abs(want) + spread)).all()


def test_plain_pool_keeps_its_counts():
    rng = np.random.default_rng(1)
    pool = paged.Pool(rng.standard_normal((1, 20, 1, PAGE, 256)).astype(np.float32), 4, 6)
    pool.reserve([0, 1], [40, 17])
    pool.lens = [40, 17, 0, 0]
    pool.fork([0, 0], [2, 3])
    assert pool.tables == [[0, 1, 2], [3, 4], [0, 1, 5], [0, 1, 6]] and pool.ref[:7] == [3, 3, 1, 1, 1, 1, 1]
    np.testing.assert_array_equal(pool.kv[:, 5], pool.kv[:, 2])
    pool.free([1, 0])
    remap, live = pool.compact()
    assert live == 4 and pool.tables == [[], [], [0, 1, 2], [0, 1, 3]] and remap[5] == 2 and remap[6] == 3 and pool.bad == 0
