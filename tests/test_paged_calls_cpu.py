"""How the prompt, shared-prefix and page calls reach the library, without a GPU."""
import inspect

import pytest
import torch


def test_direct_calls_count_versions_of_what_they_write(fb, monkeypatch):
    """The places of the written arguments are those of the registered ops' schemas, and each counts a version."""
    ops = fb.ops
    for name, (fn, written) in ops._DIRECT.items():
        schema = getattr(torch.ops.flint_b200, name).default._schema
        assert [i for i, a in enumerate(schema.arguments) if a.alias_info is not None and a.alias_info.is_write] == list(written)
        args, got = [torch.zeros(2) for _ in inspect.signature(fn).parameters], []
        monkeypatch.setitem(ops._DIRECT, name, (lambda *a: got.append(a), written))
        ops.run(name, *args)
        assert [t._version for t in args] == [int(i in written) for i in range(len(args))]
        assert len(got) == 1 and all(a is b for a, b in zip(got[0], args))


def test_subclasses_see_the_registered_op(fb):
    """A tensor subclass outside any mode is asked, as with every other op."""
    seen = []

    class Watching(torch.Tensor):
        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            seen.append(str(func))

    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    from flint_b200 import kv_pages
    kv_pages.flint_kv_free(i(9), i(2, 3).as_subclass(Watching), i(2), i(2), i(1))
    assert seen == ["flint_b200.kv_free"]
    with pytest.raises(fb._lib.FlintError, match="CUDA"):
        kv_pages.flint_kv_free(i(9), i(2, 3), i(2), torch.nn.Parameter(i(2), requires_grad=False), i(1))


def test_workspaces_are_sized_for_their_device(fb, monkeypatch):
    """A size found on one device is not another's, and a call for another device than the current one is refused: the
    launch takes the current device's number of blocks."""
    ops, current, sized = fb.ops, [0], []

    class Library:
        def flint_kv_pages_workspace_bytes(self, blocks):
            return blocks * (100 + current[0])

    monkeypatch.setattr(ops, "lib", Library)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(fb._lib, "workspace_and_stream", lambda dev, kind, n: sized.append((dev, kind, n)) or (1, 2))
    blocks = 7919
    for current[0] in (0, 1):
        assert ops._workspace("kv_free", current[0], "kv_pages", blocks) == (1, 2)
    assert sized == [(0, "kv_pages", 100 * blocks), (1, "kv_pages", 101 * blocks)]
    with pytest.raises(fb._lib.FlintError, match="cuda:0, but the current device is cuda:1"):
        ops._workspace("kv_free", 0, "kv_pages", blocks)
    ops._bytes_of.cache_clear()
