"""Calls of the key/value cache operators that their documentation allows or refuses, checked without a device: on which
stream memory is taken, which row tensors are accepted, how large a workspace is."""
import contextlib

import pytest

torch = pytest.importorskip("torch")

from ferrule_amd import abi
from ferrule_amd import provider as P


def _host_context(monkeypatch, own_stream):
    """A context over host tensors whose stream is the text `own_stream`, and a list that takes the stream that was
    current at each allocation."""
    ctx = object.__new__(P.HipArtifactOperatorContext)
    ctx.lib, ctx.device, ctx._stream, ctx.kernel_launches = abi.load(), torch.device("cpu"), own_stream, 0
    current, taken = ["torch's own"], []

    @contextlib.contextmanager
    def stream(s):
        current.append(s)
        try:
            yield
        finally:
            current.pop()

    monkeypatch.setattr(torch.cuda, "stream", stream)
    for name in ("zeros", "empty"):
        plain = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, plain=plain, **kw: taken.append(current[-1]) or plain(*a, **kw))
    return ctx, taken


def test_a_new_cache_is_filled_on_the_contexts_stream(monkeypatch):
    ctx, taken = _host_context(monkeypatch, "side")
    cache = ctx.kv_cache(3, 64, 2, 128)
    assert taken == ["side"] * 4
    assert all(not t.any() for t in (cache.k_payload, cache.k_scales, cache.v_payload, cache.v_scales))


@pytest.mark.parametrize("length", [0, 5000])
def test_the_workspace_of_a_side_context_belongs_to_its_stream(monkeypatch, length):
    """Also where it is empty: the allocator hands a block out again in the order of the stream that it was taken on."""
    ctx, taken = _host_context(monkeypatch, "side")
    monkeypatch.setattr(ctx, "_check_kv", lambda *_: 0, raising=False)
    cache = P.HipKvCache(64, 8, 128, *(torch.empty(s, dtype=torch.uint8) for s in P.kv_cache_shapes(90, 64, 8, 128)))
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    batch = P.HipKvBatch(i32(2), i32(1), i32(1, 90), 1, 1, length)
    del taken[:]
    workspace = ctx.kv_cache_attention_workspace(cache, batch, 64)
    assert taken == ["side"] and (workspace.numel() > 0) == (length > 0)
