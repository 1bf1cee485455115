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
