"""Calls of the key/value cache operators that their documentation allows or refuses, checked without a device: on which
stream memory is taken, which row tensors are accepted, how large a workspace is."""
import contextlib
import ctypes as C
import random

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


def _attention_args(**kw):
    a = dict(batch=2, rows=10, q_heads=8, kv_heads=2, head_dim=128, page_tokens=64, page_count=9, max_pages=4, max_query_length=7,
             max_sequence_length=200, softmax_scale=0.1, q_row_stride=1024, q_head_stride=128, output_row_stride=1024,
             output_head_stride=128, q=0x100000, output=0x200000, k_payload=0x3000, k_scales=0x4000, v_payload=0x5000, v_scales=0x6000,
             query_indptr=0x7000, sequence_lengths=0x8000, page_table=0x9000, workspace=0x300000, workspace_bytes=1 << 40)
    return abi.KvAttentionArgs(**{**a, **kw})


def test_attention_in_the_queries_own_buffer_and_outputs_without_a_stride_are_refused():
    lib = abi.load()
    can, launch = lib.ferrule_hip_kv_attention_can_implement, lib.ferrule_hip_kv_attention_launch
    assert can(C.byref(_attention_args())) == abi.SUCCESS
    one = dict(rows=1, batch=1, max_query_length=1, output_row_stride=0)
    assert can(C.byref(_attention_args(**one))) == abi.SUCCESS                       # nothing is a stride away
    assert can(C.byref(_attention_args(**one, q_heads=2, kv_heads=2, output_head_stride=64))) == abi.SUCCESS
    for bad in (dict(output=0x100000), dict(output=0x100000, flags=3, q_row_stride=2048), dict(output_row_stride=0),
                dict(output_head_stride=0), dict(one, output_head_stride=0)):
        assert can(C.byref(_attention_args(**bad))) == abi.INVALID_ARGUMENT, bad
        assert launch(C.byref(_attention_args(**bad))) == abi.INVALID_ARGUMENT, bad


def _bytes(shape, base, strides, size):
    """All bytes of a row tensor, those that stand twice twice."""
    rows, heads, d = shape
    return [base + size * (r * strides[0] + h * strides[1]) + i for r in range(rows) for h in range(heads) for i in range(d * size)]


def test_shared_bytes_of_row_tensors_are_found_exactly():
    rng = random.Random(3)
    answers, twice = [], []
    for _ in range(4000):
        shape = rng.randint(1, 4), rng.randint(1, 4), rng.choice((2, 4))
        pick = lambda: (rng.choice((0, 2, 3, 4, 5, 8, 12, 16, 24, 32)), rng.choice((0, 1, 2, 4, 6, 8, 16, 20)))  # noqa: E731
        first = 1000, pick(), rng.choice((2, 4))
        second = 1000 + rng.randint(-60, 160), pick(), rng.choice((2, 4))
        if rng.random() < 0.5:                                  # two views of one buffer have byte strides in common
            second = (second[0], first[1], first[2])
        a, b = _bytes(shape, *first), _bytes(shape, *second)
        answers.append(bool(set(a) & set(b)))
        assert P._kv_rows_meet(shape, *first, *second) == answers[-1], (shape, first, second)
        twice.append(len(set(a)) != len(a))
        assert P._kv_rows_repeat(shape, first[1]) == twice[-1], (shape, first)
    assert 400 < sum(answers) < 3600 and 400 < sum(twice) < 3600
