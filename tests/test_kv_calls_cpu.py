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


class _Stream:
    """torch's current stream, which keeps what it waited for."""

    def __init__(self, waited):
        self.waited = waited

    def wait_stream(self, other):
        self.waited.append(other)


def test_a_new_cache_is_filled_on_the_contexts_stream_and_torchs_waits_for_it(monkeypatch):
    """Whoever writes to it next finds it filled: the context's operators, and torch on its current stream."""
    ctx, taken = _host_context(monkeypatch, "side")
    waited = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: _Stream(waited))
    cache = ctx.kv_cache(3, 64, 2, 128)
    assert waited == ["side"]
    del waited[:]
    ctx._stream = own = torch.cuda.current_stream()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *_: own)
    ctx.kv_cache(3, 64, 2, 128)
    assert waited == [] and taken[4:] == [own] * 4
    del taken[4:]
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


def _cache_args(**kw):
    a = dict(batch=2, rows=10, kv_heads=2, head_dim=128, page_tokens=64, page_count=9, max_pages=4, max_query_length=7,
             value_type=abi.KV_BF16, key_row_stride=256, key_head_stride=128, value_row_stride=256, value_head_stride=128,
             keys=0x100000, values=0x200000, k_payload=0x3000, k_scales=0x4000, v_payload=0x5000, v_scales=0x6000,
             query_indptr=0x7000, sequence_lengths=0x8000, page_table=0x9000)
    return abi.KvCacheArgs(**{**a, **kw})


def test_row_tensors_that_read_and_attention_may_write_are_told_from_those_that_they_may_not(monkeypatch):
    """The Python entries' answers, before any call into the library, are those of the bytes."""
    ctx, _ = _host_context(monkeypatch, None)
    monkeypatch.setattr(ctx, "_check_kv", lambda *_: -1, raising=False)
    cache = P.HipKvCache(64, 2, 64, *(torch.empty(s, dtype=torch.uint8) for s in P.kv_cache_shapes(3, 64, 2, 64)))
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    memory = torch.zeros(1 << 14, dtype=torch.uint8)
    launched = []
    monkeypatch.setattr(ctx, "_kv_launch", lambda *_: launched.append(True), raising=False)
    rng, answers = random.Random(5), []
    for _ in range(1500):
        n, attention = rng.randint(1, 4), rng.random() < 0.5
        batch = P.HipKvBatch(i32(2), i32(1), i32(1, 3), n)
        heads = rng.choice((2, 4)) if attention else 2
        types = [rng.choice((torch.bfloat16, torch.float32))] * 2
        if attention and rng.random() < 0.3:
            types[1] = rng.choice((torch.bfloat16, torch.float32))
        tensors, places, strides = [], [], None
        for t in types:
            size = 2 if t is torch.bfloat16 else 4
            if strides is None or rng.random() < 0.4:
                strides = rng.choice((64 * heads, 64 * heads, 128 * heads, 64, 0)), rng.choice((64, 64, 128, 64 * n, 0))
            base = 16 * rng.randint(0, 160)
            tensors.append(torch.as_strided(memory.view(t), (n, heads, 64), (*strides, 1), base // size))
            places.append(_bytes((n, heads, 64), base, strides, size))
        bad = bool(set(places[0]) & set(places[1])) or any(len(set(p)) < len(p) for p in (places[1:] if attention else places))
        answers.append(bad)
        del launched[:]
        with (pytest.raises(ValueError) if bad else contextlib.nullcontext()):
            if attention:
                ctx.kv_cache_attention_into(cache, batch, *tensors, 0.1, workspace=memory)
            else:
                ctx.kv_cache_read_into(cache, batch, *tensors)
        assert bool(launched) != bad, (places, types)
    assert 300 < sum(answers) < 1400


def test_read_refuses_one_place_for_keys_and_values_and_append_does_not():
    lib = abi.load()
    can, launch = lib.ferrule_hip_kv_cache_read_can_implement, lib.ferrule_hip_kv_cache_read_launch
    append = lib.ferrule_hip_kv_cache_append_can_implement
    assert can(C.byref(_cache_args())) == abi.SUCCESS
    one = dict(rows=1, batch=1, max_query_length=1, key_row_stride=0, value_row_stride=0)
    assert can(C.byref(_cache_args(**one))) == abi.SUCCESS
    assert can(C.byref(_cache_args(**one, kv_heads=1, key_head_stride=0, value_head_stride=0))) == abi.SUCCESS
    for bad in (dict(values=0x100000), dict(key_row_stride=0), dict(value_row_stride=0), dict(key_head_stride=0), dict(value_head_stride=0)):
        assert can(C.byref(_cache_args(**bad))) == abi.INVALID_ARGUMENT, bad
        assert launch(C.byref(_cache_args(**bad))) == abi.INVALID_ARGUMENT, bad
        assert append(C.byref(_cache_args(**bad))) == abi.SUCCESS, bad               # what is only read may stand twice


@pytest.mark.parametrize("d", abi.KV_HEAD_DIMS)
def test_rows_behind_the_last_sequence_take_no_workspace(d):
    """A row tensor may be longer than what its sequences can have; also by so much that bytes would not count in 64 bits."""
    lib = abi.load()
    size = lambda **kw: lib.ferrule_hip_kv_attention_workspace_size(C.byref(_attention_args(head_dim=d, **kw)))  # noqa: E731
    for q_heads, batch, most, length in ((64, 1, 1, 65536), (8, 3, 2, 30000), (64, 2, 100, 9000), (2048, 1, 1, 1 << 24)):
        shape = dict(q_heads=q_heads, batch=batch, max_query_length=most, max_pages=1 << 19, max_sequence_length=length)
        least = size(rows=batch * most, **shape)
        assert least > 0
        for rows in (batch * most + 1, 100000, 0x7fffffff):
            assert size(rows=rows, **shape) <= least, (rows, shape)
            # and the launch is content with that much
            args = _attention_args(head_dim=d, rows=rows, workspace_bytes=least, **shape)
            assert lib.ferrule_hip_kv_attention_can_implement(C.byref(args)) == abi.SUCCESS


def _smaller(rng, most):
    """A block with no larger a bound than `most`."""
    log = lambda n: min(n, max(1, round(n ** rng.random())))  # noqa: E731
    pick = lambda n: rng.choice((n, log(n), rng.randint(1, n)))  # noqa: E731
    return dict(batch=pick(most["batch"]), rows=pick(most["rows"]), max_query_length=pick(most["max_query_length"]),
                max_sequence_length=pick(most["max_sequence_length"]))


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("d", abi.KV_HEAD_DIMS)
def test_a_workspace_sized_by_the_largest_bounds_holds_every_smaller_block(d, seed):
    lib = abi.load()
    can, sizes = lib.ferrule_hip_kv_attention_can_implement, lib.ferrule_hip_kv_attention_workspace_size
    rng = random.Random(1000 * d + seed)
    split = 0
    for _ in range(60):
        group, kv_heads = rng.choice((1, 2, 3, 4, 5, 8, 16, 24, 40, 64, 100, 128)), rng.choice((1, 2, 3, 4, 6, 8, 16))
        window, sinks = rng.choice(((0, 0), (0, 0), (rng.randint(1, 9000), rng.choice((0, 4, 40)))))
        fixed = dict(q_heads=group * kv_heads, kv_heads=kv_heads, head_dim=d, max_pages=2048)
        most = dict(batch=rng.choice((1, 2, 5, 17, 64, 100, 300)), rows=rng.choice((1, 3, 64, 100, 700, 2048, 8193)),
                    max_query_length=rng.choice((1, 2, 5, 33, 64, 300, 2048, 8192)), max_sequence_length=rng.choice((1, 600, 4000, 8192, 60000, 131072)))
        size = sizes(C.byref(_attention_args(**fixed, **most, window=window, sinks=sinks)))
        for _ in range(60):
            small = _smaller(rng, most)
            less = sizes(C.byref(_attention_args(**fixed, **small, window=window, sinks=sinks)))
            assert less <= size, (fixed, most, small, window, sinks)
            # sized without a window it holds for every window
            narrow = (window, sinks) if window else rng.choice(((0, 0), (rng.randint(1, 9000), rng.choice((0, 4, 40)))))
            block = dict(fixed, **small, window=narrow[0], sinks=narrow[1], workspace=0x300000 if size else 0)
            assert can(C.byref(_attention_args(**block, workspace_bytes=size))) == abi.SUCCESS, (block, most, size)
            split += can(C.byref(_attention_args(**block, workspace_bytes=0))) != abi.SUCCESS
    assert split > 300                                          # of the smaller blocks need some


def test_the_workspace_of_the_largest_bounds_is_not_much_larger_than_what_a_block_needs():
    lib = abi.load()
    size = lambda **kw: lib.ferrule_hip_kv_attention_workspace_size(C.byref(_attention_args(max_pages=2048, **kw)))  # noqa: E731
    decode = dict(rows=1, max_query_length=1, q_heads=64, kv_heads=8, max_sequence_length=8192)
    # 1024 parts of eight heads, and one more for each row
    for batch in (32, 64, 100, 1024):
        assert 0 < size(**dict(decode, batch=batch, rows=batch)) <= 2 * 1024 * 8 * (128 + 2) * 4
    assert size(**dict(decode, batch=1, max_sequence_length=200)) == 0       # one part
    prompt = dict(batch=1, rows=8192, max_query_length=8192, q_heads=32, kv_heads=8, max_sequence_length=8192)
    assert 0 < size(**prompt) <= 2 * 256 * 256 * (128 + 2) * 4


def test_a_stride_that_nothing_takes_may_be_any():
    """One row, or one head: every row that there is stands on 16 bytes."""
    lib = abi.load()
    row = dict(batch=1, rows=1, max_query_length=1)
    can = lib.ferrule_hip_kv_cache_append_can_implement
    assert can(C.byref(_cache_args(**row, key_row_stride=577, value_row_stride=3))) == abi.SUCCESS
    assert can(C.byref(_cache_args(kv_heads=1, key_head_stride=577, value_head_stride=1))) == abi.SUCCESS
    for bad in (dict(row, key_head_stride=577), dict(row, kv_heads=1, keys=0x100008), dict(kv_heads=1, value_row_stride=577)):
        assert can(C.byref(_cache_args(**bad))) == abi.INVALID_ARGUMENT, bad
    can = lib.ferrule_hip_kv_attention_can_implement
    assert can(C.byref(_attention_args(**row, q_row_stride=577, output_row_stride=1))) == abi.SUCCESS
    assert can(C.byref(_attention_args(q_heads=1, kv_heads=1, q_head_stride=577, output_head_stride=1))) == abi.SUCCESS
    for bad in (dict(row, q_head_stride=577), dict(row, output_head_stride=129), dict(q_heads=1, kv_heads=1, output_row_stride=577)):
        assert can(C.byref(_attention_args(**bad))) == abi.INVALID_ARGUMENT, bad
