"""Refusals of the key/value cache entry points and of their Python handles, which touch no device, and the
test helpers' quantiser against the oracle's."""
import ctypes as C

import numpy as np
import pytest

from ferrule_amd import abi
from oracle import pyoracle as po
from tests import kv_helpers as K


def _cache_args(**kw):
    a = dict(batch=2, rows=10, kv_heads=2, head_dim=128, page_tokens=64, page_count=9, max_pages=4, max_query_length=7,
             value_type=abi.KV_BF16, key_row_stride=256, key_head_stride=128, value_row_stride=256, value_head_stride=128,
             keys=0x1000, values=0x2000, k_payload=0x3000, k_scales=0x4000, v_payload=0x5000, v_scales=0x6000,
             query_indptr=0x7000, sequence_lengths=0x8000, page_table=0x9000)
    a.update(kw)
    return abi.KvCacheArgs(**a)


def _attention_args(**kw):
    a = dict(batch=2, rows=10, q_heads=8, kv_heads=2, head_dim=128, page_tokens=64, page_count=9, max_pages=4,
             max_query_length=7, max_sequence_length=200, softmax_scale=0.1, q_row_stride=1024, q_head_stride=128,
             output_row_stride=1024, output_head_stride=128, q=0x1000, output=0x2000, k_payload=0x3000, k_scales=0x4000,
             v_payload=0x5000, v_scales=0x6000, query_indptr=0x7000, sequence_lengths=0x8000, page_table=0x9000,
             workspace=0x100000, workspace_bytes=1 << 40)
    a.update(kw)
    return abi.KvAttentionArgs(**a)


BAD_CACHE = [dict(kv_heads=0), dict(head_dim=0), dict(page_count=0), dict(max_pages=0), dict(max_query_length=0),
             dict(page_tokens=16), dict(page_tokens=48), dict(page_tokens=2048), dict(value_type=2), dict(reserved=1),
             dict(keys=0), dict(keys=0x1008), dict(values=0), dict(key_row_stride=260), dict(value_head_stride=4),
             dict(k_payload=0), dict(k_scales=0x4004), dict(v_payload=0x5008), dict(v_scales=0), dict(query_indptr=0),
             dict(sequence_lengths=0), dict(page_table=0), dict(page_table=0x9002), dict(error=0x9001),
             dict(rows=0x80000000), dict(page_count=0x80000000)]


@pytest.mark.parametrize("entry", ["append", "read"])
def test_cache_refusals(entry):
    lib = abi.load()
    can = getattr(lib, f"ferrule_hip_kv_cache_{entry}_can_implement")
    launch = getattr(lib, f"ferrule_hip_kv_cache_{entry}_launch")
    assert can(None) == abi.INVALID_ARGUMENT and launch(None) == abi.INVALID_ARGUMENT
    for d in abi.KV_HEAD_DIMS:
        assert can(C.byref(_cache_args(head_dim=d))) == abi.SUCCESS
    assert can(C.byref(_cache_args(value_type=abi.KV_F32, key_row_stride=260))) == abi.SUCCESS     # 16 bytes of f32
    for bad in BAD_CACHE:
        assert can(C.byref(_cache_args(**bad))) == abi.INVALID_ARGUMENT, bad
        assert launch(C.byref(_cache_args(**bad))) == abi.INVALID_ARGUMENT, bad
    for odd in (dict(head_dim=96), dict(batch=65536), dict(max_query_length=0x7fffffff, kv_heads=64)):
        assert can(C.byref(_cache_args(**odd))) == abi.UNSUPPORTED, odd
        assert launch(C.byref(_cache_args(**odd))) == abi.UNSUPPORTED, odd
    for nothing in (dict(rows=0), dict(batch=0)):
        assert can(C.byref(_cache_args(**nothing))) == abi.SUCCESS
        assert launch(C.byref(_cache_args(**nothing))) == abi.SUCCESS      # returns before any device call


BAD_ATTENTION = [dict(kv_heads=0), dict(q_heads=0), dict(q_heads=7), dict(head_dim=0), dict(page_count=0), dict(max_pages=0),
                 dict(max_query_length=0), dict(page_tokens=16), dict(page_tokens=96), dict(flags=4),
                 dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=float("nan")),
                 dict(softmax_scale=float("inf")), dict(window=0x80000000), dict(sinks=0x80000000), dict(q=0),
                 dict(q=0x1004), dict(output=0), dict(output_row_stride=1025), dict(q_head_stride=4), dict(k_payload=0x3001),
                 dict(k_scales=0), dict(v_payload=0), dict(v_scales=0x6008), dict(query_indptr=0), dict(sequence_lengths=0),
                 dict(page_table=0), dict(error=2), dict(rows=0x80000000)]


def test_attention_refusals():
    lib = abi.load()
    can, launch = lib.ferrule_hip_kv_attention_can_implement, lib.ferrule_hip_kv_attention_launch
    assert can(None) == abi.INVALID_ARGUMENT and launch(None) == abi.INVALID_ARGUMENT
    assert lib.ferrule_hip_kv_attention_workspace_size(None) == 0
    for d in abi.KV_HEAD_DIMS:
        assert can(C.byref(_attention_args(head_dim=d))) == abi.SUCCESS
    assert can(C.byref(_attention_args(flags=3, q_row_stride=1028))) == abi.SUCCESS
    for bad in BAD_ATTENTION:
        assert can(C.byref(_attention_args(**bad))) == abi.INVALID_ARGUMENT, bad
        assert launch(C.byref(_attention_args(**bad))) == abi.INVALID_ARGUMENT, bad
    for odd in (dict(head_dim=80), dict(batch=65536), dict(max_pages=0x7fffffff)):
        assert can(C.byref(_attention_args(**odd))) == abi.UNSUPPORTED, odd
        assert launch(C.byref(_attention_args(**odd))) == abi.UNSUPPORTED, odd
    for nothing in (dict(rows=0), dict(batch=0)):
        assert can(C.byref(_attention_args(**nothing))) == abi.SUCCESS
        assert launch(C.byref(_attention_args(**nothing))) == abi.SUCCESS


def test_attention_refuses_a_workspace_that_is_missing_short_or_unaligned():
    lib = abi.load()
    # one long sequence has to be split
    long = dict(batch=1, rows=1, max_query_length=1, max_pages=1024, page_count=1024, max_sequence_length=65536)
    args = _attention_args(**long, workspace=0, workspace_bytes=0)
    size = lib.ferrule_hip_kv_attention_workspace_size(C.byref(args))
    if size == 0:
        pytest.skip("no split at this size")
    can = lib.ferrule_hip_kv_attention_can_implement
    assert can(C.byref(args)) == abi.INVALID_ARGUMENT
    assert can(C.byref(_attention_args(**long, workspace=0x100000, workspace_bytes=size - 1))) == abi.INVALID_ARGUMENT
    assert can(C.byref(_attention_args(**long, workspace=0x100010, workspace_bytes=size))) == abi.INVALID_ARGUMENT
    assert can(C.byref(_attention_args(**long, workspace=0x100000, workspace_bytes=size))) == abi.SUCCESS


def test_cache_and_batch_handles_refuse_what_does_not_fit():
    import torch
    from ferrule_amd.provider import HipKvBatch, HipKvCache, kv_cache_shapes

    def arrays(p=3, t=64, h=2, d=128):
        return [torch.zeros(s, dtype=torch.uint8) for s in kv_cache_shapes(p, t, h, d)]

    HipKvCache(64, 2, 128, *arrays())
    for args in ((48, 2, 128), (16, 2, 128), (64, 0, 128), (64, 2, 96), (64, 3, 128), (128, 2, 128)):
        with pytest.raises(ValueError):
            HipKvCache(*args, *arrays())
    wrong = arrays()
    wrong[1] = wrong[1].to(torch.int8)
    with pytest.raises(ValueError):
        HipKvCache(64, 2, 128, *wrong)
    wrong = arrays()
    wrong[2] = wrong[2][:2]
    with pytest.raises(ValueError):
        HipKvCache(64, 2, 128, *wrong)
    with pytest.raises(ValueError):
        HipKvCache(64, 2, 128, *arrays(p=0))

    def i32(*shape):
        return torch.zeros(shape, dtype=torch.int32)

    HipKvBatch(i32(3), i32(2), i32(2, 4), 5)
    for ptr, lengths, table in ((i32(2), i32(2), i32(2, 4)), (i32(3), i32(2), i32(3, 4)), (i32(3), i32(2, 1), i32(2, 4)),
                                (i32(3).long(), i32(2), i32(2, 4)), (i32(3), i32(2), i32(4, 2).T)):
        with pytest.raises(ValueError):
            HipKvBatch(ptr, lengths, table, 5)
    with pytest.raises(ValueError):
        HipKvBatch(i32(3), i32(2), i32(2, 4), -1)
    with pytest.raises(ValueError):
        HipKvBatch(i32(3), i32(2), i32(2, 4), 5, max_query_length=0)


def test_the_helpers_quantiser_is_the_oracles_on_bf16_values():
    rng = np.random.default_rng(5)
    x = K.bf16(rng.standard_normal((64, 128)) * np.exp(rng.uniform(-60, 60, (64, 1))))
    x[3] = 0
    x[4, :32] = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6] * 4) * np.array([1, -1] * 16)
    code, scale = K.quantise(x)
    packed, scales = po.pack_fp4_act(x.ravel(), 128)
    assert (np.asarray(scales).reshape(scale.shape) == scale).all()
    packed = np.asarray(packed).reshape(64, 64)
    assert (packed == (code[:, 0::2] | code[:, 1::2] << 4)).all()


def test_grids_that_a_launch_cannot_count_are_refused_and_the_largest_that_it_can_are_not():
    lib = abi.load()
    can = lib.ferrule_hip_kv_cache_append_can_implement
    # 2^24 - 1 tiles of 32 rows: the first row is the last one of its tile, then full tiles
    most = 1 + (0xffffff - 1) * 32
    assert can(C.byref(_cache_args(rows=most, max_query_length=most, kv_heads=1))) == abi.SUCCESS
    assert can(C.byref(_cache_args(rows=most, max_query_length=most + 1, kv_heads=1))) == abi.UNSUPPORTED
    assert can(C.byref(_cache_args(kv_heads=0x1000000))) == abi.UNSUPPORTED
    can = lib.ferrule_hip_kv_attention_can_implement
    # a prompt of 131072 tokens with 64 heads: 2^23 rows and heads
    long = dict(rows=131072, max_query_length=131072, q_heads=64, kv_heads=8)
    assert can(C.byref(_attention_args(**long))) == abi.SUCCESS
    assert can(C.byref(_attention_args(**dict(long, rows=0x400000, max_query_length=0x400000)))) == abi.UNSUPPORTED
    # one row with as many heads as the cache: a workgroup for each
    assert can(C.byref(_attention_args(rows=1, max_query_length=1, q_heads=0x800000, kv_heads=0x800000))) == abi.UNSUPPORTED
    assert can(C.byref(_attention_args(softmax_scale=2.0 ** 127))) == abi.SUCCESS
    assert can(C.byref(_attention_args(softmax_scale=2.5e38))) == abi.INVALID_ARGUMENT


def test_batches_beyond_31_bits_are_refused():
    import torch
    from ferrule_amd.provider import HipKvBatch
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    HipKvBatch(i32(2), i32(1), i32(1, 4), 0x7fffffff, 0x7fffffff, 0x7fffffff)
    for more in ((2 ** 31, 1, 1), (1, 2 ** 32 + 1, 1), (1, 1, 2 ** 32)):
        with pytest.raises(ValueError):
            HipKvBatch(i32(2), i32(1), i32(1, 4), *more)


def test_the_workspace_of_a_prompt_beside_a_long_decode_row_stays_small():
    lib = abi.load()
    size = lambda **kw: lib.ferrule_hip_kv_attention_workspace_size(C.byref(_attention_args(**kw)))  # noqa: E731
    mixed = dict(batch=2, rows=8193, q_heads=64, kv_heads=8, max_query_length=8192, max_pages=1024, page_count=2048,
                 max_sequence_length=65536)
    # parts of a decode launch hold four rows a sequence, at most 1024 of 16 packed rows in two tiles
    assert 0 < size(**mixed) <= 2 * 1024 * 16 * (128 + 2) * 4 + 512 * 256 * (128 + 2) * 4
    for d in abi.KV_HEAD_DIMS:
        for rows, batch, longest in ((1, 1, 65536), (64, 64, 8192), (600, 3, 60000), (8192, 4, 8192), (4000, 200, 30000)):
            got = size(batch=batch, rows=rows, q_heads=64, kv_heads=8, head_dim=d, max_query_length=max(1, rows // 2), max_pages=1024,
                       page_count=2048, max_sequence_length=longest)
            assert got <= 600 << 20, (d, rows, batch, longest, got)
