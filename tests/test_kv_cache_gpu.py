"""The MXFP4 key/value cache on the GPU: append and read against numpy byte for byte, attention against
float64 within a bound derived from its arithmetic (tests/kv_helpers.py), and the three of them in a layer."""
import numpy as np
import pytest

from oracle import parity as P
from oracle import pyoracle as po
from tests import kv_helpers as K

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    from ferrule_amd.provider import HipArtifactOperatorContext
    return HipArtifactOperatorContext(0)


def _rows_to_device(x, dtype, pad=0):
    """[rows, heads, d] with `pad` values behind every head's row and one spare row stride."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dtype).cuda()
    if not pad:
        return t
    wide = torch.full((t.shape[0], t.shape[1] + 1, t.shape[2] + pad), float("nan"), dtype=dtype, device="cuda")
    view = wide[:, :t.shape[1], :t.shape[2]]
    view.copy_(t)
    return view


def _f32(x):
    with np.errstate(over="ignore"):        # 6 * 2^126 and more is an infinity in f32
        return x.astype(np.float32)


def _flag():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _same_bytes(cache, host):
    for i, (t, a) in enumerate(zip((cache.k_payload, cache.k_scales, cache.v_payload, cache.v_scales), host.arrays)):
        got = t.cpu().numpy().ravel()
        assert (got == a).all(), f"array {i}: {int((got != a).sum())} bytes differ, first at {int(np.argmax(got != a))}"


APPENDS = [  # new rows, lengths, page tokens, heads, head size
    ([1], [1], 32, 1, 64), ([1, 1, 1], [33, 64, 7], 32, 2, 128), ([5, 0, 8, 17], [5, 40, 64, 100], 64, 3, 128),
    ([7, 9], [900, 12], 128, 1, 512), ([40, 3], [40, 259], 32, 2, 256), ([130], [333], 1024, 2, 64),
    ([31, 33, 32], [95, 33, 64], 32, 8, 128),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("new,lengths,page,heads,d", APPENDS)
def test_append_writes_the_rows_bytes_and_no_others(ctx, new, lengths, page, heads, d, dtype):
    rng = np.random.default_rng(sum(new) + d)
    batch = K.HostBatch(rng, new, lengths, page)
    k, v = (rng.standard_normal((batch.total, heads, d)).astype(np.float32) * np.exp(rng.uniform(-3, 3, (1, heads, d)))
            for _ in range(2))
    if dtype == "bf16":
        k, v = K.bf16(k), K.bf16(v)
    host = K.HostCache(batch.pages, page, heads, d, fill=0xA5)
    cache = host.device()
    tdtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    flag = _flag()
    ctx.kv_cache_append(cache, batch.device(), _rows_to_device(k, tdtype, 16), _rows_to_device(v, tdtype), flag)
    for b in range(len(new)):
        for i, p in enumerate(batch.positions(b)):
            page_id, t = batch.place(b, p)
            for h in range(heads):
                for which, x in enumerate((k, v)):
                    host.put(page_id, h, t, which, *K.quantise(x[batch.indptr[b] + i, h]))
    _same_bytes(cache, host)
    assert flag.item() == 0


def test_append_edge_values(ctx):
    """Ties, the smallest and largest magnitudes, zeros of both signs, and blocks with an infinity or a NaN."""
    d, heads = 128, 2
    rng = np.random.default_rng(1)
    x = rng.standard_normal((16, heads, d)).astype(np.float32)
    x[0] = 0.0
    x[1] = -0.0
    x[2, 0] = np.tile(np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6], np.float32), 16) * np.tile([1, -1], 64)
    x[2, 1] = np.nextafter(x[2, 0], np.float32(np.inf))
    x[3] *= np.float32(1e-38)
    x[4] *= np.float32(1e-43)                       # subnormal
    x[5, :, 7] = 3.4028234e38
    x[6, :, 40] = np.inf
    x[7, :, 70] = np.nan
    x[8, :, 100] = -np.inf
    for n in range(32):                             # the scale's step: amax 6 * 2^n and the neighbours
        x[9, 0, n] = 0.1
    x[9, 0, 0], x[9, 0, 32], x[9, 0, 64], x[9, 0, 96] = 6.0, np.nextafter(np.float32(6), np.float32(7)), 1.5 * 2.0 ** -20, \
        np.nextafter(np.float32(1.5 * 2.0 ** -20), np.float32(1))
    batch = K.HostBatch(rng, [16], [19], 32)
    host = K.HostCache(batch.pages, 32, heads, d)
    cache = host.device()
    xd = torch.from_numpy(x).cuda()
    ctx.kv_cache_append(cache, batch.device(), xd, xd)
    for i, p in enumerate(batch.positions(0)):
        for h in range(heads):
            for which in (0, 1):
                host.put(*_place(batch, 0, p, h), which, *K.quantise(x[i, h]))
    _same_bytes(cache, host)
    # and what comes back: finite blocks at most half a level's step off, NaN where the block held one
    kd, vd = torch.empty_like(xd), torch.empty_like(xd)
    ctx.kv_cache_read_into(cache, batch.device(), kd, vd)
    want = np.stack([[K.dequantise(*K.quantise(x[i, h])) for h in range(heads)] for i in range(16)])
    assert np.array_equal(kd.cpu().numpy(), _f32(want), equal_nan=True)
    assert np.array_equal(vd.cpu().numpy(), _f32(want), equal_nan=True)
    assert np.isnan(want[6, :, 32:64]).all() and np.isnan(want[7, :, 64:96]).all() and np.isfinite(want[6, :, :32]).all()


def _place(batch, b, p, h):
    page, t = batch.place(b, p)
    return page, h, t


def test_append_equals_the_activation_packer_on_bf16_rows(ctx):
    rng = np.random.default_rng(2)
    x = torch.from_numpy(K.bf16(rng.standard_normal((24, 128)))).cuda()
    packed, scales = ctx.pack_fp4_rows_from_f32(x)
    batch = K.HostBatch(rng, [24], [24], 32)
    cache = ctx.kv_cache(batch.pages, 32, 1, 128)
    ctx.kv_cache_append(cache, batch.device(), x.view(24, 1, 128), x.view(24, 1, 128))
    page = batch.table[0, 0]
    assert torch.equal(cache.k_payload[page, 0, 0, 0, :24], packed)
    assert torch.equal(cache.k_scales[page, 0, 0, :, :24].T, scales)
    assert torch.equal(cache.v_payload[page, 0].transpose(1, 2).reshape(32, 64)[:24], packed)
    assert torch.equal(cache.v_scales[page, 0].transpose(1, 2).reshape(32, 4)[:24], scales)


def test_rows_without_a_place_are_dropped_read_as_zeros_and_reported(ctx):
    rng = np.random.default_rng(3)
    # sequence 0: a page number out of range and one that is negative; 1: more rows than tokens; 2: beyond the table
    batch = K.HostBatch(rng, [70, 5, 4, 2], [96, 3, 64, 32], 32, extra_columns=0)
    batch.table[0, 1], batch.table[0, 2] = batch.pages, -7
    batch.lengths[2] = 97                                       # the table holds 96: one row falls outside
    host = K.HostCache(batch.pages, 32, 2, 64, fill=0x5A)
    x = rng.standard_normal((batch.total + 3, 2, 64)).astype(np.float32)
    flag = _flag()
    batch.table[2, 2] = batch.table[2, 1]                       # row positions 93..95 have a page
    cache = host.device()
    dev = batch.device(rows=batch.total + 3)
    xd = torch.from_numpy(x).cuda()
    ctx.kv_cache_append(cache, dev, xd, xd, flag)
    want = np.zeros_like(x)
    for b in range(4):
        for i, p in enumerate(batch.positions(b)):
            place = batch.place(b, p)
            if place is not None:
                r = batch.indptr[b] + i
                for h in range(2):
                    for which in (0, 1):
                        host.put(place[0], h, place[1], which, *K.quantise(x[r, h]))
                    want[r, h] = K.dequantise(*K.quantise(x[r, h]))
    _same_bytes(cache, host)
    assert flag.item() == 1
    kd, vd = torch.full_like(xd, 7.0), torch.full_like(xd, 7.0)
    want[batch.total:] = 7.0                                    # rows behind the last sequence stay as they were
    flag.zero_()
    ctx.kv_cache_read_into(cache, dev, kd, vd, flag)
    assert np.array_equal(kd.cpu().numpy(), want) and np.array_equal(vd.cpu().numpy(), want)
    assert flag.item() == 1


def test_bad_indices_and_lengths_stay_inside_the_tensors(ctx):
    """Row indices beyond the tensors or out of order, negative and huge lengths: reported, nothing outside touched."""
    from ferrule_amd.provider import HipKvBatch
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    host = K.HostCache(4, 32, 1, 64).random(np.random.default_rng(4))
    for indptr, lengths in (((0, 5, 90), (5, 85)), ((0, -3, 4), (7, 9)), ((6, 2, 4), (5, 5)), ((0, 2, 4), (-1, 2 ** 31 - 1)),
                            ((0, 8, 8), (8, 0))):
        cache = host.device()
        batch = HipKvBatch(i32(*indptr), i32(*lengths), torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2), 8,
                           max_query_length=4)
        guard = torch.full((10, 1, 64), 3.0, device="cuda")
        rows = guard[1:9]
        flag = _flag()
        ctx.kv_cache_read_into(cache, batch, rows, rows.clone(), flag)
        q, out = torch.ones_like(rows), rows
        ctx.kv_cache_attention_into(cache, batch, q, out, 0.1, error=flag)
        ctx.kv_cache_append(cache, batch, q, q, flag)
        torch.cuda.synchronize()
        assert (guard[0] == 3).all() and (guard[9] == 3).all() and flag.item() == 1, (indptr, lengths)


@pytest.mark.parametrize("d,page", [(64, 32), (128, 64), (256, 256), (512, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_read_is_exact_for_every_nibble_and_ordinary_scale(ctx, d, page, dtype):
    rng = np.random.default_rng(d)
    batch = K.HostBatch(rng, [20, 65, 1], [20, 77, 300], page)
    host = K.HostCache(batch.pages, page, 2, d).random(rng, 1, 255)
    host.arrays[1][rng.integers(0, host.arrays[1].size, 50)] = 255
    host.arrays[3][rng.integers(0, host.arrays[3].size, 50)] = 255
    tdtype = torch.bfloat16 if dtype == "bf16" else torch.float32
    k = torch.empty((batch.total, 3, d + 8), dtype=tdtype, device="cuda")[:, :2, :d]
    v = torch.empty((batch.total, 2, d), dtype=tdtype, device="cuda")
    ctx.kv_cache_read_into(host.device(), batch.device(), k, v)
    for b in range(3):
        for i, p in enumerate(batch.positions(b)):
            for h in range(2):
                place = _place(batch, b, p, h)
                for which, t in enumerate((k, v)):
                    got = t[batch.indptr[b] + i, h].float().cpu().numpy()
                    assert np.array_equal(got, _f32(host.value(*place, which)), equal_nan=True)


# -- attention ---------------------------------------------------------------------------------
def _attend(ctx, host, batch, q, scale, window=0, sinks=0, out_dtype=torch.bfloat16, q_dtype=torch.bfloat16, pad=0, **kw):
    qd = _rows_to_device(q, q_dtype, pad)
    out = _rows_to_device(np.full(q.shape, 9.0), out_dtype, pad)
    ctx.kv_cache_attention_into(host.device(), batch.device(**kw), qd, out, scale, window=window, sinks=sinks)
    return out.float().cpu().numpy()


def _case(rng, new, lengths, page, heads, group, d, lo=124, hi=128):
    batch = K.HostBatch(rng, new, lengths, page)
    host = K.HostCache(batch.pages, page, heads, d).random(rng, lo, hi)
    q = K.bf16(rng.standard_normal((batch.total, heads * group, d)))
    return batch, host, q


SHAPES = [  # new rows, lengths, page, kv heads, group, head size
    ([1], [1], 32, 1, 1, 64), ([1], [2], 64, 2, 1, 128), ([1, 1, 1], [31, 32, 33], 32, 1, 4, 128),
    ([1], [700], 64, 2, 8, 128), ([1, 1], [257, 1025], 256, 1, 5, 64), ([1, 2], [300, 90], 32, 1, 16, 256),
    ([1, 1], [513, 64], 64, 1, 40, 512), ([3, 5, 1], [3, 130, 77], 64, 2, 6, 128), ([17], [17], 32, 1, 3, 64),
    ([70, 33], [70, 200], 64, 2, 2, 128), ([150], [170], 128, 1, 2, 256), ([40], [50], 32, 1, 2, 512),
    ([0, 1, 0, 2], [5, 40, 0, 70], 32, 2, 2, 64), ([130], [1000], 32, 1, 1, 64),
]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 4), (100, 0), (33, 40)])
@pytest.mark.parametrize("new,lengths,page,heads,group,d", SHAPES)
def test_attention_equals_float64(ctx, new, lengths, page, heads, group, d, window, sinks):
    rng = np.random.default_rng(d + sum(lengths))
    batch, host, q = _case(rng, new, lengths, page, heads, group, d)
    scale = float(d) ** -0.5
    want, bound = K.attention_reference(host, batch, q, scale, window, sinks)
    K.check_attention(_attend(ctx, host, batch, q, scale, window, sinks), want, bound)


@pytest.mark.parametrize("q_dtype,out_dtype", [("f32", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("new,lengths,d", [([1, 1], [90, 400], 128), ([40, 3], [60, 33], 64), ([2, 20], [70, 100], 512)])
def test_attention_types_and_strides(ctx, new, lengths, d, q_dtype, out_dtype):
    """f32 queries enter rounded to BF16, f32 outputs are not rounded; rows and heads of both are strided."""
    rng = np.random.default_rng(7)
    batch, host, _ = _case(rng, new, lengths, 32, 2, 3, d)
    q = rng.standard_normal((batch.total, 6, d)).astype(np.float32)
    t = dict(bf16=torch.bfloat16, f32=torch.float32)
    if q_dtype == "bf16":
        q = K.bf16(q)
    want, bound = K.attention_reference(host, batch, K.bf16(q), 0.11, 50, 3, f32_output=out_dtype == "f32")
    got = _attend(ctx, host, batch, q, 0.11, 50, 3, t[out_dtype], t[q_dtype], pad=8)
    K.check_attention(got, want, bound)


@pytest.mark.parametrize("new,lengths", [([1], [300]), ([50], [300]), ([1, 1, 1, 1], [40, 3000, 1, 500])])
def test_attention_of_one_dominant_score_and_of_equal_scores(ctx, new, lengths):
    """A key that takes all the weight, at the first, a middle and the last position; and keys that are all alike."""
    rng = np.random.default_rng(11)
    batch, host, q = _case(rng, new, lengths, 64, 1, 2, 128)
    for where in (0, lengths[0] // 2, lengths[0] - new[0]):
        place = batch.place(0, where)
        host.put(place[0], 0, place[1], 0, np.full(128, 7, np.uint8), np.full(4, 131, np.uint8))
    q[0] = 3.0
    want, bound = K.attention_reference(host, batch, q, 0.3)
    K.check_attention(_attend(ctx, host, batch, q, 0.3), want, bound)
    host.arrays[0][:] = 0
    want, bound = K.attention_reference(host, batch, q, 0.3)
    K.check_attention(_attend(ctx, host, batch, q, 0.3), want, bound)


@pytest.mark.parametrize("new,lengths,d,window,sinks", [([1], [200], 128, 40, 3), ([1], [200], 512, 0, 0), ([20], [150], 64, 30, 5),
                                                        ([90], [100], 128, 17, 0), ([1, 3], [65, 40], 256, 0, 0)])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, new, lengths, d, window, sinks):
    """Every token that no row sees, the rest of the last pages and all unused pages hold blocks of NaN."""
    rng = np.random.default_rng(13)
    batch, host, q = _case(rng, new, lengths, 64, 2, 4, d)
    want, bound = K.attention_reference(host, batch, q, 0.1, window, sinks)
    keep = K.HostCache(batch.pages, 64, 2, d, fill=255)
    for b in range(len(new)):
        for j in range(lengths[b]):
            if any(j <= p and (not window or p - j < window or j < sinks) for p in batch.positions(b)):
                for h in range(2):
                    for which in (0, 1):
                        keep.put(*_place(batch, b, j, h), which, *host.get(*_place(batch, b, j, h), which))
    K.check_attention(_attend(ctx, keep, batch, q, 0.1, window, sinks), want, bound)


@pytest.mark.parametrize("new,length,window", [(1, 100, 0), (30, 100, 20), (70, 70, 8)])
def test_a_block_of_nan_reaches_exactly_the_rows_that_see_it(ctx, new, length, window):
    rng = np.random.default_rng(17)
    batch, host, q = _case(rng, [new], [length], 32, 1, 3, 128)
    bad_value, bad_key = length - new // 2 - 1, max(length - 3, 0)
    code, scale = host.get(*_place(batch, 0, bad_value, 0), 1)
    scale = scale.copy()
    scale[2] = 255
    host.put(*_place(batch, 0, bad_value, 0), 1, code, scale)       # values 64..95 of one token
    want, bound = K.attention_reference(host, batch, q, 0.1, window)
    assert np.isnan(want).any()
    K.check_attention(_attend(ctx, host, batch, q, 0.1, window), want, bound)
    code, scale = host.get(*_place(batch, 0, bad_key, 0), 0)
    scale = scale.copy()
    scale[0] = 255
    host.put(*_place(batch, 0, bad_key, 0), 0, code, scale)
    want, bound = K.attention_reference(host, batch, q, 0.1, window)
    K.check_attention(_attend(ctx, host, batch, q, 0.1, window), want, bound)


def test_rows_that_see_nothing_write_zeros_and_rows_behind_the_last_stay(ctx):
    rng = np.random.default_rng(19)
    batch, host, _ = _case(rng, [4, 2, 3], [2, 0, 64], 32, 1, 2, 64)   # two rows before position 0; an empty sequence
    q = K.bf16(rng.standard_normal((batch.total + 2, 2, 64)))
    want, bound = K.attention_reference(host, batch, q, 0.2)
    out = torch.full((batch.total + 2, 2, 64), 9.0, device="cuda")
    flag = _flag()
    ctx.kv_cache_attention_into(host.device(), batch.device(rows=batch.total + 2), torch.from_numpy(q).cuda(), out, 0.2, error=flag)
    got = out.cpu().numpy()
    assert (got[batch.total:] == 9).all() and (got[:2] == 0).all() and (got[4:6] == 0).all()
    K.check_attention(got[:batch.total], want[:batch.total], bound[:batch.total])


@pytest.mark.parametrize("new", [1, 40])
def test_attention_over_invalid_pages_skips_them_and_reports(ctx, new):
    rng = np.random.default_rng(23)
    batch, host, q = _case(rng, [new, 1], [200, 60], 32, 1, 2, 128)
    batch.table[0, 2], batch.table[0, 4] = batch.pages + 5, -1
    batch.table[1, :2] = -1                                         # the second sequence has no valid page at all
    want, bound = K.attention_reference(host, batch, q, 0.1)
    out = torch.empty((batch.total, 2, 128), dtype=torch.bfloat16, device="cuda")
    flag = _flag()
    ctx.kv_cache_attention_into(host.device(), batch.device(), torch.from_numpy(q).bfloat16().cuda(), out, 0.1, error=flag)
    K.check_attention(out.float().cpu().numpy(), want, bound)
    assert flag.item() == 1 and (out[new] == 0).all()


def test_attention_is_the_same_bits_again_and_whatever_stands_in_the_workspace(ctx):
    rng = np.random.default_rng(29)
    batch, host, q = _case(rng, [1, 1, 30], [4000, 40, 900], 64, 2, 8, 128)
    cache, dev = host.device(), batch.device()
    qd = torch.from_numpy(q).bfloat16().cuda()
    ws = ctx.kv_cache_attention_workspace(cache, dev, 16)
    outs = []
    for fill in (0, 255, 127):
        ws.fill_(fill)
        outs.append(ctx.kv_cache_attention_into(cache, dev, qd, torch.empty_like(qd), 0.09, workspace=ws))
    outs.append(ctx.kv_cache_attention_into(cache, dev, qd, torch.empty_like(qd), 0.09))
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    want, bound = K.attention_reference(host, batch, q, 0.09)
    K.check_attention(outs[0].float().cpu().numpy(), want, bound)


@pytest.mark.parametrize("bound_length", [1, 2000, 100000])
def test_the_bound_of_the_lengths_only_sizes_the_split(ctx, bound_length):
    rng = np.random.default_rng(31)
    batch, host, q = _case(rng, [1, 1], [1500, 2000], 128, 1, 8, 64)
    want, bound = K.attention_reference(host, batch, q, 0.125)
    K.check_attention(_attend(ctx, host, batch, q, 0.125, max_sequence_length=bound_length), want, bound)


def test_a_shared_prefix_and_the_same_page_twice(ctx):
    rng = np.random.default_rng(37)
    batch, host, q = _case(rng, [1, 2], [100, 100], 32, 1, 4, 128)
    batch.table[1, :3] = batch.table[0, :3]
    batch.table[0, 1] = batch.table[0, 0]
    want, bound = K.attention_reference(host, batch, q, 0.1)
    K.check_attention(_attend(ctx, host, batch, q, 0.1), want, bound)


def test_offsets_beyond_32_bits(ctx):
    """A cache of more than 4 GiB per array, the sequence on its last pages."""
    from ferrule_amd.provider import HipKvBatch
    heads, d, page = 8, 512, 1024
    pages = (1 << 32) // (heads * page * d // 2) + 3
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of GPU memory")
    cache = ctx.kv_cache(pages, page, heads, d)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    n = page + 40
    k, v = (torch.randn((n, heads, d), generator=gen, device="cuda").bfloat16() for _ in range(2))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = HipKvBatch(i32(0, n), i32(n), i32(pages - 1, pages - 2).view(1, 2), n)
    ctx.kv_cache_append(cache, batch, k, v)
    kd, vd = torch.empty_like(k), torch.empty_like(v)
    ctx.kv_cache_read_into(cache, batch, kd, vd)
    small = ctx.kv_cache(2, page, heads, d)
    near = HipKvBatch(i32(0, n), i32(n), i32(1, 0).view(1, 2), n)
    ctx.kv_cache_append(small, near, k, v)
    ks, vs = torch.empty_like(k), torch.empty_like(v)
    ctx.kv_cache_read_into(small, near, ks, vs)
    same = torch.equal(kd, ks) and torch.equal(vd, vs)
    # values below 6 have a scale of at most 1, whose widest step, 4 to 6, is off by half of it at most
    near_enough = ((kd.float() - k.float()).abs() <= 1.0).all().item() and k.abs().max().item() < 6
    assert same and near_enough
    q = torch.randn((n, heads, d), generator=gen, device="cuda").bfloat16()
    far, here = torch.empty_like(q), torch.empty_like(q)
    ctx.kv_cache_attention_into(cache, batch, q, far, 0.05)
    ctx.kv_cache_attention_into(small, near, q, here, 0.05)
    same = torch.equal(far, here) and torch.isfinite(far.float()).all().item()
    assert same


def test_a_step_captured_in_a_graph_follows_its_inputs(ctx):
    """append and attention of a decode step in one graph, replayed with new rows, lengths and tables, each replay
    against the eager run; eager work and synchronisations stand between the replays."""
    from ferrule_amd.provider import HipArtifactOperatorContext
    rng = np.random.default_rng(41)
    page, heads, group, d, seqs = 32, 2, 4, 128, 5
    cols, pages = 40, 200
    cache, eager = (K.HostCache(pages, page, heads, d).random(np.random.default_rng(43), 124, 128).device() for _ in range(2))
    from ferrule_amd.provider import HipKvBatch
    indptr = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    lengths = torch.ones(seqs, dtype=torch.int32, device="cuda")
    table = torch.zeros((seqs, cols), dtype=torch.int32, device="cuda")
    batch = HipKvBatch(indptr, lengths, table, seqs, 1, cols * page)
    k, v = (torch.zeros((seqs, heads, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros((seqs, heads * group, d), dtype=torch.bfloat16, device="cuda")
    out, want = torch.empty_like(q), torch.empty_like(q)
    stream = torch.cuda.Stream()
    side = HipArtifactOperatorContext(0, stream)
    ws = side.kv_cache_attention_workspace(cache, batch, heads * group, 900, 4)

    def refill():
        lengths.copy_(torch.from_numpy(rng.integers(1, cols * page, seqs).astype(np.int32)))
        table.copy_(torch.from_numpy(rng.permutation(pages).astype(np.int32)[:seqs * cols].reshape(seqs, cols)
                                     if pages >= seqs * cols else rng.integers(0, pages, (seqs, cols)).astype(np.int32)))
        for t in (k, v, q):
            t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
        torch.cuda.synchronize()

    refill()
    side.kv_cache_append(cache, batch, k, v)
    side.kv_cache_attention_into(cache, batch, q, out, 0.1, 900, 4, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        side.kv_cache_append(cache, batch, k, v)
        side.kv_cache_attention_into(cache, batch, q, out, 0.1, 900, 4, workspace=ws)
    ctx.kv_cache_append(eager, batch, k, v)
    for _ in range(4):
        refill()
        graph.replay()
        torch.cuda.synchronize()
        ctx.kv_cache_append(eager, batch, k, v)
        ctx.kv_cache_attention_into(eager, batch, q, want, 0.1, 900, 4)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip((cache.k_payload, cache.k_scales, cache.v_payload, cache.v_scales),
                        (eager.k_payload, eager.k_scales, eager.v_payload, eager.v_scales)):
            assert torch.equal(a, b)


def test_two_streams_with_their_own_workspaces(ctx):
    from ferrule_amd.provider import HipArtifactOperatorContext
    rng = np.random.default_rng(47)
    batch, host, q = _case(rng, [1, 1], [6000, 200], 64, 2, 8, 128)
    cache, dev = host.device(), batch.device()
    qd = torch.from_numpy(q).bfloat16().cuda()
    want = ctx.kv_cache_attention_into(cache, dev, qd, torch.empty_like(qd), 0.09)
    torch.cuda.synchronize()
    sides = [HipArtifactOperatorContext(0, torch.cuda.Stream()) for _ in range(2)]
    outs = [torch.empty_like(qd) for _ in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        sides[i % 2].kv_cache_attention_into(cache, dev, qd, o, 0.09)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_python_refusals(ctx):
    from ferrule_amd.provider import HipKvBatch, ProviderError
    cache = ctx.kv_cache(4, 32, 2, 64)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = HipKvBatch(i32(0, 2), i32(2), i32(0, 1).view(1, 2), 2)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    ctx.kv_cache_append(cache, batch, k, k)
    for bad in (k.half(), k[:1], k[:, :1], k.float(), torch.zeros((2, 2, 128), dtype=torch.bfloat16, device="cuda")[..., ::2]):
        with pytest.raises(ValueError):
            ctx.kv_cache_append(cache, batch, k, bad)
    with pytest.raises(ValueError):
        ctx.kv_cache_append(cache, batch, k, k.cpu())
    with pytest.raises(ValueError):
        ctx.kv_cache_append(cache, batch, k, k, error=torch.zeros(1, device="cuda"))
    odd = torch.zeros(2 * 2 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 2, 64)
    with pytest.raises(ProviderError):
        ctx.kv_cache_append(cache, batch, odd, k)                   # rows must start on 16 bytes
    q, out = (torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ctx.kv_cache_attention_into(cache, batch, q, out, 0.1)
    for kw in (dict(softmax_scale=0.0), dict(softmax_scale=float("nan"))):
        with pytest.raises(ProviderError):
            ctx.kv_cache_attention_into(cache, batch, q, out, **kw)
    for kw in (dict(window=-1), dict(window=3, sinks=-2), dict(workspace=torch.zeros(4, device="cuda"))):
        with pytest.raises(ValueError):
            ctx.kv_cache_attention_into(cache, batch, q, out, 0.1, **kw)
    with pytest.raises(ValueError):
        ctx.kv_cache_attention_into(cache, batch, q[:, :3], out[:, :3], 0.1)
    with pytest.raises(ValueError):
        ctx.kv_cache_attention_into(cache, batch, q, out[:, :2], 0.1)
    none = HipKvBatch(i32(0, 0), i32(0), i32(0, 1).view(1, 2), 0)
    ctx.kv_cache_append(cache, none, k[:0], k[:0])
    ctx.kv_cache_attention_into(cache, none, q[:0], out[:0], 0.1)


def test_projection_append_attention_and_output_projection_as_a_layer_runs_them(ctx):
    """Packed activations -> query and key/value rows (FP8 projections, f32 rows) -> cache -> attention over old and new
    tokens -> MXFP4 output projection, against the oracle's quantisers and float64."""
    from ferrule_amd.provider import HipArtifactLinearShape
    rng = np.random.default_rng(53)
    hidden, heads, group, d = 512, 2, 4, 128
    new, lengths = [5, 1, 2], [5, 90, 64]
    batch = K.HostBatch(rng, new, lengths, 32)
    host = K.HostCache(batch.pages, 32, heads, d).random(rng, 122, 126)
    cache, dev = host.device(), batch.device()
    x = K.bf16(rng.standard_normal((batch.total, hidden)))
    xq, xs = ctx.pack_fp8_rows_from_f32(torch.from_numpy(x).cuda())
    wq, sq = P.fp8_weight_e8m0(rng, heads * group * d, hidden)
    wkv, skv = P.fp8_weight_e8m0(rng, 2 * heads * d, hidden)
    dv = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    q, kv = ctx.fp8_query_a_kv(xq, xs, dv(wq), dv(sq), dv(wkv), dv(skv))
    q, kv = q.view(batch.total, heads * group, d), kv.view(batch.total, 2, heads, d)
    ctx.kv_cache_append(cache, dev, kv[:, 0], kv[:, 1])             # strided views of the projection's output
    attended = torch.empty((batch.total, heads * group, d), dtype=torch.bfloat16, device="cuda")
    ctx.kv_cache_attention_into(cache, dev, q, attended, d ** -0.5, window=40, sinks=4)
    wo, so = P.mxfp4_weight(rng, 256, heads * group * d)
    handle = ctx.upload_artifact_linear(HipArtifactLinearShape.fp4_e2m1_packed_with_e8m0_scale(256, heads * group * d), wo, so)
    y = ctx.artifact_linear_gemv_bf16(handle, attended.view(batch.total, -1))
    torch.cuda.synchronize()
    rows = kv.cpu().numpy()
    for b in range(3):
        for i, p in enumerate(batch.positions(b)):
            for h in range(heads):
                for which in (0, 1):
                    host.put(*_place(batch, b, p, h), which, *K.quantise(rows[batch.indptr[b] + i, which, h]))
    _same_bytes(cache, host)
    want, bound = K.attention_reference(host, batch, q.cpu().numpy(), d ** -0.5, 40, 4)
    K.check_attention(attended.float().cpu().numpy(), want, bound)
    a = attended.float().cpu().numpy().reshape(batch.total, -1).astype(np.float32)
    deq = po.dequantize_fp4(wo, so, 256, heads * group * d).astype(np.float64)
    worst, _ = P.compare_bf16(y.view(torch.int16).cpu().numpy().view(np.uint16),
                              po.linear_fp4(wo, so, 256, heads * group * d, a), np.abs(a.astype(np.float64)) @ np.abs(deq).T,
                              heads * group * d)
    assert worst <= 2
