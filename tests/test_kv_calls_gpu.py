"""Calls of the key/value cache operators that their documentation allows: contexts with streams of their own, padded row
tensors, rows in front of position 0, several sequences in each order of workgroups.  Same float64 reference and derived
bound as tests/test_kv_cache_gpu.py."""
import numpy as np
import pytest

from tests import kv_helpers as K
from tests.test_kv_cache_gpu import _attend, _case, ctx  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_rows_appended_at_once_to_a_new_cache_of_a_side_context_stay(ctx):  # noqa: F811
    """A cache of 1.1 GB, whose fill takes a while, and rows on its last pages; nothing waits in between."""
    from ferrule_amd.provider import HipArtifactOperatorContext, HipKvBatch
    pages, page, heads, d, n = 4096, 64, 16, 256, 100
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    k, v = (torch.randn((n, heads, d), generator=gen, device="cuda").bfloat16() for _ in range(2))
    batch = HipKvBatch(_i32(0, n), _i32(n), _i32(pages - 1, pages - 2).view(1, 2), n)
    near = HipKvBatch(_i32(0, n), _i32(n), _i32(1, 0).view(1, 2), n)
    small = ctx.kv_cache(2, page, heads, d)
    ctx.kv_cache_append(small, near, k, v)
    torch.cuda.synchronize()
    side = HipArtifactOperatorContext(0, torch.cuda.Stream())
    cache = side.kv_cache(pages, page, heads, d)
    side.kv_cache_append(cache, batch, k, v)
    torch.cuda.synchronize()
    for far, here in zip((cache.k_payload, cache.k_scales, cache.v_payload, cache.v_scales),
                         (small.k_payload, small.k_scales, small.v_payload, small.v_scales)):
        assert torch.equal(far[-2:], here) and not far[:-2].any()


def test_a_workspace_dropped_after_its_call_is_not_handed_out_while_it_is_in_use(ctx):  # noqa: F811
    """A split decode step on a side stream whose workspace nobody keeps; torch's own stream takes blocks of that size and
    fills them at once."""
    from ferrule_amd.provider import HipArtifactOperatorContext
    rng = np.random.default_rng(131)
    batch, host, q = _case(rng, [1, 1], [6000, 2000], 64, 2, 8, 128)
    cache, dev = host.device(), batch.device()
    qd = torch.from_numpy(q).bfloat16().cuda()
    want = ctx.kv_cache_attention_into(cache, dev, qd, torch.empty_like(qd), 0.09)
    size = ctx.kv_cache_attention_workspace(cache, dev, 16).numel()
    assert size > 0
    side = HipArtifactOperatorContext(0, torch.cuda.Stream())
    outs = [torch.empty_like(qd) for _ in range(8)]
    torch.cuda.synchronize()
    for out in outs:
        side.kv_cache_attention_into(cache, dev, qd, out, 0.09, workspace=side.kv_cache_attention_workspace(cache, dev, 16))
        torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    same = [torch.equal(out, want) for out in outs]
    assert all(same), same


@pytest.mark.parametrize("new,lengths,d", [([1], [1000], 128), ([3, 1], [700, 90], 256), ([40], [200], 64), ([1, 1], [6000, 100], 512)])
def test_outputs_over_the_queries_are_refused_and_beside_them_in_one_buffer_are_not(ctx, new, lengths, d):  # noqa: F811
    from ferrule_amd.provider import ProviderError
    rng = np.random.default_rng(137)
    batch, host, q = _case(rng, new, lengths, 64, 2, 4, d)
    cache, dev, rows, heads = host.device(), batch.device(), batch.total, 8
    qd = torch.from_numpy(q).bfloat16().cuda()
    want = ctx.kv_cache_attention_into(cache, dev, qd, torch.empty_like(qd), 0.09)

    def views(buffer, type_q, type_o, split):
        b = torch.zeros(buffer, dtype=torch.uint8, device="cuda").view(*buffer[:-1], -1)
        first, second = split(b)
        first, second = first.view(type_q), second.view(type_o)
        return first.copy_(qd), second

    half, full = torch.bfloat16, torch.float32
    for kind in (half, full):
        size = 2 if kind is half else 4
        for first, second in (views((rows, 2, heads, size * d), kind, kind, lambda b: (b[:, 0], b[:, 1])),
                              views((rows, heads, 2, size * d), kind, kind, lambda b: (b[:, :, 1], b[:, :, 0])),
                              views((2, rows, heads, size * d), kind, kind, lambda b: (b[1], b[0])),
                              views((heads, rows, 2, size * d), kind, kind, lambda b: (b[:, :, 0].transpose(0, 1), b[:, :, 1].transpose(0, 1)))):
            ctx.kv_cache_attention_into(cache, dev, first, second, 0.09)
            assert torch.equal(first.bfloat16(), qd) and torch.equal(second.bfloat16(), want)
    n, shift = qd.numel(), heads // 2 * d                         # half a row
    flat = torch.zeros(n + shift, dtype=half, device="cuda")
    front, back = flat[:n].view_as(qd), flat[shift:].view_as(qd)
    wide = torch.zeros((rows, heads, 2 * d), dtype=half, device="cuda")
    for a, b in ((front, front), (front, back), (back, front), (wide[..., :d], wide[..., d // 2:d // 2 + d]),
                 (qd, torch.empty((1, 1, d), dtype=half, device="cuda").expand(rows, heads, d))):
        with pytest.raises((ValueError, ProviderError)):
            ctx.kv_cache_attention_into(cache, dev, a, b, 0.09)


def test_read_into_one_place_is_refused_and_side_by_side_is_not(ctx):  # noqa: F811
    from ferrule_amd.provider import ProviderError
    rng = np.random.default_rng(139)
    batch, host, _ = _case(rng, [40, 7], [90, 7], 32, 2, 1, 128)
    cache, dev, n = host.device(), batch.device(), batch.total
    want = [torch.empty((n, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ctx.kv_cache_read_into(cache, dev, *want)
    for both in (torch.empty((n, 2, 2, 128), dtype=torch.bfloat16, device="cuda"), torch.empty((n, 2, 2, 128), device="cuda")):
        for k, v in ((both[:, 0], both[:, 1]), (both[:, :, 1], both[:, :, 0])):
            ctx.kv_cache_read_into(cache, dev, k, v)
            assert torch.equal(k.bfloat16(), want[0]) and torch.equal(v.bfloat16(), want[1])
    k, v = want
    for pair in ((k, k), (k, k.view(-1)[:128].view(1, 1, 128).expand(n, 2, 128)), (v[:1].expand(n, 2, 128), k),
                 (both[:, 0, :1].expand(n, 2, 128), both[:, 1])):
        with pytest.raises((ValueError, ProviderError)):
            ctx.kv_cache_read_into(cache, dev, *pair)


@pytest.mark.parametrize("new,lengths,heads,group,d,most", [
    ([1], [9000], 1, 8, 128, 1), ([2, 1, 2], [3000, 700, 5000], 2, 4, 64, 2), ([1, 0, 1], [6000, 0, 40], 1, 16, 512, 1),
    ([40, 33], [2500, 4000], 1, 2, 128, 45), ([20, 1], [3000, 4000], 1, 8, 256, 20)])
@pytest.mark.parametrize("behind", [1, 300])
def test_partials_of_row_tensors_longer_than_their_sequences_stay_in_the_workspace(ctx, new, lengths, heads, group, d, most, behind):  # noqa: F811
    """Split ranges; the workspace is what the entry asks for, and what stands behind it stays as it was."""
    rng = np.random.default_rng(149 + d)
    batch, host, q = _case(rng, new, lengths, 64, heads, group, d)
    want, bound = K.attention_reference(host, batch, q, 0.09)
    rows = len(new) * most + behind
    qd = torch.ones((rows, heads * group, d), dtype=torch.bfloat16, device="cuda")
    qd[:batch.total].copy_(torch.from_numpy(q))
    out = torch.full_like(qd, 9.0)
    cache, dev = host.device(), batch.device(rows=rows, max_query_length=most)
    size = ctx.kv_cache_attention_workspace(cache, dev, heads * group).numel()
    assert size > 0
    memory = torch.full((size + 4096,), 129, dtype=torch.uint8, device="cuda")
    ctx.kv_cache_attention_into(cache, dev, qd, out, 0.09, workspace=memory[:size])
    got = out.float().cpu().numpy()
    assert (got[batch.total:] == 9).all() and (memory[size:] == 129).all()
    K.check_attention(got[:batch.total], want, bound)


@pytest.mark.parametrize("d,group", [(64, 8), (128, 8), (256, 4), (512, 16)])
def test_one_workspace_of_the_largest_bounds_serves_every_smaller_step(ctx, d, group):  # noqa: F811
    """Asked for once; steps of fewer sequences, rows and tokens, with windows and without, decode rows beside a prompt."""
    from ferrule_amd.provider import HipKvBatch
    rng = np.random.default_rng(151 + d)
    heads, page, longest = 2, 64, 9000
    most = HipKvBatch(_i32(*range(65)), _i32(*[longest] * 64), torch.zeros((64, 141), dtype=torch.int32, device="cuda"), 700, 600, longest)
    cache = K.HostCache(900, page, heads, d).random(rng, 124, 128).device()
    size = ctx.kv_cache_attention_workspace(cache, most, heads * group).numel()
    memory = torch.full((size + 4096,), 129, dtype=torch.uint8, device="cuda")
    cut = 0
    for new, lengths in (([1], [9000]), ([1] * 5, [8000, 3, 700, 2500, 9000]), ([1] * 33, [2100] * 33), ([1] * 64, [4000] * 64), ([600], [600]),
                         ([300], [8000]), ([64, 1, 3], [64, 9000, 5000]), ([500, 1, 1, 1], [5000, 40, 9000, 6000]), ([2] * 17, [5000] * 17)):
        table = torch.from_numpy(rng.integers(0, 900, (len(new), 141)).astype(np.int32)).cuda()
        starts = np.concatenate([[0], np.cumsum(new)]).tolist()
        dev = HipKvBatch(_i32(*starts), _i32(*lengths), table, sum(new), max(new), max(lengths))
        q = torch.randn((sum(new), heads * group, d), device="cuda").bfloat16()
        for window, sinks in ((0, 0), (700, 4), (8000, 0)):
            memory[:size] = 255
            got = ctx.kv_cache_attention_into(cache, dev, q, torch.empty_like(q), 0.09, window, sinks, workspace=memory[:size])
            cut += not bool((memory[:size] == 255).all())
            want = ctx.kv_cache_attention_into(cache, dev, q, torch.empty_like(q), 0.09, window, sinks)
            same = torch.equal(got, want) and bool(torch.isfinite(got).all()) and bool((memory[size:] == 129).all())
            assert same, (new, lengths, window)
    assert cut >= 8                                             # steps that used it


@pytest.mark.parametrize("new,lengths,heads,group,d,window,sinks", [
    # 17 to 32 packed rows over more than 2048 tokens: both tiles of every sequence, ragged, in several heads
    ([3, 3, 3], [2500, 4100, 2070], 3, 8, 128, 0, 0), ([5, 5], [2600, 5000], 2, 5, 64, 0, 0), ([4, 4, 4, 4], [2300, 40, 4, 3000], 2, 8, 128, 2200, 3),
    ([2, 2, 2], [2200, 2900, 700], 2, 16, 256, 0, 0), ([32, 32], [2400, 3300], 3, 1, 64, 2250, 40), ([2, 2], [2700, 2100], 4, 9, 256, 2090, 5),
    # bounds that fit the rows though no sequence has so many: 16 = 4 * 4 rows, 24 = 3 * 8
    ([13, 1, 1, 1], [2500, 4000, 2600, 50], 2, 8, 128, 0, 0), ([20, 3, 1], [2600, 2400, 3000], 2, 4, 64, 2300, 4),
    # as many rows as sequences times the bound, not all of them there
    ([3, 1, 2], [2500, 2600, 4000], 2, 8, 128, 0, 0)])
@pytest.mark.parametrize("types", ["bf16", "f32"])
def test_two_tiles_of_few_rows_in_every_order_of_workgroups(ctx, new, lengths, heads, group, d, window, sinks, types):  # noqa: F811
    rng = np.random.default_rng(157 + d)
    batch, host, q = _case(rng, new, lengths, 64, heads, group, d)
    want, bound = K.attention_reference(host, batch, q, 0.09, window, sinks, f32_output=types == "f32")
    t = torch.float32 if types == "f32" else torch.bfloat16
    K.check_attention(_attend(ctx, host, batch, q, 0.09, window, sinks, t, t), want, bound)
    rows = len(new) * max(new)                                  # padded to the bound
    qd = torch.ones((rows, heads * group, d), dtype=t, device="cuda")
    qd[:batch.total].copy_(torch.from_numpy(q))
    out = torch.full_like(qd, 9.0)
    ctx.kv_cache_attention_into(host.device(), batch.device(rows=rows), qd, out, 0.09, window=window, sinks=sinks)
    got = out.float().cpu().numpy()
    assert (got[batch.total:] == 9).all()
    K.check_attention(got[:batch.total], want, bound)


@pytest.mark.parametrize("new,lengths,heads,group,d", [
    # one token a sequence, verification rows, and rows for each of the kernels; over short ranges and split ones
    ([1, 2, 1], [40, 1, 300], 2, 4, 128), ([1, 1], [9, 0], 1, 8, 64), ([2, 3], [5000, 2], 1, 4, 256), ([1, 4], [300, 3], 1, 16, 512),
    ([90, 40], [60, 300], 1, 2, 64), ([270, 3], [269, 3], 1, 1, 128), ([150], [1], 1, 1, 256), ([60, 1], [40, 1], 1, 2, 512),
    ([40, 1, 2], [2500, 4000, 1], 1, 8, 128)])
def test_rows_in_front_of_position_0_are_reported_by_all_three_operators(ctx, new, lengths, heads, group, d):  # noqa: F811
    rng = np.random.default_rng(163 + d)
    for short in (True, False):
        tokens = lengths if short else [max(n, length) for n, length in zip(new, lengths)]
        batch, host, q = _case(rng, new, tokens, 32, heads, group, d)
        want, bound = K.attention_reference(host, batch, q, 0.1)
        cache, dev = host.device(), batch.device()
        rows = torch.ones((batch.total, heads, d), device="cuda")
        qd = torch.from_numpy(q).cuda()
        out = torch.full_like(qd, 9.0)
        flags = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(3)]
        ctx.kv_cache_attention_into(cache, dev, qd, out, 0.1, error=flags[0])
        ctx.kv_cache_read_into(cache, dev, torch.empty_like(rows), torch.empty_like(rows), flags[1])
        ctx.kv_cache_append(cache, dev, rows, rows, flags[2])
        K.check_attention(out.cpu().numpy(), want, bound)
        assert [f.item() for f in flags] == [int(short)] * 3


def test_one_row_with_a_stride_off_16_bytes(ctx):  # noqa: F811
    """A projection's single row of an odd width: keys, values and queries are views of it."""
    rng = np.random.default_rng(167)
    batch, host, _ = _case(rng, [1], [90], 32, 2, 4, 64)
    cache, dev, width = host.device(), batch.device(), 12 * 64 + 1
    row = torch.randn(width, device="cuda").bfloat16()
    view = lambda first, heads: torch.as_strided(row, (1, heads, 64), (width, 64, 1), 64 * first)  # noqa: E731
    ctx.kv_cache_append(cache, dev, view(0, 2), view(2, 2))
    k, v = (torch.as_strided(torch.empty(130, dtype=torch.bfloat16, device="cuda"), (1, 2, 64), (129, 64, 1)) for _ in range(2))
    ctx.kv_cache_read_into(cache, dev, k, v)
    out = torch.as_strided(torch.empty(520, dtype=torch.bfloat16, device="cuda"), (1, 8, 64), (519, 64, 1))
    ctx.kv_cache_attention_into(cache, dev, view(4, 8), out, 0.1)
    x = row.float().cpu().numpy()
    for h in range(2):
        for which in (0, 1):
            at = 64 * (2 * which + h)
            host.put(batch.table[0, 2], h, 89 - 64, which, *K.quantise(x[at:at + 64]))
            assert np.array_equal((k, v)[which][0, h].float().cpu().numpy(), host.value(batch.table[0, 2], h, 89 - 64, which).astype(np.float32))
    want, bound = K.attention_reference(host, batch, x[256:768].reshape(1, 8, 64), 0.1)
    K.check_attention(out.float().cpu().numpy(), want, bound)


def test_offsets_of_scale_bytes_beyond_32_bits(ctx):  # noqa: F811
    """Scale arrays of more than 4 GiB (and so payloads of more than 64), the sequence on the last pages; nothing is filled."""
    from ferrule_amd.provider import HipKvBatch, HipKvCache, kv_cache_shapes
    heads, d, page = 8, 64, 1024
    pages = (1 << 32) // (heads * page * d // 32) + 3
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GiB of GPU memory")
    cache = HipKvCache(page, heads, d, *(torch.empty(s, dtype=torch.uint8, device="cuda") for s in kv_cache_shapes(pages, page, heads, d)))
    assert cache.k_scales.numel() > 1 << 32 and cache.v_scales.numel() > 1 << 32
    small = ctx.kv_cache(2, page, heads, d)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7)
    n = page + 40
    k, v, q = (torch.randn((n, heads, d), generator=gen, device="cuda").bfloat16() for _ in range(3))
    outs = []
    for held, table in ((cache, _i32(pages - 1, pages - 2)), (small, _i32(1, 0))):
        batch = HipKvBatch(_i32(0, n), _i32(n), table.view(1, 2), n)
        ctx.kv_cache_append(held, batch, k, v)
        kd, vd, rows = (torch.empty_like(k) for _ in range(3))
        ctx.kv_cache_read_into(held, batch, kd, vd)
        ctx.kv_cache_attention_into(held, batch, q, rows, 0.1)
        last = HipKvBatch(_i32(0, 1), _i32(n), table.view(1, 2), 1)
        one = ctx.kv_cache_attention_into(held, last, q[-1:], torch.empty_like(q[-1:]), 0.1)
        outs.append((kd, vd, rows, one))
    same = [torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(*outs)]
    del cache
    torch.cuda.empty_cache()
    assert all(same), same
    assert ((outs[0][0] - k).abs() <= 1).all() and ((outs[0][1] - v).abs() <= 1).all() and k.abs().max().item() < 6 > v.abs().max().item()


def test_bytes_copied_at_once_into_a_new_cache_of_a_side_context_stay():
    """On torch's own stream, with nothing waited for; the cache is large, so that its fill takes a while."""
    from ferrule_amd.provider import HipArtifactOperatorContext
    side = HipArtifactOperatorContext(0, torch.cuda.Stream())
    cache = side.kv_cache(4096, 64, 16, 256)
    for t in (cache.v_scales, cache.k_scales, cache.v_payload, cache.k_payload):
        t[-1].fill_(77)
    torch.cuda.synchronize()
    for t in (cache.v_scales, cache.k_scales, cache.v_payload, cache.k_payload):
        assert (t[-1] == 77).all() and not t[:-1].any()
