"""Attention over the MXFP4 cache in each of its kernels: token ranges in several parts and their joins, short ranges,
blocks that are not finite, graphs.  Same float64 reference and derived bound as tests/test_kv_cache_gpu.py."""
import numpy as np
import pytest

from tests import kv_helpers as K
from tests.test_kv_cache_gpu import _attend, _case, _place, ctx  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

MANY = [1] * 135  # two key/value heads: more segments than the card has CUs


def _many_lengths():
    rng = np.random.default_rng(3)
    lengths = rng.integers(1, 60, len(MANY))
    lengths[[0, 7, 77, 134]] = 600, 513, 512, 255
    return lengths.tolist()


PARTS = [  # new rows, lengths, page, kv heads, group, head size, window, sinks
    # few rows: parts of eight 32-token tiles, joined eight or fewer at a time or in chunks
    ([1], [5000], 64, 1, 2, 64, 0, 0), ([1, 1], [5000, 330], 32, 1, 8, 128, 0, 0), ([2], [4700], 128, 1, 8, 256, 0, 0),
    ([1, 2], [4700, 257], 64, 1, 16, 512, 0, 0), ([1], [500], 32, 1, 16, 512, 0, 0), ([3], [6000], 64, 1, 8, 128, 4500, 40),
    (MANY, _many_lengths(), 32, 2, 2, 64, 0, 0), (MANY, _many_lengths(), 64, 2, 3, 128, 300, 5),
    # many rows: parts of sixteen tiles and more
    ([100], [5000], 64, 1, 1, 64, 0, 0), ([20, 9], [3100, 1700], 64, 1, 2, 128, 0, 0), ([60], [2500], 32, 1, 2, 128, 0, 0),
    ([300], [2000], 64, 1, 1, 64, 0, 0), ([300, 1], [2000, 700], 128, 1, 1, 128, 1500, 40), ([150], [2000], 256, 1, 1, 256, 0, 0),
    ([50], [1800], 32, 1, 1, 256, 0, 0), ([70], [1500], 64, 1, 1, 512, 0, 0), ([2], [1200], 64, 1, 64, 512, 900, 3),
]


@pytest.mark.parametrize("types", ["bf16", "f32"])
@pytest.mark.parametrize("new,lengths,page,heads,group,d,window,sinks", PARTS)
def test_ranges_in_parts_equal_float64(ctx, new, lengths, page, heads, group, d, window, sinks, types):  # noqa: F811
    rng = np.random.default_rng(len(new) + d + lengths[0])
    batch, host, q = _case(rng, new, lengths, page, heads, group, d)
    scale = float(d) ** -0.5
    want, bound = K.attention_reference(host, batch, q, scale, window, sinks, f32_output=types == "f32")
    t = torch.float32 if types == "f32" else torch.bfloat16
    K.check_attention(_attend(ctx, host, batch, q, scale, window, sinks, t, t), want, bound)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("length", [255, 256, 257, 289, 513, 2015, 2016, 2047, 2049])
def test_short_ranges_around_the_shares_of_the_waves(ctx, d, length):  # noqa: F811
    rng = np.random.default_rng(length)
    batch, host, q = _case(rng, [1, 2], [length, 1 + length // 3], 64, 1, 3, d)
    for window, sinks in ((0, 0), (length - 20, 1)):
        want, bound = K.attention_reference(host, batch, q, 0.1, window, sinks)
        K.check_attention(_attend(ctx, host, batch, q, 0.1, window, sinks), want, bound)


@pytest.mark.parametrize("new,lengths,group,window,sinks", [
    ([1, 1, 1], [16, 700, 129], 64, 128, 4), ([2, 1], [90, 5], 32, 0, 0), ([1, 3], [300, 64], 16, 100, 0), ([1], [1], 33, 0, 0),
    ([1, 1], [2000, 250], 64, 160, 4)])
def test_heads_of_512_over_short_ranges(ctx, new, lengths, group, window, sinks):  # noqa: F811
    rng = np.random.default_rng(61)
    batch, host, q = _case(rng, new, lengths, 64, 1, group, 512)
    want, bound = K.attention_reference(host, batch, q, 0.05, window, sinks)
    K.check_attention(_attend(ctx, host, batch, q, 0.05, window, sinks), want, bound)


def test_more_sequences_than_a_small_table(ctx):  # noqa: F811
    rng = np.random.default_rng(67)
    lengths = rng.integers(0, 5, 700).tolist()
    batch, host, q = _case(rng, [min(n, 1) for n in lengths], lengths, 32, 1, 2, 64)
    want, bound = K.attention_reference(host, batch, q, 0.1)
    K.check_attention(_attend(ctx, host, batch, q, 0.1), want, bound)


EVERY_KERNEL = [  # new rows, lengths, group, head size, window, sinks
    ([1], [300], 4, 64, 0, 0), ([1], [300], 4, 128, 100, 5), ([1, 2], [2300, 40], 4, 128, 0, 0), ([1], [300], 4, 256, 0, 0),
    ([1], [2300], 2, 256, 2100, 1), ([1], [400], 16, 512, 0, 0), ([1], [130], 64, 512, 100, 3), ([50], [130], 1, 64, 20, 2),
    ([100], [130], 1, 64, 0, 0), ([270], [300], 1, 64, 50, 0), ([50], [700], 1, 128, 0, 0), ([100], [130], 1, 128, 33, 1),
    ([270], [300], 1, 128, 0, 0), ([50], [130], 1, 256, 0, 0), ([100], [700], 1, 256, 40, 0), ([50], [130], 2, 512, 30, 3),
    ([270], [700], 1, 64, 0, 0), ([100], [700], 1, 64, 0, 0), ([270], [800], 1, 128, 600, 3), ([100], [700], 1, 128, 0, 0),
    ([100], [800], 1, 256, 620, 2), ([40, 3], [2500, 600], 1, 128, 0, 0), ([60], [2400], 1, 64, 0, 0), ([45], [2500], 1, 256, 2200, 3),
    ([30], [700], 2, 512, 0, 0),
]


@pytest.mark.parametrize("scale_byte,nibbles", [(255, 0x00), (254, 0xf7), (253, 0x6e)])
@pytest.mark.parametrize("new,lengths,group,d,window,sinks", EVERY_KERNEL)
def test_unseen_blocks_of_nan_and_beyond_the_range_of_f32_reach_nobody(ctx, new, lengths, group, d, window, sinks,  # noqa: F811
                                                                       scale_byte, nibbles):
    rng = np.random.default_rng(71)
    batch, host, q = _case(rng, new, lengths, 64, 1, group, d)
    want, bound = K.attention_reference(host, batch, q, 0.1, window, sinks)
    keep = K.HostCache(batch.pages, 64, 1, d, fill=nibbles)
    keep.arrays[1][:] = keep.arrays[3][:] = scale_byte
    for b in range(len(new)):
        seen = np.zeros(lengths[b], bool)
        for p in batch.positions(b):
            j = np.arange(lengths[b])
            seen |= (j <= p) & ((window == 0) | (p - j < window) | (j < sinks))
        for j in np.flatnonzero(seen):
            for which in (0, 1):
                keep.put(*_place(batch, b, j, 0), which, *host.get(*_place(batch, b, j, 0), which))
    K.check_attention(_attend(ctx, keep, batch, q, 0.1, window, sinks), want, bound)


@pytest.mark.parametrize("new,lengths,group,d,window,sinks", EVERY_KERNEL)
def test_a_row_takes_its_own_nan_and_not_its_neighbours(ctx, new, lengths, group, d, window, sinks):  # noqa: F811
    """One block of NaN at the first rows' position: the rows from there on see it, within the window."""
    rng = np.random.default_rng(73)
    batch, host, q = _case(rng, new, lengths, 32, 1, group, d)
    places = [(0, lengths[0] - (new[0] + 1) // 2, d // 32 - 1), (0, max(0, lengths[0] - 40), 0)]
    for b, j, block in places:
        code, scale = host.get(*_place(batch, b, j, 0), 1)
        scale = scale.copy()
        scale[block] = 255
        host.put(*_place(batch, b, j, 0), 1, code, scale)
    want, bound = K.attention_reference(host, batch, q, 0.1, window, sinks)
    assert np.isnan(want).any()
    K.check_attention(_attend(ctx, host, batch, q, 0.1, window, sinks), want, bound)


def test_the_widest_window_is_no_window(ctx):  # noqa: F811
    """Also with rows in front of position 0, which see nothing."""
    rng = np.random.default_rng(79)
    for new, lengths in (([1, 4], [300, 2]), ([90, 40], [60, 300])):
        batch, host, q = _case(rng, new, lengths, 32, 1, 2, 64)
        want = _attend(ctx, host, batch, q, 0.1)
        for sinks in (0, 0x7fffffff):
            got = _attend(ctx, host, batch, q, 0.1, 0x7fffffff, sinks)
            assert np.array_equal(got, want)
        reference, bound = K.attention_reference(host, batch, q, 0.1)
        K.check_attention(want, reference, bound)


def test_an_infinity_or_a_nan_of_a_query_stays_in_its_row(ctx):  # noqa: F811
    rng = np.random.default_rng(83)
    for new, lengths, d in (([2], [300], 128), ([1, 1], [300, 40], 512), ([60], [90], 64)):
        batch, host, q = _case(rng, new, lengths, 32, 1, 2, d)
        want, bound = K.attention_reference(host, batch, q, 0.1)
        q[0, 1, 5], q[1, 0, d - 1] = np.inf, np.nan
        got = _attend(ctx, host, batch, q, 0.1)
        lost = np.zeros(got.shape, bool)
        lost[0, 1], lost[1, 0] = True, True
        K.check_attention(got, np.where(lost, np.nan, want), bound)


def test_two_graphs_share_a_workspace_when_they_follow_each_other(ctx):  # noqa: F811
    """A split decode step and a split prompt chunk, captured with one workspace and replayed in turn on one stream."""
    from ferrule_amd.provider import HipArtifactOperatorContext
    rng = np.random.default_rng(89)
    steps = []
    for new, lengths, group, d in (([1, 1], [3500, 2600], 4, 128), ([70], [2400], 1, 128)):
        batch, host, q = _case(rng, new, lengths, 64, 2, group, d)
        steps.append((host.device(), batch.device(), torch.from_numpy(q).bfloat16().cuda(), 2 * group))
    stream = torch.cuda.Stream()
    side = HipArtifactOperatorContext(0, stream)
    ws = max((side.kv_cache_attention_workspace(c, b, heads) for c, b, _, heads in steps), key=lambda t: t.numel())
    outs = [torch.empty_like(q) for _, _, q, _ in steps]
    run = lambda who, i, out, **kw: who.kv_cache_attention_into(*steps[i][:2], steps[i][2], out, 0.09, **kw)  # noqa: E731
    torch.cuda.synchronize()
    for i in range(2):
        run(side, i, outs[i], workspace=ws)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=stream):
            run(side, i, outs[i], workspace=ws)
    for turn in range(4):
        for _, _, q, _ in steps:
            q.copy_(torch.from_numpy(rng.standard_normal(q.shape).astype(np.float32)))
        torch.cuda.synchronize()
        for i in range(2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = run(ctx, i, torch.empty_like(outs[i]))
            same = torch.equal(outs[i], want)
            assert same, (turn, i)


@pytest.mark.parametrize("new,d", [(1, 64), (1, 128), (1, 256), (1, 512), (90, 64), (90, 128)])
def test_value_blocks_beyond_the_range_of_f32_count_as_nan(ctx, new, d):  # noqa: F811
    rng = np.random.default_rng(97)
    batch, host, q = _case(rng, [new], [200], 32, 1, 1, d)
    for j, byte in ((100, 253), (90, 254), (80, 252)):                  # 2^125 * 6 is finite: a value like any other
        code, scale = host.get(*_place(batch, 0, j, 0), 1)
        scale = scale.copy()
        scale[(byte - 252) % (d // 32)] = byte
        host.put(*_place(batch, 0, j, 0), 1, code, scale)
    got = _attend(ctx, host, batch, q, 0.1)
    blocks = np.isnan(got).reshape(*got.shape[:2], -1, 32)
    lost = np.zeros(d // 32, bool)
    lost[[1 % (d // 32), 2 % (d // 32)]] = True
    assert (blocks == lost[None, None, :, None]).all()


@pytest.mark.parametrize("n,length,heads,group,d,window,sinks", [
    (2100, 2100, 1, 64, 64, 0, 0), (2100, 2300, 2, 32, 128, 0, 0), (1100, 1100, 2, 32, 256, 0, 0), (2200, 2200, 1, 64, 128, 900, 7),
    (1030, 1030, 4, 16, 128, 0, 0), (600, 600, 1, 64, 512, 0, 0), (2100, 2100, 1, 64, 64, 700, 3), (1100, 1100, 1, 64, 256, 600, 1),
    (1100, 1100, 1, 64, 128, 600, 40), (1100, 1200, 1, 64, 64, 530, 0), (300, 300, 1, 64, 512, 128, 4)])
def test_prompts_of_many_rows_equal_float64(ctx, n, length, heads, group, d, window, sinks):  # noqa: F811
    """Enough rows for the largest workgroups.  The reference is float64 on the GPU over the values that the read operator
    gives back (exact), the bound that of tests/kv_helpers.py."""
    rng = np.random.default_rng(n + d)
    batch, host, q = _case(rng, [n], [length], 64, heads, group, d)
    cache, dev = host.device(), batch.device()
    qd = torch.from_numpy(q).bfloat16().cuda()
    out = ctx.kv_cache_attention_into(cache, dev, qd, torch.empty_like(qd), d ** -0.5, window=window, sinks=sinks)
    every = K.HostBatch.__new__(K.HostBatch)                            # all tokens as rows
    every.__dict__ = dict(batch.__dict__, new=[length], indptr=np.array([0, length], np.int32))
    k, v = (torch.empty((length, heads, d), device="cuda") for _ in range(2))
    ctx.kv_cache_read_into(cache, every.device(), k, v)
    p = torch.arange(length - n, length, device="cuda")[:, None]
    j = torch.arange(length, device="cuda")[None, :]
    seen = (j <= p) & ((p - j < window) | (j < sinks)) if window else j <= p
    count = seen.sum(1, keepdim=True).double()
    for h in range(heads * group):
        qs, ks, vs = qd[:, h].double(), k[:, h // group].double(), v[:, h // group].double()
        w = torch.softmax((qs @ ks.T * d ** -0.5).masked_fill(~seen, -np.inf), -1)
        want, size = w @ vs, w @ vs.abs()
        most = (qs.abs() @ ks.abs().T * d ** -0.5).masked_fill(~seen, 0).amax(-1, keepdim=True)
        e = most * (32 * 2.0 ** -20 + d * 2.0 ** -23 + 2.0 ** -20) + 2.0 ** -20
        bound = size * (2.0 ** -8 + 2.2 * e + 2 * count * 2.0 ** -23) + want.abs() * 2.0 ** -8 + 1e-37
        worst = ((out[:, h].double() - want).abs() / bound).max().item()
        assert worst <= 1, (h, worst)


def test_windows_beyond_31_bits_are_refused(ctx):  # noqa: F811
    rng = np.random.default_rng(1)
    batch, host, q = _case(rng, [1], [40], 32, 1, 1, 64)
    for kw in (dict(window=2 ** 31), dict(window=2 ** 32 + 5), dict(window=5, sinks=2 ** 32)):
        with pytest.raises(ValueError):
            _attend(ctx, host, batch, q, 0.1, **kw)


MIXED = [  # new rows, lengths, kv heads, group, head size, window, sinks
    ([300, 1, 1, 3, 40, 1], [2500, 3000, 40, 2200, 2100, 1], 1, 2, 128, 0, 0), ([1, 70, 0, 2], [4000, 2100, 0, 600], 2, 4, 64, 0, 0),
    ([100, 1, 2], [2300, 2700, 2048], 1, 4, 256, 0, 0), ([40, 1, 1], [2200, 2300, 50], 1, 8, 512, 0, 0),
    ([150, 1, 5, 1], [2600, 2600, 2600, 90], 1, 8, 128, 2100, 3), ([200, 1, 1], [2400, 2400, 3], 1, 40, 64, 0, 0),
]


@pytest.mark.parametrize("types", ["bf16", "f32"])
@pytest.mark.parametrize("new,lengths,heads,group,d,window,sinks", MIXED)
def test_sequences_of_few_and_of_many_rows_in_one_batch(ctx, new, lengths, heads, group, d, window, sinks, types):  # noqa: F811
    rng = np.random.default_rng(101 + d)
    batch, host, q = _case(rng, new, lengths, 64, heads, group, d)
    want, bound = K.attention_reference(host, batch, q, 0.09, window, sinks, f32_output=types == "f32")
    t = torch.float32 if types == "f32" else torch.bfloat16
    K.check_attention(_attend(ctx, host, batch, q, 0.09, window, sinks, t, t), want, bound)


def test_a_batch_without_a_bound_of_its_query_lengths(ctx):  # noqa: F811
    """Decode rows and a bound that would allow one sequence all of them; and rows behind the last sequence."""
    rng = np.random.default_rng(103)
    new, lengths = [1] * 9 + [0, 2], rng.integers(1, 2600, 11).tolist()
    batch, host, q = _case(rng, new, lengths, 64, 2, 4, 128)
    want, bound = K.attention_reference(host, batch, q, 0.09)
    q = np.concatenate([q, np.ones((5, 8, 128), np.float32)])
    qd = torch.from_numpy(q).bfloat16().cuda()
    out = torch.full_like(qd, 9.0)
    dev = batch.device(rows=batch.total + 5, max_query_length=batch.total + 5)
    ws = ctx.kv_cache_attention_workspace(host.device(), dev, 8)
    ws.fill_(255)
    ctx.kv_cache_attention_into(host.device(), dev, qd, out, 0.09, workspace=ws)
    got = out.float().cpu().numpy()
    assert (got[batch.total:] == 9).all()
    K.check_attention(got[:batch.total], want, bound)


@pytest.mark.parametrize("d,longest", [(64, 300), (128, 300), (64, 2400), (512, 300)])
def test_tiles_of_more_sequences_than_a_wave_has_lanes(ctx, d, longest):  # noqa: F811
    """90 sequences, few of them with many rows, the first and the last ones among those; rows behind the last sequence."""
    rng = np.random.default_rng(107 + d)
    new = rng.integers(0, 4, 90)
    new[[0, 5, 63, 64, 88]] = 70, 33, 90, 41, 65
    lengths = new + rng.integers(0, 60, 90)
    lengths[[5, 70]] = longest, longest - 7
    batch, host, q = _case(rng, new.tolist(), lengths.tolist(), 32, 1, 2, d)
    want, bound = K.attention_reference(host, batch, q, 0.09)
    qd = torch.from_numpy(np.concatenate([q, np.ones((3, 2, d), np.float32)])).bfloat16().cuda()
    out = torch.full_like(qd, 9.0)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    ctx.kv_cache_attention_into(host.device(), batch.device(rows=batch.total + 3), qd, out, 0.09, error=flag)
    got = out.float().cpu().numpy()
    assert (got[batch.total:] == 9).all() and flag.item() == 0
    K.check_attention(got[:batch.total], want, bound)


@pytest.mark.parametrize("indptr,lengths,most", [
    ((0, 200, 100, 300), (200, 50, 300), 300), ((-5, 100, 400, 900), (100, 300, 500), 300), ((0, 100, 200, 300), (-7, 2 ** 31 - 1, 300), 300),
    ((0, 100, 200, 300), (100, 100, 100), 40)])
@pytest.mark.parametrize("longest", [300, 9000])
def test_bad_indices_of_many_rows_stay_inside_the_tensors(ctx, indptr, lengths, most, longest):  # noqa: F811
    from ferrule_amd.provider import HipKvBatch
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = K.HostCache(30, 32, 1, 64).random(np.random.default_rng(5), 124, 128).device()
    table = torch.arange(30, dtype=torch.int32, device="cuda").view(3, 10)
    batch = HipKvBatch(i32(*indptr), i32(*lengths), table, 300, most, longest)
    guard = torch.full((304, 4, 64), 3.0, device="cuda")
    q = torch.ones((300, 4, 64), device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    ctx.kv_cache_attention_into(cache, batch, q, guard[2:302], 0.1, error=flag)
    torch.cuda.synchronize()
    assert (guard[:2] == 3).all() and (guard[302:] == 3).all() and flag.item() == 1


@pytest.mark.parametrize("broken", [False, True])
@pytest.mark.parametrize("new,length,group,d", [(270, 700, 1, 64), (100, 700, 1, 64), (50, 300, 1, 64), (270, 700, 1, 128), (100, 700, 1, 128),
                                                (50, 300, 1, 128), (100, 700, 1, 256), (50, 300, 1, 256), (50, 300, 2, 512)])
def test_every_tile_of_rows_under_a_distant_bound_of_the_lengths(ctx, new, length, group, d, broken):  # noqa: F811
    """The bound makes the tiles as large as the rows allow.  Broken: some values are NaN, what is behind the last token
    and on unused pages cannot be held in f32."""
    rng = np.random.default_rng(109 + d)
    batch, host, q = _case(rng, [new, 3], [length, 90], 64, 1, group, d)
    if broken:
        for b, j, block in ((0, length - new // 2, d // 32 - 1), (1, 89, 0)):
            code, scale = host.get(*_place(batch, b, j, 0), 1)
            scale = scale.copy()
            scale[block] = 255
            host.put(*_place(batch, b, j, 0), 1, code, scale)
        keep = K.HostCache(batch.pages, 64, 1, d, fill=0xf7)
        keep.arrays[1][:] = keep.arrays[3][:] = 254
        for b, n in ((0, length), (1, 90)):
            for j in range(n):
                for which in (0, 1):
                    keep.put(*_place(batch, b, j, 0), which, *host.get(*_place(batch, b, j, 0), which))
        host = keep
    want, bound = K.attention_reference(host, batch, q, 0.1)
    assert np.isnan(want).any() == broken
    K.check_attention(_attend(ctx, host, batch, q, 0.1, max_sequence_length=200000), want, bound)


def test_a_captured_mixed_step_follows_new_row_counts(ctx):  # noqa: F811
    """Captured with bounds; between the replays the rows move from one sequence to another, eager work in between."""
    from ferrule_amd.provider import HipArtifactOperatorContext, HipKvBatch
    rng = np.random.default_rng(113)
    rows, heads, group, d = 64, 2, 4, 128
    cache = K.HostCache(300, 64, heads, d).random(rng, 124, 128).device()
    put = lambda t, v: t.copy_(torch.tensor(v, dtype=torch.int32))  # noqa: E731
    indptr, lengths = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    table = torch.arange(300, dtype=torch.int32, device="cuda").view(3, 100)
    batch = HipKvBatch(indptr, lengths, table, rows, rows, 5000)
    q = torch.randn((rows, heads * group, d), device="cuda").bfloat16()
    out = torch.full_like(q, 9.0)
    stream = torch.cuda.Stream()
    side = HipArtifactOperatorContext(0, stream)
    ws = side.kv_cache_attention_workspace(cache, batch, heads * group)
    run = lambda who, o, **kw: who.kv_cache_attention_into(cache, batch, q, o, 0.09, **kw)  # noqa: E731
    put(indptr, [0, 62, 63, 64])
    put(lengths, [3000, 4000, 1])
    torch.cuda.synchronize()
    run(side, out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(side, out, workspace=ws)
    for starts, tokens in (([0, 62, 63, 64], [3000, 4000, 1]), ([0, 1, 2, 64], [5000, 700, 62]), ([0, 3, 40, 44], [2500, 4800, 2600]),
                           ([0, 0, 1, 1], [0, 5000, 10])):
        put(indptr, starts)
        put(lengths, tokens)
        ws.fill_(255)
        out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.full_like(q, 9.0)
        run(ctx, want)
        torch.cuda.synchronize()
        same = torch.equal(out, want) and bool((out[starts[-1]:] == 9).all()) and not bool((out[:starts[-1]] == 9).all(-1).any())
        assert same, starts


@pytest.mark.parametrize("d", [64, 128, 256])
def test_short_ranges_of_most_of_the_card(ctx, d):  # noqa: F811
    """140 segments: eight waves to each, and no second workgroup; one of the values' blocks is NaN."""
    rng = np.random.default_rng(127 + d)
    lengths = rng.integers(1, 30, 70)
    lengths[[0, 33, 69]] = 500, 290, 321
    batch, host, q = _case(rng, [1] * 70, lengths.tolist(), 32, 2, 3, d)
    code, scale = host.get(*_place(batch, 33, 100, 1), 1)
    scale = scale.copy()
    scale[d // 32 - 1] = 255
    host.put(*_place(batch, 33, 100, 1), 1, code, scale)
    for window, sinks in ((0, 0), (310, 2)):
        want, bound = K.attention_reference(host, batch, q, 0.1, window, sinks)
        assert np.isnan(want).any()
        K.check_attention(_attend(ctx, host, batch, q, 0.1, window, sinks), want, bound)
