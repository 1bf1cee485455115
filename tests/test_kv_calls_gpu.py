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
