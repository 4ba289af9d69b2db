"""Buffers of more than 4 GiB: what lies past 32 bits of bytes, or of elements, is read and written where it is."""

import pytest
import torch

from common import gen_kv
from test_gpu_rotate import tables
from test_gpu_tree import filled
from turbopolar_amd import SharedPrefixCache
from turbopolar_amd.kernels import rotate_tokens

pytestmark = pytest.mark.gpu
FAR_PAGES = 80000  # the last of 8 heads begins 7 capacities of at least 80,000 pages of 8 KB, 4.5 GB, into its buffer


def far(cache):
    """The same cache in buffers of a large capacity."""
    rt = cache.runtime
    B, H, dev = rt._batch_size, rt._num_kv_heads, rt._tail_k.device
    rt.k_storage.reserve(FAR_PAGES, rt.polar_encoder, B, H, dev)
    rt.v_storage.reserve(FAR_PAGES, B, H, dev)
    assert rt.v_storage.codes[0, -1, 0].storage_offset() > 2 ** 32
    return cache


@pytest.mark.parametrize("layout", ["default", "fast"])
def test_far_pages(device, layout):
    near = filled(device, layout, 1, 8, 8, 64 * 30 + 9, seed=1)
    cache = far(near.fork())
    g = torch.Generator(device=device).manual_seed(1)
    q = torch.randn((1, 8, 1, 128), generator=g, device=device).half()
    assert torch.equal(cache.runtime.page_bounds(), near.runtime.page_bounds())
    assert torch.equal(cache.selected_attention(q, 0.1, 7), near.selected_attention(q, 0.1, 7))
    # As the prefix, and as the sequences' own cache.
    qs = torch.randn((3, 8, 1, 128), generator=g, device=device).half()
    want = SharedPrefixCache(near, None)
    got = SharedPrefixCache(cache, None)
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(5, 3, 8, 70))
    want.append(k, v), got.append(k, v)
    assert torch.equal(got.attention(qs, 0.1), want.attention(qs, 0.1))
    prefix = filled(device, layout, 1, 8, 8, 100, seed=2)
    assert torch.equal(SharedPrefixCache(prefix, cache).attention(q, 0.1), SharedPrefixCache(prefix, near).attention(q, 0.1))


def test_far_rotated_tokens(device):
    """2^31 query elements and more; the last tokens are what they are alone."""
    T, hq = 2 ** 19 + 70, 32
    q = torch.empty((1, T, hq, 128), dtype=torch.float16, device=device)
    for t in range(0, T, 2 ** 16):
        q[:, t:t + 2 ** 16].normal_()
    assert q.numel() > 2 ** 31
    q = q.transpose(1, 2)
    k, v = (torch.randn((1, 1, T, 128), dtype=torch.float16, device=device) for _ in range(2))
    cos, sin = tables(device, 0, T, 64, False, torch.float32)
    got = rotate_tokens(q, k, v, cos, sin)
    for a, b in ((0, 40), (2 ** 18 - 3, 2 ** 18 + 3), (2 ** 19 - 20, T)):
        want = rotate_tokens(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], cos[a:b], sin[a:b])
        assert all(torch.equal(x[:, :, a:b], y) for x, y in zip(got, want))


def test_more_rotated_tokens_than_a_grid_holds(device):
    """2^24 tokens and more, a workgroup each, every row of the batch the same one in memory."""
    B, T = 4099, 4097
    assert B * T > 2 ** 24
    q, k, v = (torch.randn((1, 1, T, 128), dtype=torch.float16, device=device) for _ in range(3))
    cos, sin = tables(device, 0, T, 64, False, torch.float32)
    want = rotate_tokens(q, k, v, cos, sin)
    got = rotate_tokens(*(t.expand(B, -1, -1, -1) for t in (q, k, v)), cos, sin)
    for x, y in zip(got, want):
        assert x.shape[0] == B
        for b in range(0, B, 512):
            assert torch.equal(x[b:b + 512], y.expand(min(512, B - b), -1, -1, -1)), b
