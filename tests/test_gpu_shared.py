"""Attention behind a shared prefix (tp_shared_attention) against attention in float64 over the oracle's decode.

Error of an output element: weights, a record and the result are rounded once each (eps = 2^-11 relative, the
record's weighted by its share), sums are fp32; a key component is rounded from fp32 as the page decoder rounds it, and
differs from the oracle's by one fp16 step (2 eps) where their cosines differ in the last bit, so a score is off by ds =
scale (2 eps + 129 2^-24) sum|q||k|, a weight by exp(2 ds) - 1 (its own and the sum's).  Values are the same numbers on
both sides."""

import numpy as np
import pytest
import torch

from common import ATOL, LAYOUTS, RTOL_L2, gen_kv, rel_l2
from test_gpu_rotate import config, draw, tables
from test_gpu_tree import filled, history
from turbopolar_amd import SharedPrefixCache, TurboPolarFastCache
from turbopolar_amd.kernels import fp16_scale, rotate_tokens

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -11


def made(device, layout, B, hq, hkv, prefix, own, seed=0):
    cache = SharedPrefixCache(filled(device, layout, 1, hq, hkv, prefix, seed=seed + 1),
                              filled(device, layout, B, hq, hkv, own, seed=seed + 2))
    g = torch.Generator(device=device).manual_seed(seed + 3)
    return cache, torch.randn((B, hq, 1, 128), generator=g, device=device).half()


def expected(q, cache, scale16, keys=None):
    """The result in float64 and the bound of an element's error."""
    B, hq = q.shape[:2]
    hkv = cache.config.num_kv_heads
    parts = [history(c.runtime) if c.offset else None for c in (cache.prefix, cache.own)]
    q64 = q.double().cpu().numpy()
    want, tol = np.zeros((B, hq, 128)), np.zeros((B, hq, 128))
    for b in range(B):
        for h in range(hq):
            kv = h // (hq // hkv)
            k, v = (np.concatenate([p[i][0 if j == 0 else b, kv] for j, p in enumerate(parts) if p is not None]) for i in (0, 1))
            x = q64[b, h, 0]
            s = k @ x * scale16
            w = np.exp(s - s.max())
            w /= w.sum()
            want[b, h] = w @ v
            ds = abs(scale16) * (2 * EPS + 129 * 2.0 ** -24) * (np.abs(k) @ np.abs(x)).max()
            tol[b, h] = (w @ np.abs(v)) * (3 * EPS + np.expm1(2 * ds) + (len(s) + 16) * 2.0 ** -23)
            tol[b, h] += (len(s) + 2) * 2.0 ** -25 * np.abs(v).max()
    return want, tol


def check(got, q, cache, scale, what):
    want, tol = expected(q, cache, fp16_scale(scale))
    assert got.shape == want.shape and got.dtype is torch.float16
    got = got.double().cpu().numpy()
    off = np.abs(got - want)
    print(f"[shared] {what}: max-abs {off.max():.3g}, rel L2 {rel_l2(got, want):.3g}, {(off / tol).max():.3g} of the bound",
          flush=True)
    assert np.all(off <= tol), what
    # ATOL is for results of about 1; a larger one's rounding alone may be as much, so half a step is allowed besides.
    assert np.all(off <= ATOL + EPS * np.abs(want)) and rel_l2(got, want) <= RTOL_L2


CASES = [
    # layout, B, hq, hkv, prefix, own: one part empty; tails alone; whole pages alone; both; rows of 1 to over 256 a
    # head, own heads of more than one row block; many splits and one
    ("default", 1, 4, 1, 1, 0), ("default", 3, 8, 2, 0, 1), ("default", 2, 8, 2, 64, 0), ("default", 2, 8, 2, 0, 128),
    ("default", 4, 8, 2, 20, 5), ("default", 5, 32, 8, 1000, 50), ("default", 33, 8, 8, 130, 65), ("default", 9, 28, 4, 700, 63),
    ("default", 32, 32, 8, 2000, 70), ("default", 50, 8, 1, 333, 3), ("default", 1, 70, 1, 200, 100), ("default", 2, 300, 1, 100, 70),
    ("default", 1, 1, 1, 63, 64), ("default", 7, 40, 2, 4500, 1), ("default", 3, 8, 2, 65, 4000),
    ("fast", 1, 8, 2, 64, 64), ("fast", 16, 64, 8, 700, 40), ("fast", 3, 8, 8, 333, 129), ("fast", 40, 8, 2, 90, 200),
    ("fast", 64, 8, 1, 1000, 20), ("fast", 70, 8, 1, 64, 0), ("deep2", 3, 8, 2, 333, 70), ("deep2", 40, 8, 2, 150, 30),
    ("l1_8bit", 2, 8, 2, 333, 200), ("odd_split", 2, 8, 2, 333, 70), ("odd_split", 30, 16, 4, 200, 64), ("odd_split", 64, 8, 1, 130, 9),
    ("int8_default_angles", 5, 8, 2, 333, 70), ("int8_default_angles", 40, 16, 1, 64, 130),
]


@pytest.mark.parametrize("case", CASES)
def test_shared_against_oracle(device, case):
    print(f"[shared] {case}", flush=True)
    cache, q = made(device, *case, seed=case[4] + case[5])
    assert cache.offset == case[4] + case[5]
    check(cache.attention(q, cache.config.attention_scale), q, cache, cache.config.attention_scale, f"{case}")


@pytest.mark.parametrize("scale", [0.0, -0.09, 0.5])
def test_scales(device, scale):
    cache, q = made(device, "default", 3, 8, 2, 300, 40)
    check(cache.attention(q, scale), q, cache, scale, f"scale {scale}")


def test_a_fork_of_the_prefix_attends_the_same(device):
    """Behind a prefix and in a copy of it with the same tokens appended: the keys of whole pages differ only by
    where their pages begin, so whole prefix pages are used."""
    B, hq, hkv = 4, 8, 2
    cache, q = made(device, "default", B, hq, hkv, 320, 0)
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(5, B, hkv, 70))
    copy = cache.prefix.fork(rows=[0] * B)
    cache.append(k, v)
    copy.runtime.append(k, v)
    rows = [copy.fork(rows=[b]) for b in range(B)]
    got = cache.attention(q, 0.09)
    for b in range(B):
        want = rows[b].selected_attention(q[b:b + 1], 0.09, 100)
        # Both are within twice the bound of the decode kernel's contract of each other.
        assert (got[b] - want[0]).abs().max() <= 2 * ATOL


def test_a_serving_loop(device):
    """Prompt, branches, rotated steps, beams re-ordered, a cut back and a fork: every step against float64."""
    hq, hkv, B = 8, 2, 3
    prefix = TurboPolarFastCache(config("fast", hq, hkv))
    q, k, v = draw(device, 1, hq, hkv, 200, torch.bfloat16, 1, spread=0.5)
    prefix.update_rotated(q, k, v, *tables(device, 0, 200, 128, False, torch.float32))
    held = [t.clone() for t in (prefix.runtime.k_storage.radii, prefix.runtime.partial_k)]
    cache = SharedPrefixCache(prefix)
    scale = prefix.config.attention_scale

    def step(cache, i, B):
        q, k, v = draw(device, B, hq, hkv, 1, torch.bfloat16, 50 + i, spread=0.5)
        q16 = cache.append_rotated(q, k, v, *tables(device, cache.offset, 1, 128, False, torch.float32))
        check(cache.attention(q16, scale), q16, cache, scale, f"step {i}")

    for i in range(3):
        step(cache, i, B)
    q, k, v = draw(device, B, hq, hkv, 60, torch.bfloat16, 7, spread=0.5)
    cache.append_rotated(q, k, v, *tables(device, cache.offset, 60, 128, False, torch.float32))
    for i in range(3, 6):
        step(cache, i, B)
    cache.select_rows([2, 2, 0, 1])
    step(cache, 6, 4)
    branch = cache.fork(rows=[3, 1])
    step(branch, 7, 2)
    cache.truncate(201)
    step(cache, 8, 4)
    assert cache.offset == 202 and branch.offset == 268
    q, k, v = draw(device, 4, hq, hkv, 1, torch.float16, 77, spread=0.5)
    out = cache.decode_attention(q, k, v, scale)
    check(out, q, cache, scale, "step 9")
    assert torch.equal(held[0], prefix.runtime.k_storage.radii) and torch.equal(held[1], prefix.runtime.partial_k)


def test_refusals(device):
    cache, q = made(device, "default", 3, 8, 2, 100, 70)
    with pytest.raises(ValueError, match="batch of q"):
        cache.attention(q[:2], 0.1)
    with pytest.raises(ValueError, match="finite"):
        cache.attention(q, float("nan"))
    with pytest.raises(ValueError, match="no gradients"):
        cache.attention(q.clone().requires_grad_(), 0.1)
    with pytest.raises(ValueError, match="one HIP device"):
        cache.attention(q.cpu(), 0.1)
    before = cache.offset
    bad = torch.zeros(3, 2, 1, 128, device=device).half()
    bad[2, 1, 0, 5] = float("inf")
    with pytest.raises(ValueError, match="finite"):
        cache.decode_attention(q, bad, bad, 0.1)
    assert cache.offset == before


def test_queries_of_any_stride_and_type(device):
    cache, q = made(device, "default", 4, 8, 2, 130, 70)
    want = cache.attention(q, 0.1)
    wide = torch.zeros(4, 3, 8, 128, dtype=torch.float16, device=device)
    wide[:, 1] = q[:, :, 0]
    assert torch.equal(cache.attention(wide[:, 1:2].transpose(1, 2), 0.1), want)
    assert torch.equal(cache.attention(q.float(), 0.1), want)
    assert torch.equal(cache.attention(q, 0.1), want)  # nothing is left behind by a call


def test_streams_and_graphs(device):
    """Two streams at once, and two captured graphs replayed side by side with eager calls between."""
    one, q1 = made(device, "default", 4, 8, 2, 1500, 70, seed=1)
    two, q2 = made(device, "fast", 9, 8, 2, 700, 130, seed=2)
    want = [one.attention(q1, 0.1), two.attention(q2, 0.1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s, cache, q in zip(streams, (one, two), (q1, q2)):
        with torch.cuda.stream(s):
            got.append([cache.attention(q, 0.1) for _ in range(5)])
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)
    graphs, outs = [], []
    for cache, q in ((one, q1), (two, q2)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(cache.attention(q, 0.1))
        graphs.append(graph)
    for seed in range(3):
        g = torch.Generator(device=device).manual_seed(seed)
        for q in (q1, q2):
            q.copy_(torch.randn(q.shape, generator=g, device=device))
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], one.attention(q1, 0.1)) and torch.equal(outs[1], two.attention(q2, 0.1))


def test_layouts_are_all_covered():
    assert {c[0] for c in CASES} == set(LAYOUTS)


def test_rotated_queries_feed_attention(device):
    """What rotate_tokens returns is read in place."""
    cache, _ = made(device, "default", 2, 8, 2, 100, 5)
    q, k, v = draw(device, 2, 8, 2, 1, torch.bfloat16, 3, spread=0.5)
    cos, sin = tables(device, cache.offset, 1, 128, False, torch.bfloat16)
    want = rotate_tokens(q, k, v, cos, sin)
    q16 = cache.append_rotated(q, k, v, cos, sin)
    assert torch.equal(q16, want[0])
    check(cache.attention(q16, 0.1), q16, cache, 0.1, "rotated")


@pytest.mark.parametrize("layout", ["default", "odd_split"])
def test_own_tokens_by_a_launch_of_their_own(device, layout):
    """More tiles of own tokens than go along with the prefix's, and a prefix of more rows than four waves hold."""
    for B, hq, hkv, prefix, own in ((12, 32, 8, 70, 64 * 65), (33, 8, 1, 130, 200), (40, 16, 4, 64, 70)):
        cache, q = made(device, layout, B, hq, hkv, prefix, own, seed=B)
        check(cache.attention(q, 0.09), q, cache, 0.09, f"{layout} {B} {hq} {hkv} {prefix} {own}")


def test_a_refused_step_leaves_the_sequences(device):
    cache, q = made(device, "default", 3, 8, 2, 100, 70)
    new = torch.ones(3, 2, 1, 128, device=device).half()
    for args in ((q[:, :7], new, new, 0.1), (q, new, new, float("inf")), (q.clone().requires_grad_(), new, new, 0.1),
                 (q.cpu(), new, new, 0.1), (q[..., :64], new, new, 0.1), (q.long(), new, new, 0.1)):
        with pytest.raises(ValueError):
            cache.decode_attention(*args)
        assert cache.offset == 170
    with pytest.raises(ValueError):  # the first step's batch too
        SharedPrefixCache(cache.prefix).decode_attention(q[:, :7], new, new, 0.1)
    with pytest.raises(ValueError, match="one HIP device"):
        SharedPrefixCache(cache.prefix).decode_attention(q, new.cpu(), new.cpu(), 0.1)
    assert cache.decode_attention(q, new, new, 0.1).shape == (3, 8, 128) and cache.offset == 171


def test_float32_caches(device):
    """Tokens appended in float32 stay so in the dense tail: attended as their rounding to fp16, which these are."""
    cache, q = made(device, "default", 3, 8, 2, 100, 70, seed=4)
    wide = SharedPrefixCache(TurboPolarFastCache(cache.config), TurboPolarFastCache(cache.config))
    for seed, c, B, T in ((5, wide.prefix, 1, 100), (6, wide.own, 3, 70)):
        k, v = (torch.from_numpy(t).to(device) for t in gen_kv(seed, B, 2, T))
        assert torch.equal(k.half().float(), k.float())
        c.runtime.append(k.float(), v.float())
    wide = SharedPrefixCache(wide.prefix, wide.own)  # counts the prefix's tokens
    assert wide.own.runtime._tail_k.dtype is torch.float32
    check(wide.attention(q, 0.1), q, wide, 0.1, "float32")


def test_a_large_batch(device):
    """More (sequence, head) rows than a workgroup takes, many times over."""
    case = ("default", 700, 8, 2, 70, 3)
    cache, q = made(device, *case, seed=8)
    check(cache.attention(q, 0.1), q, cache, 0.1, f"{case}")


def test_compacted_prefixes_are_refused(device):
    """Pages in another order, or others, are another prefix of the same length; the same ones in place are not."""
    cache, q = made(device, "default", 2, 8, 2, 64 * 3 + 9, 5)
    want = cache.attention(q, 0.1)
    cache.prefix.keep_pages([0, 1, 2])
    assert torch.equal(cache.attention(q, 0.1), want)
    cache.prefix.keep_pages(torch.tensor([0, 2, 1]))
    assert cache.prefix.offset == cache.prefix_tokens
    with pytest.raises(ValueError, match="tokens are others"):
        cache.attention(q, 0.1)
    # What an append that is refused later leaves is what was there.
    cache, q = made(device, "default", 2, 8, 2, 64 * 3 + 9, 5)
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(3, 1, 2, 1))
    bad = torch.full_like(k, float("nan"))
    cache.prefix.runtime.append(bad, v, defer_check=True)
    with pytest.raises(ValueError, match="finite"):
        cache.prefix.runtime.resolve_deferred_check()
    assert torch.equal(cache.attention(q, 0.1), want)
    # Cut inside of its pages and filled again, and only a few of its pages shared.
    cache.prefix.truncate(64 * 2 + 3)
    cache.prefix.runtime.append(*(t.expand(-1, -1, 70, -1) for t in (k, v)))
    with pytest.raises(ValueError, match="tokens are others"):
        cache.attention(q, 0.1)
