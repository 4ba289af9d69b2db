"""Page bounds, the pages that scores select and attention over them, against float64.

Scores are float64 sums of 128 exact products, off by 127 2^-53 of the sum of their sizes on either side, so the
selection has to be the definition's wherever the last page taken and the first one left differ by more than that
(asserted for the inputs used).  Attention's error as in test_gpu_attention: max-abs 2e-3 (for
results of about 1) and relative L2 1e-3."""

import numpy as np
import pytest
import torch

import oracle
from common import ATOL, LAYOUTS, PAGE, RTOL_L2, gen_kv, rel_l2, within_f16_ulp
from test_gpu_rotate import draw, tables
from test_gpu_tree import filled, pages64
from turbopolar_amd import HipKernelBridge, TurboPolarConfig, TurboPolarFastCache, _lib
from turbopolar_amd.kernels import fp16_scale, selected_attention, tail_args

pytestmark = pytest.mark.gpu


def queries(device, B, hq, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn((B, hq, 128), generator=g, device=device).half()


def scores64(q, bounds, sign=1):
    """[B, hkv, pages] in float64 and the bound of a score's error."""
    B, hq, _ = q.shape
    hkv = bounds.shape[1]
    x = sign * q.double().cpu().numpy().reshape(B, hkv, hq // hkv, 1, 128)
    b = bounds.double().cpu().numpy()
    lo, hi = b[:, :, None, :, 0], b[:, :, None, :, 1]
    with np.errstate(invalid="ignore"):
        terms = np.fmax(x * lo, x * hi)
        s = terms.sum(-1)
    s = np.where(np.isnan(s), np.inf, s)
    return s.max(2), 2.0 ** -45 * np.abs(terms).sum(-1).max(2)


def chosen64(scores, n, first, last):
    B, H, S = scores.shape
    out = np.empty((B, H, n), np.int32)
    for b in range(B):
        for h in range(H):
            forced = [i < first or i >= S - last for i in range(S)]
            out[b, h] = sorted(sorted(range(S), key=lambda i: (not forced[i], -scores[b, h, i], i))[:n])
    return out


def bridge_call(cache, q, bounds, n, first, last):
    key, value, tail_k, tail_v, _, _ = cache.runtime.get_fused_attention_inputs()
    out, trace = HipKernelBridge().execute_selected_attention_quant_v_dense_tail(
        q, key, value, bounds, tail_k, tail_v, cache.config, pages=n, first=first, last=last)
    return out, trace["selected"]


def attended(q, cache, selected, scale16):
    """Attention over the selected pages and the tail, float64."""
    B, hq, _ = q.shape
    k64, v64 = pages64(cache.runtime)
    hkv, g = k64.shape[1], hq // k64.shape[1]
    rt = cache.runtime
    tail = [t.double().cpu().numpy() for t in (rt.partial_k, rt.partial_v)] if rt._tail_len else None
    x = q.double().cpu().numpy()
    out = np.empty(x.shape)
    for b in range(B):
        for h in range(hq):
            kv = h // g
            at = (np.asarray(selected[b, kv])[:, None] * PAGE + np.arange(PAGE)).ravel()
            k, v = k64[b, kv, at], v64[b, kv, at]
            if tail:
                k, v = np.concatenate((k, tail[0][b, kv])), np.concatenate((v, tail[1][b, kv]))
            s = k @ x[b, h] * scale16
            p = np.exp(s - s.max())
            out[b, h] = p @ v / p.sum()
    return out


def close(got, want, what):
    got = got.double().cpu().numpy()
    off = np.abs(got - want)
    print(f"[select] {what}: max-abs {off.max():.3g}, rel L2 {rel_l2(got, want):.3g}", flush=True)
    assert np.all(off <= ATOL + 2.0 ** -11 * np.abs(want)) and rel_l2(got, want) <= RTOL_L2, what


def near(bounds, keys):
    for i, x in enumerate((keys.amin(3), keys.amax(3))):
        assert within_f16_ulp(bounds[:, :, :, i].cpu().numpy(), x.cpu().numpy())


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_bounds(device, layout):
    """Of the oracle's keys and of the page decoder's, within a step of fp16 of each: all round the same r cos a, r sin a,
    the oracle with its own cosines (an fp32 step apart), the decoder without the rounding to fp32 between, so each is
    within half a step and 2^-22 of itself of that product, and two such numbers are at most neighbours; so are the
    smallest, and the largest, of such numbers."""
    for B, hkv, S in ((1, 1, 1), (2, 3, 5), (1, 8, 40)):
        cache = filled(device, layout, B, hkv, hkv, S * PAGE, seed=S)
        key = cache.runtime.get_fused_attention_inputs()[0]
        got, trace = HipKernelBridge().execute_page_bounds(key)
        assert got.shape == (B, hkv, S, 2, 128) and got.dtype is torch.float16 and trace["pages"] == S
        keys = cache.runtime.fetch_blocks().view(B, hkv, S, PAGE, 128)
        near(got, keys)
        k64 = pages64(cache.runtime)[0].reshape(B, hkv, S, PAGE, 128)
        assert within_f16_ulp(got[:, :, :, 0].cpu().numpy(), k64.min(3)) and within_f16_ulp(got[:, :, :, 1].cpu().numpy(), k64.max(3))
        assert torch.equal(cache.runtime.page_bounds(), got)


CASES = [
    # layout, B, hq, hkv, tokens, pages, first, last: every page, one page, forced pages alone, none forced; a tail and
    # none; more heads a group than one turn takes; more pages than threads; counts around the splits of attention
    ("default", 1, 8, 2, 64, 1, 0, 0), ("default", 1, 8, 2, 64, 1, 1, 0), ("default", 1, 8, 2, 200, 2, 1, 1),
    ("default", 1, 8, 2, 200, 3, 0, 0), ("default", 2, 8, 2, 640, 1, 0, 0), ("default", 2, 8, 2, 640, 4, 2, 2),
    ("default", 2, 8, 2, 700, 5, 0, 1), ("default", 1, 32, 8, 5000, 20, 1, 2), ("default", 1, 40, 2, 1500, 9, 1, 1),
    ("default", 1, 64, 1, 1500, 9, 1, 1), ("default", 1, 300, 1, 700, 5, 0, 2), ("default", 1, 4, 1, 64 * 1100 + 3, 33, 1, 1),
    ("default", 4, 28, 4, 1100, 16, 1, 1), ("default", 33, 8, 8, 400, 3, 1, 1), ("default", 1, 8, 8, 9000, 100, 1, 4),
    ("default", 1, 4, 1, 64 * 300, 270, 1, 1),
    ("fast", 1, 8, 2, 640, 4, 1, 1), ("fast", 2, 64, 8, 2000, 30, 0, 1), ("fast", 1, 8, 1, 4500, 65, 1, 1),
    ("deep2", 2, 8, 2, 700, 5, 1, 1), ("l1_8bit", 1, 8, 2, 700, 5, 1, 1), ("odd_split", 3, 8, 2, 700, 6, 1, 1),
    ("int8_default_angles", 1, 24, 2, 700, 6, 1, 1),
]


@pytest.mark.parametrize("case", CASES)
def test_selection_and_attention(device, case):
    layout, B, hq, hkv, tokens, n, first, last = case
    print(f"[select] {case}", flush=True)
    cache = filled(device, layout, B, hq, hkv, tokens, seed=tokens + n)
    q = queries(device, B, hq, n)
    bounds = cache.runtime.page_bounds()
    scores, slack = scores64(q, bounds)
    want = chosen64(scores, n, first, last)
    for b in range(B):  # the inputs tell the last page taken from the first one left
        for h in range(hkv):
            middle = range(first, tokens // PAGE - last)
            left = [i for i in middle if i not in want[b, h]]
            taken = [i for i in middle if i in want[b, h]]
            if left and taken:
                assert min(scores[b, h, taken]) - max(scores[b, h, left]) > slack[b, h].max()
    got, selected = bridge_call(cache, q, bounds, n, first, last)
    assert selected.dtype is torch.int32 and np.array_equal(selected.cpu().numpy(), want)
    scale = fp16_scale(cache.config.attention_scale)
    close(got, attended(q, cache, want, scale), f"{case}")
    through = cache.selected_attention(q[:, :, None], cache.config.attention_scale, n, first, last)
    if n < tokens // PAGE:
        assert torch.equal(through, got)
    else:  # every page: the decode step's own kernel
        close(through, attended(q, cache, want, scale), "whole cache")


def test_ties_take_the_lower_index(device):
    """Equal pages, equal scores of both signs and zeros of both signs."""
    cache = TurboPolarFastCache(TurboPolarConfig(num_q_heads=2, num_kv_heads=1))
    page, v = (torch.from_numpy(t).to(device) for t in gen_kv(1, 1, 1, PAGE))
    S = 40
    cache.runtime.append(page.repeat(1, 1, S, 1), v.repeat(1, 1, S, 1))
    q = queries(device, 1, 2, 1)
    bounds = cache.runtime.page_bounds().clone()
    for n, first, last in ((7, 0, 0), (7, 1, 2), (39, 0, 0), (40, 0, 0)):
        got = bridge_call(cache, q, bounds, n, first, last)[1]
        assert got.flatten().tolist() == sorted(list(range(n - last)) + list(range(S - last, S)))
    bounds[:, :, [3, 9, 11]] = 0.0
    bounds[:, :, 5:8] = -0.0
    bounds[:, :, [20, 30]] *= 2
    scores = scores64(q, bounds)[0]
    for n in (1, 2, 3, 20, 36, 38):
        got = bridge_call(cache, q, bounds, n, 0, 0)[1]
        assert np.array_equal(got.cpu().numpy(), chosen64(scores, n, 0, 0)), n
    bounds.zero_()
    assert bridge_call(cache, q, bounds, 9, 0, 0)[1].flatten().tolist() == list(range(9))


def test_many_equal_scores_among_others(device):
    """Few distinct scores over more pages than a workgroup has threads, in every digit of the keys."""
    cache = filled(device, "default", 1, 2, 2, 64 * 3000, seed=3)
    g = torch.Generator(device=device).manual_seed(1)
    q = torch.zeros((1, 2, 128), device=device).half()
    q[..., 0] = 1.0
    bounds = torch.zeros((1, 2, 3000, 2, 128), device=device).half()
    for values in ([1.0, 1.0009765625, 2.0], [-1.0, 0.0, 1.0], [6e-8, 65504.0, -65504.0, 1.2e-7], [3.0]):
        pick = torch.tensor(values, device=device).half()[torch.randint(len(values), (1, 2, 3000), generator=g, device=device)]
        bounds[..., 0] = pick[..., None]
        scores = scores64(q, bounds)[0]
        for n in (1, 999, 1000, 1024, 1025, 2500, 2999):
            got = bridge_call(cache, q, bounds, n, 0, 0)[1]
            assert np.array_equal(got.cpu().numpy(), chosen64(scores, n, 0, 0)), (values, n)


@pytest.mark.parametrize("S", [1, 64, 65, 511, 512, 513, 2047, 2048, 2049, 4096, 4097, 8191, 8192, 8193, 9001])
def test_any_number_of_pages(device, S):
    """The entry point alone, around the numbers of pages at which the kernel takes another form, and one call right
    behind another in one workspace."""
    B, hq, hkv = 2, 6, 2
    g = torch.Generator(device=device).manual_seed(S)
    bounds = torch.randn((B, hkv, S, 2, 128), generator=g, device=device).sort(dim=3).values.half().contiguous()
    q = queries(device, B, hq, S)
    scores, err = scores64(q, bounds)
    L = _lib.lib()
    ws = torch.zeros(int(L.tp_select_workspace_bytes(B, hq, hkv, S)), dtype=torch.uint8, device=device)
    asked = [(min(S, n), min(f, S), min(la, S - min(f, S))) for n, f, la in ((1, 0, 0), (33, 1, 2), (S // 3 + 3, 2, 1), (S, 0, 1))]
    outs = []
    for n, first, last in asked:
        outs.append(torch.full((B, hkv, n), -1, dtype=torch.int32, device=device))
        st = L.tp_select_pages(q.data_ptr(), B, hq, hkv, bounds.data_ptr(), S, S, first, min(last, n - first), n, 0.1,
                               outs[-1].data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert st == 0
    for (n, first, last), got in zip(asked, outs):
        last = min(last, n - first)
        between = np.sort(scores[:, :, first:S - last], axis=-1)[..., ::-1]
        take = n - first - last
        if 0 < take < between.shape[-1]:  # no score within rounding of the border: as the input was drawn
            assert np.all(between[..., take - 1] - between[..., take] > 2 * err.max())
        assert np.array_equal(got.cpu().numpy(), chosen64(scores, n, first, last)), (n, first, last)


def test_negative_scales_and_bounds_that_are_not_finite(device):
    cache = filled(device, "default", 1, 8, 2, 64 * 30 + 5, seed=2)
    q = queries(device, 1, 8, 4)
    bounds = cache.runtime.page_bounds()
    rt, lay = cache.runtime, cache.runtime.polar_encoder.layout
    tail = tail_args(rt._tail_k, rt._tail_v, rt._tail_len)
    out, selected = selected_attention(q, lay, cache._store_pages(), 30, 2, bounds, int(rt._bounds.shape[2]), tail, -0.1, 6,
                                       1, 1)
    want = chosen64(scores64(q, bounds, -1)[0], 6, 1, 1)
    assert np.array_equal(selected.cpu().numpy(), want)
    close(out, attended(q, cache, want, np.float64(np.float32(-0.1))), "negative scale")
    odd = bounds.clone()
    odd[0, 0, 7, 1, 3] = float("inf")
    odd[0, 0, 9, 0, 3] = odd[0, 0, 9, 1, 3] = float("nan")
    odd[0, 1, 11, 0, 5], odd[0, 1, 11, 1, 5] = float("-inf"), float("inf")
    odd[0, 1, 13] = float("nan")
    scores = scores64(q, odd)[0]
    got = bridge_call(cache, q, odd, 6, 0, 0)[1]
    assert np.array_equal(got.cpu().numpy(), chosen64(scores, 6, 0, 0))


def test_bounds_follow_the_cache(device):
    """Appends, cuts inside and between pages, re-ordered rows, kept pages, forks, resets and undone appends."""
    cache = TurboPolarFastCache(TurboPolarConfig(num_q_heads=4, num_kv_heads=2))

    def add(T, seed):
        k, v = gen_kv(seed, cache.runtime._batch_size or 3, 2, T)
        cache.runtime.append(torch.from_numpy(k).to(device), torch.from_numpy(v).to(device))

    def check(c=cache):
        got = c.runtime.page_bounds()
        keys = c.runtime.fetch_blocks()
        keys = keys.view(*keys.shape[:2], -1, PAGE, 128)
        near(got, keys)
        # And what a page's bounds are does not depend on when they were taken.
        assert torch.equal(got, HipKernelBridge().execute_page_bounds(c.runtime.get_fused_attention_inputs()[0])[0])

    add(100, 1); check(); add(300, 2); check(); add(64, 3); check()  # noqa: E702
    cache.truncate(200); check(); add(70, 4); check()  # noqa: E702
    cache.truncate(128); add(200, 5); check()  # noqa: E702
    cache.select_rows([2, 0, 0, 1]); check(); add(64, 6); check()  # noqa: E702
    branch = cache.fork(); check(branch); cache.keep_pages([3, 0, 1]); check(); add(65, 7); check(); check(branch)  # noqa: E702
    cache.truncate(0)
    with pytest.raises(ValueError, match="no pages"):
        cache.runtime.page_bounds()
    add(130, 8); check()  # noqa: E702
    cache.runtime.reset()
    add(70, 9); check()  # noqa: E702
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(10, 3, 2, 1))
    bad = k.clone()
    bad[0, 0, 0, 0] = float("nan")
    while cache.runtime._tail_len < PAGE - 1:
        cache.runtime.append(k, v, defer_check=True)
    cache.runtime.append(bad, v, defer_check=True)  # completes a page
    with pytest.raises(ValueError, match="finite"):
        cache.runtime.page_bounds()
    check(); add(64, 11); check()  # noqa: E702


def test_a_serving_loop(device):
    """A rotated prompt, then rotated steps that attend part of the cache, across page ends."""
    cache = TurboPolarFastCache(TurboPolarConfig(num_q_heads=8, num_kv_heads=2, use_int8_radii=True, k_angle_bits_deep=8,
                                                 split_dim=0))
    B, scale = 2, cache.config.attention_scale
    q, k, v = draw(device, B, 8, 2, 64 * 9 + 60, torch.bfloat16, 1, spread=0.5)
    cache.append_rotated(q, k, v, *tables(device, 0, q.shape[2], 128, False, torch.float32))
    for i in range(8):
        q, k, v = draw(device, B, 8, 2, 1, torch.bfloat16, 20 + i, spread=0.5)
        q16 = cache.append_rotated(q, k, v, *tables(device, cache.offset, 1, 128, False, torch.float32))
        got = cache.selected_attention(q16, scale, 4, first=1, last=1)
        S = cache.runtime.k_storage.block_count
        assert S == (9 if i < 3 else 10)
        want = chosen64(scores64(q16[:, :, 0], cache.runtime.page_bounds())[0], 4, 1, 1)
        close(got, attended(q16[:, :, 0], cache, want, fp16_scale(scale)), f"step {i}")


def test_repeated_and_unowned_bounds(device):
    """Bounds with rows apart and a strided view give the same; results do not depend on what ran before."""
    cache = filled(device, "default", 2, 8, 2, 64 * 20 + 9, seed=1)
    q = queries(device, 2, 8, 1)
    bounds = cache.runtime.page_bounds()
    want = bridge_call(cache, q, bounds, 5, 1, 1)
    wide = torch.zeros((2, 2, 20, 2, 256), dtype=torch.float16, device=device)
    wide[..., ::2] = bounds
    for b in (bounds.contiguous(), wide[..., ::2], bounds.clone()):
        for _ in range(3):
            got = bridge_call(cache, q, b, 5, 1, 1)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(device):
    cache = filled(device, "default", 2, 8, 2, 64 * 20 + 9, seed=1)
    q = queries(device, 2, 8, 1)
    bounds = cache.runtime.page_bounds()
    for bad in (bounds[:, :, :19], bounds.float(), bounds[:1], None, bounds.cpu()):
        with pytest.raises(ValueError, match="bounds"):
            bridge_call(cache, q, bad, 5, 1, 1)
    with pytest.raises(ValueError, match="does not match"):
        bridge_call(cache, q[:1], bounds, 5, 1, 1)
    with pytest.raises(ValueError, match="does not match"):
        bridge_call(cache, q[:, :7], bounds, 5, 1, 1)
    with pytest.raises(ValueError, match="cannot select"):
        bridge_call(cache, q, bounds, 5, 3, 3)
    with pytest.raises(ValueError, match="no gradients"):
        bridge_call(cache, q.clone().requires_grad_(), bounds, 5, 1, 1)
    with pytest.raises(ValueError, match="finite"):
        cache.selected_attention(q[:, :, None], float("inf"), 5)
    out, selected = bridge_call(cache, q, bounds, 25, 3, 3)
    assert selected.shape[-1] == 20


def test_streams_and_graphs(device):
    """Two streams at once, and two captured graphs replayed side by side with eager calls between."""
    caches = [filled(device, "default", 2, 8, 2, 64 * 70 + 9, seed=1), filled(device, "fast", 1, 32, 8, 64 * 50, seed=2)]
    qs = [queries(device, 2, 8, 1)[:, :, None], queries(device, 1, 32, 2)[:, :, None]]
    call = lambda i: caches[i].selected_attention(qs[i], 0.1, 20, 1, 2)  # noqa: E731
    want = [call(0), call(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(x, want[i]) for x in got[i])
    graphs, outs = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(i))
        graphs.append(graph)
    for seed in range(3):
        for i in (0, 1):
            qs[i].copy_(queries(device, qs[i].shape[0], qs[i].shape[1], 10 + seed)[:, :, None])
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(outs[i], call(i))
    # Pages stored since the last call have no bounds yet: not inside a capture.
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(3, 1, 8, PAGE))
    caches[1].runtime.append(k, v)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured graph"):
        with torch.cuda.graph(graph):
            call(1)
    torch.cuda.synchronize()
    assert call(1).shape == (1, 32, 128)


def test_bounds_taken_on_another_stream(device):
    """A call on one stream takes the bounds of all pages behind other work; one on a second stream, right after it,
    waits for them."""
    cache = filled(device, "default", 2, 8, 2, 64 * 300 + 9, seed=1)
    twin = cache.fork()
    q = queries(device, 2, 8, 1)[:, :, None]
    want = twin.selected_attention(q, 0.1, 20, 1, 2)
    x = torch.randn(4096, 4096, device=device)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    with torch.cuda.stream(streams[0]):
        for _ in range(20):
            x = x @ x * 1e-3
        outs.append(cache.selected_attention(q, 0.1, 20, 1, 2))
    with torch.cuda.stream(streams[1]):
        outs.append(cache.selected_attention(q, 0.1, 20, 1, 2))
    torch.cuda.synchronize()
    # Grown and extended on the second stream, read on the first and on the default one.
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(3, 2, 2, 64 * 400))
    cache.runtime.append(k, v), twin.runtime.append(k, v)
    later = twin.selected_attention(q, 0.1, 20, 1, 2)
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[1]):
        for _ in range(20):
            x = x @ x * 1e-3
        outs.append(cache.selected_attention(q, 0.1, 20, 1, 2))
    with torch.cuda.stream(streams[0]):
        outs.append(cache.selected_attention(q, 0.1, 20, 1, 2))
    outs.append(cache.selected_attention(q, 0.1, 20, 1, 2))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs[:2]) and all(torch.equal(o, later) for o in outs[2:])


def test_graphs_of_whole_caches(device):
    """Caches of no more pages than a call takes are attended whole; two graphs of such calls share no workspace."""
    caches = [filled(device, "default", 2, 8, 2, 64 * 200 + 9, seed=1), filled(device, "fast", 1, 32, 8, 64 * 150, seed=2)]
    qs = [queries(device, 2, 8, 1)[:, :, None], queries(device, 1, 32, 2)[:, :, None]]
    call = lambda i: caches[i].selected_attention(qs[i], 0.1, 500, 1, 2)  # noqa: E731
    for i in (0, 1):
        call(i)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([call(i) for _ in range(4)])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in range(4):
        for i in (0, 1):
            qs[i].copy_(queries(device, qs[i].shape[0], qs[i].shape[1], 10 + seed)[:, :, None])
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            want = call(i)
            assert all(torch.equal(o, want) for o in outs[i])


def test_float32_caches(device):
    """Tokens appended in float32 stay so in the dense tail: attended as their rounding to fp16, which these are."""
    cache = TurboPolarFastCache(TurboPolarConfig(num_q_heads=8, num_kv_heads=2))
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(3, 2, 2, 64 * 20 + 33))
    cache.runtime.append(k.float(), v.float())
    assert cache.runtime._tail_k.dtype is torch.float32 and torch.equal(k.half().float(), k.float())
    q = queries(device, 2, 8, 4)
    scale = cache.config.attention_scale
    want = chosen64(scores64(q, cache.runtime.page_bounds())[0], 6, 1, 1)
    close(cache.selected_attention(q[:, :, None], scale, 6), attended(q, cache, want, fp16_scale(scale)), "float32")


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("hq", [8, 40])
def test_values_past_the_largest_fp16_number(device, layout, hq):
    """A value of 65504 is stored as 127 times 516, which fp16 holds as infinity: attended as what it is decoded to,
    here as by the decode step's own kernel."""
    k, v = gen_kv(5, 1, 2, PAGE * 8)
    v[0, 0, 70, 3], v[0, 1, 200, 90] = 65504, -65504
    cache = TurboPolarFastCache(filled(device, layout, 1, hq, 2, 0).config)
    cache.runtime.append(torch.from_numpy(k).to(device), torch.from_numpy(v).to(device))
    _, v64 = pages64(cache.runtime)
    assert np.isposinf(v64[0, 0, 70, 3]) and np.isneginf(v64[0, 1, 200, 90])
    q = queries(device, 1, hq, 4)
    got, selected = bridge_call(cache, q, cache.runtime.page_bounds(), 7, 5, 1)
    want = attended(q, cache, selected.cpu().numpy(), fp16_scale(cache.config.attention_scale))
    got = got.double().cpu().numpy()
    assert np.isinf(want).any() and not np.isnan(want).any()
    finite = np.isfinite(want)
    assert np.array_equal(got[~finite], want[~finite])
    # The rest of the dimensions of those tokens' groups are of the coarse scale, and rounded as any other.
    assert np.all(np.abs(got - want)[finite] <= ATOL + 2.0 ** -11 * np.abs(want[finite]))


def test_oracle_layouts_are_all_covered():
    assert {c[0] for c in CASES} == set(LAYOUTS) and oracle is not None
