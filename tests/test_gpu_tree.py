"""Attention of drafted trees over a compressed cache (tp_tree_attention), and cache branches (fork,
truncate, accept, select_rows, keep_pages) against the oracle's decode of the stored pages.

Error of an output element against attention in float64 over the oracle's fp16 keys and values: as
for the prompt kernel (weights and result rounded once each, eps = 2^-11, and fp32 sums), and the
keys: the kernel rounds the cosine, an int8 layout's radius and their product, the oracle the
product, so a key component differs by at most 4 eps of itself (and r 2^-23 for subnormal cosines
and the fp32 angle), a score by ds = scale (4 eps + 129 2^-24) sum|q||k| + scale 2^-23 sum|q| r, a
weight by exp(2 ds) - 1 (its own and the sum's).  Values are the same numbers on both sides.

The key's part is more than is needed since the kernel rounds the product alone, as the oracle does;
test_keys_are_the_page_decoders holds it to that."""

import numpy as np
import pytest
import torch

import oracle
from common import ATOL, LAYOUTS, PAGE, RTOL_L2, gen_kv, rel_l2
from turbopolar_amd import DraftTree, HipKernelBridge, TurboPolarConfig, TurboPolarFastCache, wire
from turbopolar_amd.kernels import fp16_scale, prompt_attention

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -11


def config(layout, hq, hkv):
    int8, l1, deep, split = LAYOUTS[layout]
    return TurboPolarConfig(num_q_heads=hq, num_kv_heads=hkv, use_int8_radii=int8, k_angle_bits_level1=l1,
                            k_angle_bits_deep=deep, split_dim=split)


def filled(device, layout, B, hq, hkv, tokens, seed=0, dtype=np.float16, kind="loguniform"):
    cache = TurboPolarFastCache(config(layout, hq, hkv))
    if tokens:
        k, v = gen_kv(seed, B, hkv, tokens, kind, dtype)
        cache.runtime.append(torch.from_numpy(k).to(device), torch.from_numpy(v).to(device))
    return cache


def pages64(rt):
    """The stored pages as the oracle decodes them, float64 on the host."""
    key, value, *_ = rt.get_fused_attention_inputs()
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    k = oracle.decode_block(host(key.radii), host(key.radii_scales), host(key.angle_codes_l1),
                            host(key.angle_codes_deep), key.metadata)
    v = oracle.dequantize_block(host(value.codes), host(value.scales))
    return k.astype(np.float64), v.reshape(k.shape).astype(np.float64)


def history(rt):
    """Every token held, ``[B, H, T, 128]`` in float64 on the host."""
    parts = [pages64(rt)] if rt.k_storage.block_count else []
    if rt._tail_len:
        parts.append((rt.partial_k.double().cpu().numpy(), rt.partial_v.double().cpu().numpy()))
    return tuple(np.concatenate([p[i] for p in parts], axis=2) for i in (0, 1))


def draft(device, B, hq, hkv, n, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    draw = lambda h: torch.randn((B, h, n, 128), generator=g, device=device).half()  # noqa: E731
    return draw(hq), draw(hkv), draw(hkv)


def random_parents(n, seed):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(-1, i - 5), i)) for i in range(1, n)]


def check(got, q, dk, dv, tree, held, scale16, what):
    B, hq, n, _ = q.shape
    hkv = dk.shape[1]
    q64, k64, v64 = (t.double().cpu().numpy() for t in (q, dk, dv))
    got = got.double().cpu().numpy()
    want = np.zeros(got.shape)
    for b in range(B):
        parents = tree.parents[0 if tree.shared else b]
        for i in range(n):
            if i >= len(parents):
                assert not got[b, :, i].any()
                continue
            path = tree.path_to(i, 0 if tree.shared else b)
            for h in range(hq):
                kv = h // (hq // hkv)
                k = np.concatenate(([held[0][b, kv]] if held else []) + [k64[b, kv, path]])
                v = np.concatenate(([held[1][b, kv]] if held else []) + [v64[b, kv, path]])
                s = k @ q64[b, h, i] * scale16
                p = np.exp(s - s.max())
                p /= p.sum()
                want[b, h, i] = p @ v
                qa, r = np.abs(q64[b, h, i]), np.sqrt(k[:, 0::2] ** 2 + k[:, 1::2] ** 2).max()
                ds = scale16 * ((4 * EPS + 129 * 2.0 ** -24) * (np.abs(k) @ qa).max() + 2.0 ** -23 * qa.sum() * r)
                tol = (p @ np.abs(v)) * (2 * EPS + np.expm1(2 * ds) + (len(s) + 16) * 2.0 ** -23)
                tol += (len(s) + 1) * 2.0 ** -25 * np.abs(v).max()
                assert np.all(np.abs(got[b, h, i] - want[b, h, i]) <= tol), (what, b, h, i)
    off = np.abs(got - want).max()
    print(f"[tree] {what}: max-abs {off:.3g}, rel L2 {rel_l2(got, want):.3g}", flush=True)
    # ATOL is the tolerance for results of about 1.  A larger result's rounding alone is up to 2^-11 of
    # it (2^-10, half of ATOL, from 2 on, all of it from 4 on), so that half step is allowed besides.
    assert np.all(np.abs(got - want) <= ATOL + EPS * np.abs(want)) and rel_l2(got, want) <= RTOL_L2


CASES = [
    # layout, B, hq, hkv, tokens, nodes: no cache, a tail alone, whole pages alone, both; 4 rows to over 256 a head;
    # one, two and four mask words
    ("default", 1, 4, 1, 0, 1), ("default", 1, 8, 2, 0, 70), ("default", 1, 8, 2, 20, 5), ("default", 1, 8, 2, 64, 1),
    ("default", 1, 8, 2, 320, 16), ("default", 1, 32, 8, 1000, 8), ("default", 2, 28, 4, 300, 9),
    ("default", 1, 40, 2, 130, 40), ("default", 1, 8, 8, 200, 100), ("default", 1, 8, 1, 4500, 3),
    ("default", 1, 2, 2, 130, 256), ("default", 3, 4, 4, 64 * 3 + 63, 1), ("default", 1, 24, 2, 700, 10),
    ("fast", 1, 64, 8, 700, 16), ("fast", 2, 8, 2, 333, 12), ("fast", 1, 4, 1, 128, 30), ("fast", 1, 8, 8, 90, 200),
    ("deep2", 1, 8, 2, 333, 12), ("l1_8bit", 1, 8, 2, 333, 20), ("odd_split", 2, 8, 2, 333, 40),
    ("int8_default_angles", 1, 8, 2, 333, 7), ("odd_split", 1, 8, 2, 64, 3), ("deep2", 1, 16, 1, 200, 20),
]


@pytest.mark.parametrize("case", CASES)
def test_tree_against_oracle(device, case):
    layout, B, hq, hkv, tokens, n = case
    print(f"[tree] {case}", flush=True)
    cache = filled(device, layout, B, hq, hkv, tokens, seed=tokens + n)
    q, dk, dv = draft(device, B, hq, hkv, n, seed=n)
    tree = DraftTree(random_parents(n, n) if n % 2 else list(range(-1, n - 1)))
    scale = cache.config.attention_scale
    got = cache.tree_attention(q, dk, dv, tree, scale)
    assert got.shape == q.shape and got.dtype is torch.float16 and cache.offset == tokens
    check(got, q, dk, dv, tree, history(cache.runtime) if tokens else None, fp16_scale(scale), f"{case}")


def test_trees_of_their_own(device):
    """One tree per batch row, of different sizes: padding rows are 0."""
    cache = filled(device, "default", 3, 8, 2, 150, seed=5)
    trees = [random_parents(9, 1), [-1], random_parents(66, 2)]
    q, dk, dv = draft(device, 3, 8, 2, 66, seed=6)
    tree = DraftTree(trees, device=device)
    got = cache.tree_attention(q, dk, dv, tree, cache.config.attention_scale)
    check(got, q, dk, dv, tree, history(cache.runtime), fp16_scale(cache.config.attention_scale), "own trees")


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("n", [4, 40, 90])
def test_other_branches_do_not_leak(device, bad, n):
    """What a branch holds reaches its own nodes alone, infinities and NaN too; neither does padding."""
    cache = filled(device, "default", 1, 8, 2, 100, seed=7)
    parents = [-1, 0, 0] + [2] * (n - 3)
    q, dk, dv = draft(device, 1, 8, 2, n, seed=8)
    tree, scale = DraftTree(parents), cache.config.attention_scale
    want = cache.tree_attention(q, dk, dv, tree, scale)
    for t in (dk, dv):
        x = t.clone()
        x[:, :, 1] = bad
        got = cache.tree_attention(q, x if t is dk else dk, x if t is dv else dv, tree, scale)
        others = [i for i in range(n) if i != 1]
        assert torch.equal(got[:, :, others], want[:, :, others])
        assert not torch.isfinite(got[:, :, 1]).any()


def test_infinite_pages_and_padding(device):
    """A page whose values are infinite makes every node's output so, but not a padding node's."""
    cache = filled(device, "default", 2, 8, 2, 200, seed=9)
    cache.runtime.v_storage.scales[:, :, 1] = float("inf")
    q, dk, dv = draft(device, 2, 8, 2, 3, seed=9)
    got = cache.tree_attention(q, dk, dv, DraftTree([[-1, 0, 0], [-1]]), cache.config.attention_scale)
    assert bool((got[1, :, 1:] == 0).all()) and not torch.isfinite(got[0]).any() and not torch.isfinite(got[1, :, 0]).any()


def test_strides_types_and_bridge(device):
    cache = filled(device, "fast", 2, 8, 2, 200, seed=10)
    g = torch.Generator(device=device).manual_seed(10)
    rows = torch.randn((2, 5, 12, 128), generator=g, device=device).half()
    q, dk, dv = (t.transpose(1, 2) for t in rows.split([8, 2, 2], dim=2))
    tree, scale = DraftTree([-1, 0, 1, 1, 0]), cache.config.attention_scale
    want = cache.tree_attention(q.contiguous(), dk.contiguous(), dv.contiguous(), tree, scale)
    assert torch.equal(cache.tree_attention(q, dk, dv, tree, scale), want)
    assert torch.equal(cache.tree_attention(q.float(), dk.float(), dv.float(), tree, scale), want)
    key, value, tail_k, tail_v, _, _ = cache.runtime.get_fused_attention_inputs()
    out, trace = HipKernelBridge().execute_tree_attention_quant_v_dense_tail(q, key, value, tail_k, tail_v, dk, dv, tree,
                                                                             cache.config)
    assert torch.equal(out, want) and trace["nodes"] == 5 and trace["tail_length"] == 200 % 64
    none = TurboPolarFastCache(cache.config)
    out, _ = HipKernelBridge().execute_tree_attention_quant_v_dense_tail(q, None, None, None, None, dk, dv, tree, cache.config)
    assert torch.equal(out, none.tree_attention(q, dk, dv, tree, scale))
    one = dk[:, :1].expand(2, 2, 5, 128)
    assert torch.equal(cache.tree_attention(q, one, one, tree, scale),
                       cache.tree_attention(q, one.contiguous(), one.contiguous(), tree, scale))


def test_refusals_on_the_device(device):
    cache = filled(device, "default", 2, 8, 2, 100)
    q, dk, dv = draft(device, 2, 8, 2, 3, seed=1)
    tree = DraftTree([-1, 0, 0])
    with pytest.raises(ValueError, match="batch of q"):
        cache.tree_attention(q[:1], dk[:1], dv[:1], tree, 0.1)
    with pytest.raises(ValueError, match="KV heads"):
        cache.tree_attention(q, dk[:, :1], dv[:, :1], tree, 0.1)
    with pytest.raises(ValueError, match="does not match"):
        cache.tree_attention(q, dk, dv, DraftTree([[-1, 0, 0]] * 3), 0.1)
    with pytest.raises(ValueError, match="no gradients"):
        cache.tree_attention(q.requires_grad_(), dk, dv, tree, 0.1)
    assert cache.offset == 100


def test_graphs(device):
    """Two captured trees over two caches, replayed in turn with eager calls between."""
    caches = [filled(device, "default", 1, 8, 2, 900, seed=1), filled(device, "fast", 1, 8, 2, 300, seed=2)]
    trees = [DraftTree(random_parents(12, 3), device=device), DraftTree([-1, 0, 1], device=device)]
    drafts = [draft(device, 1, 8, 2, t.nodes, seed=i) for i, t in enumerate(trees)]
    call = lambda i: caches[i].tree_attention(*drafts[i], trees[i], 0.09)  # noqa: E731
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(i))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i]) and torch.equal(call(i), want[i])
            outs[i].zero_()


def test_offsets_past_32_bits(device):
    """The last head's last page of a store whose buffers are longer than 2^32 bytes: zero keys and
    values everywhere but there, where one token's key is the query's direction."""
    H, S = 3, 180_000
    cache = TurboPolarFastCache(config("default", H, H))
    rt = cache.runtime
    rt.k_storage.reserve(S, rt.polar_encoder, 1, H, device)
    rt.v_storage.reserve(S, 1, H, device)
    assert rt.k_storage.radii.numel() * 2 > 2 ** 32
    g = torch.Generator(device=device).manual_seed(3)
    k, v = torch.randn((2, 1, H, 64, 128), generator=g, device=device).half()
    probe = filled(device, "default", 1, H, H, 0)
    probe.runtime.append(k * 12, v)
    for name in ("radii", "angle_codes_l1", "angle_codes_deep"):
        getattr(rt.k_storage, name)[:, -1, S - 1] = getattr(probe.runtime.k_storage, name)[:, -1, 0]
    for name in ("codes", "scales"):
        getattr(rt.v_storage, name)[:, -1, S - 1] = getattr(probe.runtime.v_storage, name)[:, -1, 0]
    rt._batch_size, rt._num_kv_heads, rt._head_dim, rt._input_dtype, rt._initialized = 1, H, 128, torch.float16, True
    rt.k_storage.block_count = rt.v_storage.block_count = rt.total_blocks = S
    rt.actual_seq_len = S * PAGE
    keys, values = (torch.from_numpy(x) for x in pages64(probe.runtime))
    q = keys[:, :, 17:18].half().to(device)
    dk, dv = torch.zeros((2, 1, H, 1, 128), dtype=torch.float16, device=device)
    got = cache.tree_attention(q, dk, dv, DraftTree([-1]), cache.config.attention_scale).cpu().double()
    assert not got[0, :-1].any()  # the other heads' values are 0
    assert (got[0, -1, 0] - values[0, -1, 17]).abs().max() <= 4e-3  # exp(-50) of the rest and one fp16 step
    # and the same through a copy of that store
    other = cache.fork()
    assert torch.equal(other.runtime.k_storage.radii[0, -1, S - 1], rt.k_storage.radii[0, -1, S - 1])
    again = other.tree_attention(q, dk, dv, DraftTree([-1]), cache.config.attention_scale).cpu().double()
    assert torch.equal(again, got)


# ---- branches --------------------------------------------------------------------------


def buffers(rt):
    S = rt.k_storage.block_count
    out = {}
    for store, names in ((rt.k_storage, ("radii", "angle_codes_l1", "angle_codes_deep", "radii_scales")),
                         (rt.v_storage, ("codes", "scales"))):
        for name in names:
            t = getattr(store, name)
            if t is not None:
                out[name] = t[:, :, :S].cpu()
    return out


def same_pages(rt, source, rows=slice(None), pages=slice(None)):
    mine, theirs = buffers(rt), source if isinstance(source, dict) else buffers(source)
    for name, t in mine.items():
        assert torch.equal(t, theirs[name][rows][:, :, pages]), name
    for store in (rt.k_storage, rt.v_storage):  # the spare slots are clear
        assert store.capacity in (0, 4, 8, 16, 32) and store.capacity >= store.block_count
        for t in (getattr(store, n, None) for n in ("radii", "angle_codes_l1", "radii_scales", "codes", "scales")):
            if t is not None:
                assert not bool(t[:, :, store.block_count + 1:].any())


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("tokens", [30, 64, 64 * 4, 64 * 5 + 17])
def test_fork_copies_everything(device, layout, tokens):
    cache = filled(device, layout, 2, 4, 2, tokens, seed=tokens)
    before, tail = buffers(cache.runtime), cache.runtime.partial_k
    other = cache.fork()
    same_pages(other.runtime, cache.runtime)
    assert other.offset == tokens and other.runtime.get_io_telemetry()["total_blocks"] == tokens // 64
    assert other.runtime.get_io_telemetry()["actual_cache_bytes"] == cache.runtime.get_io_telemetry()["actual_cache_bytes"]
    # The two go their own ways.
    k, v = (torch.from_numpy(x).to(device) for x in gen_kv(1, 2, 2, 150))
    other.runtime.append(k, v)
    assert cache.offset == tokens and other.offset == tokens + 150
    for name, t in buffers(cache.runtime).items():
        assert torch.equal(t, before[name])
    assert (tail is None and cache.runtime.partial_k is None) or torch.equal(cache.runtime.partial_k, tail)
    cache.runtime.append(k, v)
    same_pages(other.runtime, cache.runtime)
    # A snapshot of a copy restores to the same cache.
    restored = wire.load_state_dict(*wire.state_dict(other), device)
    same_pages(restored, other.runtime)


def test_fork_rows_and_pages(device):
    cache = filled(device, "fast", 3, 4, 2, 64 * 6 + 9, seed=4)
    for rows in ([2, 0, 0, 1], [1], torch.tensor([0, 2], device=device)):
        other = cache.fork(rows=rows)
        at = [int(x) for x in rows]
        same_pages(other.runtime, cache.runtime, rows=at)
        assert torch.equal(other.runtime.partial_k, cache.runtime.partial_k[at])
        assert torch.equal(other.runtime.partial_v, cache.runtime.partial_v[at])
    for pages in ([5, 0, 3], [], [2, 2], list(range(6))):
        other = cache.fork(pages=pages)
        same_pages(other.runtime, cache.runtime, pages=pages)
        assert other.offset == 64 * len(pages) + 9 and torch.equal(other.runtime.partial_k, cache.runtime.partial_k)
    many = [i % 6 for i in range(800)]  # past what travels with a launch
    other = cache.fork(rows=[2], pages=many)
    for name, t in buffers(other.runtime).items():
        assert torch.equal(t, buffers(cache.runtime)[name][[2]][:, :, many]), name
    both = cache.fork(rows=[1, 1], pages=[4])
    same_pages(both.runtime, cache.runtime, rows=[1, 1], pages=[4])


def test_fork_keeps_a_set_encoder(device):
    """A cache whose encoder was given another layout forks with it."""
    cache = TurboPolarFastCache(config("default", 4, 2))
    cache.runtime.polar_encoder.k_angle_bits_deep = 8
    k, v = (torch.from_numpy(x).to(device) for x in gen_kv(1, 1, 2, 200))
    cache.runtime.append(k, v)
    other = cache.fork(tokens=150)
    other.runtime.append(k[:, :, 150:].contiguous(), v[:, :, 150:].contiguous())
    assert other.runtime.k_storage.angle_codes_deep.shape == cache.runtime.k_storage.angle_codes_deep.shape
    q, dk, dv = draft(device, 1, 4, 2, 3, seed=1)
    tree = DraftTree([-1, 0, 1])
    got = other.tree_attention(q, dk, dv, tree, 0.09)
    check(got, q, dk, dv, tree, history(other.runtime), fp16_scale(0.09), "set encoder")


@pytest.mark.parametrize("layout", ["default", "fast", "odd_split"])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("keep", [0, 1, 63, 64, 100, 64 * 4, 64 * 5, 64 * 5 + 3, 64 * 5 + 17])
def test_prefix_and_truncate(device, layout, dtype, keep):
    """Whole pages stay bit for bit; a page cut in two leaves its first tokens as the oracle decodes
    them (within the one fp16 step of the page decoder) in the tail."""
    from common import within_f16_ulp

    cache = filled(device, layout, 2, 4, 2, 64 * 5 + 17, seed=keep, dtype=dtype)
    rt = cache.runtime
    held = buffers(rt)
    k64, v64 = history(rt)
    other = cache.fork(tokens=keep, rows=[1, 0])
    cache.truncate(keep)
    for x, rows in ((rt, [0, 1]), (other.runtime, [1, 0])):
        assert x.actual_seq_len == keep and x._tail_len == (keep - 64 * 5 if keep >= 64 * 5 else keep % 64)
        for name, t in buffers(x).items():
            assert torch.equal(t, held[name][rows][:, :, : keep // 64]), name
        if x._tail_len:
            start = keep - x._tail_len
            assert within_f16_ulp(x.partial_k.cpu().numpy(), k64[rows][:, :, start:keep])
            assert within_f16_ulp(x.partial_v.cpu().numpy(), v64[rows][:, :, start:keep])
            assert x.partial_k.dtype is (torch.float32 if dtype is np.float32 else torch.float16)
    assert rt.total_blocks == rt.k_storage.block_count
    # Both go on as caches do.
    k, v = (torch.from_numpy(t).to(device) for t in gen_kv(2, 2, 2, 130, dtype=dtype))
    rt.append(k, v)
    other.runtime.append(k[[1, 0]].contiguous(), v[[1, 0]].contiguous())
    if keep:
        same_pages(other.runtime, rt, rows=[1, 0])
        assert rt.bytes_written == rt.k_storage.block_count * rt._page_bytes()


def test_select_and_keep_in_place(device):
    cache = filled(device, "default", 3, 8, 2, 64 * 5 + 20, seed=6)
    before, tail = buffers(cache.runtime), cache.runtime.partial_v
    cache.select_rows([2, 2])
    same_pages(cache.runtime, before, rows=[2, 2])
    cache.keep_pages([4, 1])
    same_pages(cache.runtime, before, rows=[2, 2], pages=[4, 1])
    assert cache.offset == 148 and torch.equal(cache.runtime.partial_v, tail[[2, 2]])
    q, dk, dv = draft(device, 2, 8, 2, 5, seed=6)
    tree = DraftTree([-1, 0, 1, 0, 3])
    got = cache.tree_attention(q, dk, dv, tree, cache.config.attention_scale)
    check(got, q, dk, dv, tree, history(cache.runtime), fp16_scale(cache.config.attention_scale), "selected")


@pytest.mark.parametrize("tokens,path", [
    (0, [0]), (10, [3, 5]), (62, [0, 1]), (63, [2]), (60, [1, 2, 3, 4, 5, 6]), (64 * 4, [7]), (300, [0, 2, 4, 6]),
    (5, list(range(64)) + [3] * 90), (100, [[0, 1, 2], [5, 5, 5]]),
])
@pytest.mark.parametrize("layout,dtype", [("default", np.float16), ("fast", np.float32)])
def test_accept_is_append(device, tokens, path, layout, dtype):
    """Accepting a path leaves the cache as appending its tokens does, bit for bit."""
    one = filled(device, layout, 2, 4, 2, tokens, seed=1, dtype=dtype).runtime
    two = filled(device, layout, 2, 4, 2, tokens, seed=1, dtype=dtype).runtime
    n = 64 if len(path) > 8 else 8
    rows = torch.from_numpy(np.concatenate(gen_kv(3, 2, 2, n, dtype=dtype), axis=1)).to(device)
    k, v = rows.transpose(1, 2).contiguous().transpose(1, 2).split(2, dim=1)  # token-major views
    one.accept(k, v, path)
    per_row = path if isinstance(path[0], list) else [path] * 2
    two.append(*(torch.stack([t[b][:, per_row[b]] for b in range(2)]) for t in (k, v)))
    assert one.actual_seq_len == two.actual_seq_len and one._tail_len == two._tail_len
    if one.k_storage.block_count:
        same_pages(one, two)
    for a, b in ((one.partial_k, two.partial_k), (one.partial_v, two.partial_v)):
        assert (a is None and b is None) or torch.equal(a, b)
    one.append(k[:, :, :1].contiguous(), v[:, :, :1].contiguous())


def test_accept_refuses_and_leaves_the_cache(device):
    cache = filled(device, "default", 1, 4, 2, 100, seed=2)
    _, k, v = draft(device, 1, 4, 2, 6, seed=2)
    k[0, 1, 4, 7] = float("inf")
    before = cache.runtime.partial_k
    for path in ([4], [0, 4], [0] * 40 + [4]):
        with pytest.raises(ValueError, match="finite"):
            cache.accept(k, v, path)
        assert cache.offset == 100 and torch.equal(cache.runtime.partial_k, before)
    cache.accept(k, v, [0, 5])  # what is not taken may hold anything
    assert cache.offset == 102


def test_deferred_verdicts_come_first(device):
    cache = filled(device, "default", 1, 4, 2, 70, seed=3)
    q, k, v = draft(device, 1, 4, 2, 1, seed=3)
    bad = k.clone()
    bad[0, 0, 0, 0] = float("nan")
    for use in (lambda: cache.fork(), lambda: cache.truncate(65), lambda: cache.accept(k, v, [0]),
                lambda: cache.tree_attention(q, k, v, DraftTree([-1]), 0.1)):
        cache.decode_attention(q, bad, v, 0.1, defer_check=True)
        with pytest.raises(ValueError, match="finite"):
            use()
        assert cache.offset == 70


def test_drafted_generation(device):
    """Speculative steps end to end, over page borders: draft a tree, attend it, accept a path, roll
    a wrong one back; beside a cache that takes the same tokens one by one."""
    hq, hkv, scale = 8, 2, 128 ** -0.5
    rng = np.random.default_rng(0)
    spec, plain = (filled(device, "default", 1, hq, hkv, 50, seed=4) for _ in range(2))
    for step in range(12):
        n = 9
        parents = random_parents(n, step)
        tree = DraftTree(parents)
        q, k, v = draft(device, 1, hq, hkv, n, seed=100 + step)
        out = spec.tree_attention(q, k, v, tree, scale)
        path = tree.path_to(int(rng.integers(0, n)))
        if step % 3 == 2:  # accepted, then taken back
            held = spec.offset
            branch = spec.fork()
            branch.accept(k, v, path)
            assert spec.offset == held and branch.offset == held + len(path)
        spec.accept(k, v, path)
        for node in path:
            want = plain.decode_attention(q[:, :, node:node + 1], k[:, :, node:node + 1], v[:, :, node:node + 1], scale)
            crossed = plain.offset % PAGE == 0 or (plain.offset - len(path)) // PAGE != plain.offset // PAGE
            # Once a page is full the plain cache attends its codes, the draft its dense tokens.
            if not crossed:
                assert (out[:, :, node].double() - want.double()).abs().max() <= ATOL
        assert spec.offset == plain.offset
        assert (spec.runtime._tail_len == 0 and plain.runtime._tail_len == 0) or torch.equal(
            spec.runtime.partial_k, plain.runtime.partial_k)
    same_pages(spec.runtime, plain.runtime)
    assert spec.runtime.k_storage.block_count >= 1


# ---- a prompt through the cache ----------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_prompt_through_the_cache(device, dtype):
    """Chunks of a prompt: the same history as update_and_fetch hands out, attended causally."""
    from turbopolar_amd.kernels import prompt_attention

    cache, twin = (TurboPolarFastCache(config("fast", 8, 2)) for _ in range(2))
    g = torch.Generator(device=device).manual_seed(1)
    for T in (70, 1, 130):
        q, k, v = (torch.randn((2, h, T, 128), generator=g, device=device).to(dtype) for h in (8, 2, 2))
        out = cache.prompt_attention(q, k, v, 0.088)
        kk, vv = twin.update_and_fetch(k.half(), v.half())
        assert out.dtype is dtype and torch.equal(out, prompt_attention(q.half(), kk, vv, 0.088).to(dtype))
    assert cache.offset == 201
    with pytest.raises(ValueError):
        cache.prompt_attention(q, k[:, :, :5], v[:, :, :5], 0.088)
    assert cache.offset == 201


def test_emptied_branches(device):
    """A branch that never had a tail, cut to nothing, is forked, filled and forked again."""
    cache = filled(device, "default", 2, 8, 2, 64 * 3, seed=4)
    branch = cache.fork()
    branch.truncate(0)
    again = branch.fork(rows=[1])
    assert again.offset == 0 and branch.fork(pages=[]).offset == 0
    k, v = (torch.from_numpy(x).to(device) for x in gen_kv(5, 1, 2, 70))
    again.runtime.append(k, v)
    fresh = TurboPolarFastCache(config("default", 8, 2))
    fresh.runtime.append(k, v)
    same_pages(again.runtime, fresh.runtime)
    assert torch.equal(again.fork().runtime.partial_k, fresh.runtime.partial_k) and cache.offset == 192


def test_trees_on_another_stream(device):
    """A tree that is dropped while another stream still reads it keeps its masks' memory until then."""
    cache = filled(device, "default", 1, 8, 2, 64 * 100, seed=5)
    q, dk, dv = draft(device, 1, 8, 2, 60, seed=5)
    parents = random_parents(60, 5)
    want = cache.tree_attention(q, dk, dv, DraftTree(parents), 0.1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        tree = DraftTree(parents, device=device)
        with torch.cuda.stream(side):
            got = [cache.tree_attention(q, dk, dv, tree, 0.1) for _ in range(4)]
        del tree
        over = [torch.zeros((1, 60, 1), dtype=torch.int64, device=device) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got) and len(over) == 4


def test_prompt_in_place(device):
    q, k, v = draft(device, 1, 8, 2, 300, seed=6)
    want = prompt_attention(q, k, v, 0.1)
    assert torch.equal(prompt_attention(q, k, v, 0.1, out=q), want)


def test_branches_cut_to_nothing(device):
    """Forks of no tokens or pages own no buffers: they are forked, re-ordered, attended and filled all the same."""
    cache = filled(device, "fast", 2, 8, 2, 64 * 3, seed=8)
    kept = cache.fork()
    kept.keep_pages([])
    k, v = (torch.from_numpy(x).to(device) for x in gen_kv(9, 2, 2, 70))
    fresh = TurboPolarFastCache(cache.config)
    fresh.runtime.append(k, v)
    q, dk, dv = draft(device, 2, 8, 2, 3, seed=9)
    tree = DraftTree([-1, 0, 0])
    alone = TurboPolarFastCache(cache.config).tree_attention(q, dk, dv, tree, 0.1)
    for branch in (cache.fork(tokens=0), cache.fork(pages=[]), kept):
        assert branch.offset == 0 and branch.runtime.k_storage.radii is None and branch.runtime._tail_k is None
        for again in (branch.fork(), branch.fork(tokens=0, rows=[1, 0]), branch.fork(pages=[])):
            assert torch.equal(again.tree_attention(q, dk, dv, tree, 0.1), alone)
            again.runtime.append(k, v)
            same_pages(again.runtime, fresh.runtime)
            assert torch.equal(again.runtime.partial_v, fresh.runtime.partial_v)
        branch.select_rows([0])
        branch.keep_pages([])
        branch.runtime.append(k[:1], v[:1])
        same_pages(branch.runtime, fresh.runtime, rows=[0])
    assert cache.offset == 192


def test_prompt_refused_leaves_the_cache(device):
    """A scale that is not finite in 32 bits is refused before the chunk is appended."""
    cache = filled(device, "fast", 1, 8, 2, 100, seed=2)
    q, k, v = draft(device, 1, 8, 2, 5, seed=2)
    for scale in (float("nan"), float("-inf"), 1e300):
        with pytest.raises(ValueError, match="scale"):
            cache.prompt_attention(q, k, v, scale)
        assert cache.offset == 100
    cache.prompt_attention(q, k, v, 0.1)
    assert cache.offset == 105


@pytest.mark.parametrize("use,pages,rows", [
    (lambda c: c.select_rows([1, 1, 0]), list(range(6)), [1, 1, 0]), (lambda c: c.keep_pages([5, 0]), [5, 0], [0, 1])])
def test_replaced_buffers_outlive_their_copy(device, use, pages, rows):
    """Rows selected and pages kept on a stream other than the buffers' own: what another stream allocates
    while the copy still waits does not lie over what it reads."""
    side = torch.cuda.Stream()
    for seed in range(3):
        cache = filled(device, "fast", 2, 8, 2, 64 * 6 + 20, seed=seed)
        rt = cache.runtime
        before, tail = buffers(rt), rt.partial_k
        sizes = [(t.shape, t.dtype) for t in (*rt.k_storage._buffers(), rt.v_storage.codes, rt.v_storage.scales, rt._tail_k,
                                              rt._tail_v)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            use(cache)
        over = [torch.full(shape, 7, dtype=dtype, device=device) for shape, dtype in sizes for _ in range(2)]
        torch.cuda.synchronize()
        same_pages(rt, before, rows=rows, pages=pages)
        assert torch.equal(rt.partial_k, tail[rows]) and len(over) == 2 * len(sizes)


def test_growth_on_another_stream(device):
    """A page completed on a stream other than the store's: the outgrown buffers are not allocated anew while
    they are still copied."""
    side = torch.cuda.Stream()
    k, v = (torch.from_numpy(x).to(device) for x in gen_kv(1, 2, 2, 64 * 5))
    cut = 64 * 4 + 63
    whole = TurboPolarFastCache(config("fast", 8, 2)).runtime
    whole.append(k, v)
    for _ in range(3):
        rt = TurboPolarFastCache(config("fast", 8, 2)).runtime
        rt.append(k[:, :, :64 * 4].contiguous(), v[:, :, :64 * 4].contiguous())
        rt.append(k[:, :, 64 * 4:cut].contiguous(), v[:, :, 64 * 4:cut].contiguous())
        sizes = [(t.shape, t.dtype) for t in (*rt.k_storage._buffers(), rt.v_storage.codes, rt.v_storage.scales)]
        last = k[:, :, cut:].contiguous(), v[:, :, cut:].contiguous()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            rt.append(*last, defer_check=True)
        over = [torch.full(shape, 7, dtype=dtype, device=device) for shape, dtype in sizes for _ in range(2)]
        torch.cuda.synchronize()
        rt.resolve_deferred_check()
        assert rt.k_storage.reallocation_count == whole.k_storage.reallocation_count == 1 and len(over) == 2 * len(sizes)
        same_pages(rt, whole)


def test_compaction_frees_what_it_drops(device):
    """Nothing of a cache that was attended keeps the buffers that select_rows or keep_pages replaced."""
    import weakref

    q, dk, dv = draft(device, 2, 8, 2, 3, seed=3)
    tree = DraftTree([-1, 0, 1])
    for use in (lambda c: c.keep_pages([]), lambda c: c.keep_pages([2]), lambda c: c.select_rows([1, 0])):
        cache = filled(device, "fast", 2, 8, 2, 64 * 4, seed=3)
        cache.tree_attention(q, dk, dv, tree, 0.1)
        cache.runtime.get_fused_attention_inputs()
        held = [weakref.ref(t) for t in (*cache.runtime.k_storage._buffers(), cache.runtime.v_storage.codes,
                                         cache.runtime.v_storage.scales)]
        use(cache)
        assert [r() is None for r in held] == [True] * len(held)
        cache.tree_attention(q, dk, dv, tree, 0.1)


def test_many_small_weights(device):
    """One stored key of weight 1 beside 2,560 of e^-18, three pages of them in its workgroup.  Weights lie up to 2^7
    above 1, so each is off by 2^-32 at most; a record and the result are fp16, subnormal here."""
    B, H, T = 8, 8, 64 * 40
    cache = TurboPolarFastCache(config("default", H, H))
    k = torch.zeros((B, H, T, 128), dtype=torch.float16, device=device)
    v = torch.ones_like(k)
    k[:, :, 5, 0], v[:, :, 5] = -18.0, 0.0
    cache.runtime.append(k, v)
    q, dk = torch.zeros((2, B, H, 1, 128), dtype=torch.float16, device=device)
    q[..., 0] = -1.0
    got = cache.tree_attention(q, dk, torch.ones_like(dk), DraftTree([-1]), 1.0).double().cpu()
    keys, values = pages64(cache.runtime)
    assert (keys[0, 0, 5, 0], keys[0, 0, 6, 0], values[0, 0, 5, 0]) == (-18.0, 0.0, 0.0)
    w = np.exp(-18.0)
    want = (w * values[0, 0].sum(0) + w) / (1 + T * w)
    tol = want * (2 * EPS + 2 * 18 * 129 * 2.0 ** -24 + (T + 16) * 2.0 ** -23) + T * 2.0 ** -32 + 2 * 2.0 ** -25
    off = np.abs(got[:, :, 0].numpy() - want)
    print(f"[tree] small weights: {off.max():.3g} of {tol.max():.3g}", flush=True)
    assert (off <= tol).all()


@pytest.mark.parametrize("layout,hkv,n", [("default", 2, 5), ("default", 2, 16), ("default", 1, 16), ("deep2", 2, 16),
                                          ("l1_8bit", 1, 20)])
def test_keys_are_the_page_decoders(device, layout, hkv, n):
    """The keys attended are those that the page decoder hands out, each component rounded to fp16 once: queries of
    four large components tell scores of a few steps apart.  A score is then a sum of four products, off by
    5 2^-24 sum|q||k|, a weight by twice that and its rounding, and records and the result are rounded once."""
    cache = filled(device, layout, 1, 8, hkv, 64 * 6, seed=n)
    q, dk, dv = draft(device, 1, 8, hkv, n, seed=n + 50)
    q[..., 4:] = 0
    q *= 8
    got = cache.tree_attention(q, dk, dv, DraftTree(list(range(-1, n - 1))), 1.0).double().cpu().numpy()
    keys = cache.runtime.fetch_blocks().double().cpu().numpy()
    values = pages64(cache.runtime)[1]
    q64, k64, v64 = (t.double().cpu().numpy() for t in (q, dk, dv))
    worst = 0.0
    for i in range(n):
        for h in range(8):
            kv = h // (8 // hkv)
            k = np.concatenate((keys[0, kv], k64[0, kv, : i + 1]))
            v = np.concatenate((values[0, kv], v64[0, kv, : i + 1]))
            s = k @ q64[0, h, i]
            p = np.exp(s - s.max())
            p /= p.sum()
            ds = 5 * 2.0 ** -24 * (np.abs(k) @ np.abs(q64[0, h, i])).max()
            tol = (p @ np.abs(v)) * (3 * EPS + np.expm1(2 * ds) + (len(s) + 16) * 2.0 ** -23)
            tol += (len(s) + 2) * 2.0 ** -25 * np.abs(v).max()
            worst = max(worst, (np.abs(got[0, h, i] - p @ v) / tol).max())
    print(f"[tree] page decoder's keys, {layout}: {worst:.3g} of the bound", flush=True)
    assert worst <= 1


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_caches_filled_in_inference_mode(device, dtype):
    """They are cut, forked, re-ordered and extended outside of it like any other."""
    with torch.inference_mode():
        cache = filled(device, "default", 2, 8, 2, 64 * 3 + 9, seed=7, dtype=dtype)
    plain = filled(device, "default", 2, 8, 2, 64 * 3 + 9, seed=7, dtype=dtype)
    k, v = (torch.from_numpy(x).to(device) for x in gen_kv(8, 2, 2, 7, dtype=dtype))
    for c in (cache, plain):
        c.truncate(64 * 2 + 30)
        c.select_rows([1, 0])
        c.runtime.accept(k, v, [2, 0])
    other = cache.fork(tokens=64 + 5)
    same_pages(cache.runtime, plain.runtime)
    for a, b in ((cache, plain), (other, plain.fork(tokens=64 + 5))):
        assert a.offset == b.offset and torch.equal(a.runtime.partial_k, b.runtime.partial_k)
