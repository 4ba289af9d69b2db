"""tp_prompt_attention against attention in float64 on the same fp16 / bf16 inputs.

Error of an output element, with eps half a step of the type (2^-11 fp16, 2^-8 bf16), A = sum_j p_j
|v_j| and l >= 1 the sum of the unnormalised weights (the largest is 1): the weights are rounded
once (eps A; for fp16 those below 2^-14 by 2^-25 each, n 2^-25 max|v|), the result once (eps A, or
2^-25), and the fp32 parts are small: a score is off by at most 129 2^-24 scale sum|q||k|, hence a
weight by that, twice (its own and the sum's), plus 4 2^-23 for the exponentials and n 2^-24 for the
sums.  So |error| <= A (2 eps + 2 ds + (n + 16) 2^-23) + (n + 1) 2^-25 max|v|."""

import pytest
import torch

from turbopolar_amd import HipKernelBridge, TurboPolarConfig
from turbopolar_amd.kernels import prompt_attention

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SCALE = 128 ** -0.5


def make(device, dtype, B, hq, hkv, tq, tk, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    draw = lambda h, t: torch.randn((B, h, t, 128), generator=g, device=device).to(dtype)  # noqa: E731
    return draw(hq, tq), draw(hkv, tk), draw(hkv, tk)


def reference(q, k, v, scale, causal):
    """(attention of one batch of sequences of one length in float64, the error bound of each element)."""
    B, hq, tq, _ = q.shape
    hkv, tk = k.shape[1], k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.full(q.shape, 2.0 ** -25, dtype=torch.float64, device=q.device)
    eps = torch.finfo(q.dtype).eps / 2
    if tk == 0:
        return out, tol
    for b in range(B):
        for h in range(hq):
            qq, kk, vv = q[b, h].double(), k[b, h // (hq // hkv)].double(), v[b, h // (hq // hkv)].double()
            s = qq @ kk.T * scale
            seen = torch.ones_like(s, dtype=torch.bool)
            if causal:
                seen = seen.tril(tk - tq)
            s = s.masked_fill(~seen, float("-inf"))
            top = s.amax(-1, keepdim=True)
            w = torch.where(seen, torch.exp(s - torch.where(top.isinf(), 0.0, top)), 0.0)
            p = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            out[b, h] = p @ vv
            ds = (qq.abs() @ kk.abs().T).amax(-1, keepdim=True) * abs(scale) * 129 * 2.0 ** -24
            tol[b, h] += (p @ vv.abs()) * (2 * eps + 2 * ds + (tk + 16) * 2.0 ** -23) + (tk + 1) * 2.0 ** -25 * vv.abs().max()
    return out, tol


def close(got, want, tol, what):
    over = ((got.double() - want).abs() - tol).max().item() if got.numel() else 0.0
    print(f"[prompt] {what}: worst error past its bound {over:.3g}", flush=True)
    assert over <= 0 and torch.isfinite(got).all(), what


SHAPES = [
    # B, hq, hkv, tq, tk: one token; odd sizes; a tile's and a workgroup's borders; long keys for few rows
    (1, 4, 1, 1, 1), (2, 4, 2, 1, 7), (1, 8, 8, 3, 3), (1, 32, 8, 63, 63), (1, 32, 8, 64, 64), (1, 8, 2, 65, 65),
    (1, 28, 4, 257, 257), (3, 6, 2, 130, 130), (1, 40, 2, 77, 77), (1, 8, 1, 300, 300), (1, 4, 4, 513, 513),
    (1, 32, 8, 1, 5000), (2, 8, 2, 5, 1999), (1, 8, 2, 100, 1111), (1, 4, 2, 1025, 1025), (1, 5, 5, 200, 131),
    (1, 4, 2, 50, 3), (1, 4, 2, 9, 0),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_float64(device, shape, causal, dtype):
    print(f"[prompt] {shape} causal={causal} {dtype}", flush=True)
    q, k, v = make(device, dtype, *shape, seed=sum(shape))
    got = prompt_attention(q, k, v, SCALE, causal=causal)
    assert got.shape == q.shape and got.dtype is dtype
    close(got, *reference(q, k, v, SCALE, causal), f"{shape}")


def test_steep_scores(device):
    """Scores far apart: the running maximum moves by hundreds between tiles, both ways."""
    q, k, v = make(device, F16, 1, 8, 2, 300, 300, seed=3)
    ramp = torch.linspace(0.1, 12, 300, device=device)[:, None]
    for kk in (k * ramp.half(), k * ramp.flip(0).half()):
        close(prompt_attention(q, kk, v, SCALE), *reference(q, kk, v, SCALE, True), "steep")


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0])
def test_scales(device, scale):
    q, k, v = make(device, F16, 1, 4, 2, 90, 170, seed=4)
    close(prompt_attention(q, k, v, scale), *reference(q, k, v, scale, True), f"scale {scale}")


PACKED = [
    # lengths of the sequences' queries and keys, and rows behind the last
    ([5, 1, 0, 130, 64, 3], [5, 1, 0, 130, 64, 3], 7),
    ([1, 1, 1], [400, 1, 33], 0),
    ([70, 0, 20], [70, 9, 700], 300),
    ([4, 30, 6], [0, 10, 6], 1),
    ([0, 0], [0, 0], 12),
    ([1] * 150 + [200], [1] * 150 + [200], 2),
]


def starts_of(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


@pytest.mark.parametrize("heads", [(8, 2), (28, 4), (4, 4)])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed(device, case, heads):
    nq, nk, rest = PACKED[case]
    qs, ks = starts_of(nq), starts_of(nk)
    print(f"[prompt] packed {case} heads {heads}", flush=True)
    q, k, v = make(device, F16, 1, *heads, qs[-1] + rest, ks[-1] + 3, seed=case)
    k[:, :, ks[-1]:], v[:, :, ks[-1]:] = float("nan"), float("inf")  # no sequence's
    want, tol = torch.zeros(q.shape, dtype=torch.float64, device=device), torch.zeros_like(q, dtype=torch.float64)
    for a, b, c, d in zip(qs, qs[1:], ks, ks[1:]):
        want[:, :, a:b], tol[:, :, a:b] = reference(q[:, :, a:b], k[:, :, c:d], v[:, :, c:d], SCALE, True)
    on = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    got = prompt_attention(q, k, v, SCALE, q_starts=on(qs), k_starts=on(ks))
    close(got, want, tol, f"packed {case}")
    assert torch.equal(got, prompt_attention(q, k, v, SCALE, q_starts=qs, k_starts=ks))
    # Into a given output, the rows behind the last sequence stay as they were.
    out = torch.full(q.shape, 7.0, dtype=F16, device=device)
    back = prompt_attention(q, k, v, SCALE, q_starts=on(qs), k_starts=on(ks), out=out)
    assert back is out and torch.equal(out[:, :, :qs[-1]], got[:, :, :qs[-1]])
    assert bool((out[:, :, qs[-1]:] == 7.0).all()) and bool((got[:, :, qs[-1]:] == 0).all())


def test_packed_full(device):
    """Without the causal mask each query sees its own sequence whole, and nothing of the next."""
    qs = starts_of([40, 100, 1])
    q, k, v = make(device, BF16, 1, 8, 2, 141, 141, seed=9)
    got = prompt_attention(q, k, v, SCALE, causal=False, q_starts=qs, k_starts=qs)
    for a, b in zip(qs, qs[1:]):
        close(got[:, :, a:b], *reference(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], SCALE, False), f"rows {a}:{b}")


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("heads", [(8, 2), (4, 4)])
def test_nonfinite_where_masked(device, bad, heads):
    """Keys and values that a query does not see do not reach it; those that it sees do."""
    q, k, v = make(device, F16, 1, *heads, 400, 400, seed=11)
    want, tol = reference(q, k, v, SCALE, True)
    at = 150
    v2, k2 = v.clone(), k.clone()
    v2[:, :, at, 5] = bad
    got = prompt_attention(q, k, v2, SCALE)
    close(got[:, :, :at], want[:, :, :at], tol[:, :, :at], "before")
    assert not torch.isfinite(got[:, :, at:, 5]).any()
    others = [d for d in range(128) if d != 5]
    close(got[..., others], want[..., others], tol[..., others], "other dimensions")
    k2[:, :, at:] = bad
    got = prompt_attention(q, k2, v, SCALE)
    close(got[:, :, :at], want[:, :, :at], tol[:, :, :at], "before, keys")


def test_strides(device):
    """Token-major projections, slices of a larger buffer, heads that share memory, rows off 16 bytes."""
    g = torch.Generator(device=device).manual_seed(12)
    B, T = 2, 75
    qkv = torch.randn((B, T, 8 + 2 + 2, 128), generator=g, device=device).half()
    q, k, v = (x.transpose(1, 2) for x in qkv.split([8, 2, 2], dim=2))
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), SCALE)
    assert torch.equal(prompt_attention(q, k, v, SCALE), want)
    close(want, *reference(q, k, v, SCALE, True), "projections")
    big = torch.randn((B, 1, T + 9, 128), generator=g, device=device).half()
    shared = big[:, :, 4:4 + T].expand(B, 2, T, 128)
    assert torch.equal(prompt_attention(q, shared, shared, SCALE),
                       prompt_attention(q, shared.contiguous(), shared.contiguous(), SCALE))
    odd = torch.randn((B, 2, T, 132), generator=g, device=device).half()[..., 1:129]
    assert torch.equal(prompt_attention(q, odd, odd, SCALE), prompt_attention(q, odd.contiguous(), odd.contiguous(), SCALE))
    out = torch.zeros((B, T + 1, 8, 128), dtype=F16, device=device)
    prompt_attention(q, k, v, SCALE, out=out[:, :T].transpose(1, 2))
    assert torch.equal(out[:, :T].transpose(1, 2), want) and bool((out[:, T:] == 0).all())


def test_bridge(device):
    import numpy as np

    cfg = TurboPolarConfig(num_q_heads=8, num_kv_heads=2)
    q, k, v = make(device, F16, 1, 8, 2, 33, 33, seed=13)
    out, trace = HipKernelBridge().execute_prompt_attention(q, k, v, cfg)
    assert torch.equal(out, prompt_attention(q, k, v, float(np.float16(cfg.attention_scale))))
    assert trace["hip_used"] and trace["causal"] and not trace["packed"] and trace["num_queries_per_kv"] == 4


def test_graphs_and_streams(device):
    """Two captured graphs, replayed in turn with eager calls between, on a stream of their own."""
    cases = [make(device, F16, 1, 8, 2, 4, 3001, seed=14), make(device, F16, 1, 8, 2, 200, 200, seed=15)]
    want = [prompt_attention(*c, SCALE) for c in cases]
    fresh = [make(device, F16, 1, 8, 2, c[0].shape[2], c[1].shape[2], seed=20 + i) for i, c in enumerate(cases)]
    want2 = [prompt_attention(*c, SCALE) for c in fresh]
    torch.cuda.synchronize()
    stream, graphs, outs = torch.cuda.Stream(), [], []
    with torch.cuda.stream(stream):
        for c in cases:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(prompt_attention(*c, SCALE))
            graphs.append(graph)
        for _ in range(3):
            for graph in graphs:
                graph.replay()
            stream.synchronize()
            for o, w, c in zip(outs, want, cases):
                assert torch.equal(o, w) and torch.equal(prompt_attention(*c, SCALE), w)
                o.zero_()
        for c, f in zip(cases, fresh):
            for x, y in zip(c, f):
                x.copy_(y)
        for graph in graphs[::-1]:
            graph.replay()
        stream.synchronize()
        for o, w in zip(outs, want2):
            assert torch.equal(o, w)


def test_offsets_past_32_bits(device):
    """Rows so far apart that their offsets pass 2^32 elements."""
    step, T = 1 << 25, 140
    store = torch.empty((T, step), dtype=F16, device=device)
    k, v = store[None, None, :, :128], store[None, None, :, 128:256]
    q, k0, v0 = make(device, F16, 1, 4, 1, 70, T, seed=16)
    k.copy_(k0)
    v.copy_(v0)
    assert torch.equal(prompt_attention(q, k, v, SCALE), prompt_attention(q, k0, v0, SCALE))


def test_refuses_gradients(device):
    q, k, v = make(device, F16, 1, 4, 2, 3, 3)
    with pytest.raises(ValueError, match="no gradients"):
        prompt_attention(q.requires_grad_(), k, v, SCALE)
    with torch.no_grad():
        prompt_attention(q, k, v, SCALE)


def test_refuses_tangents(device):
    import torch.autograd.forward_ad as fw

    q, k, v = make(device, F16, 1, 4, 2, 3, 3)
    with fw.dual_level():
        for i in range(3):
            args = [fw.make_dual(t, t) if j == i else t for j, t in enumerate((q, k, v))]
            with pytest.raises(ValueError, match="no gradients"):
                prompt_attention(*args, SCALE)
        assert torch.equal(prompt_attention(q, k, v, SCALE), prompt_attention(q, k, v, SCALE, out=torch.empty_like(q)))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("at", [0, 20_000, 32_767])
def test_many_small_weights(device, at, dtype):
    """One key of weight 1 beside 32,767 of e^-18, in one workgroup's run of keys: 5e-4 of the result.  fp16 weights
    lie up to 2^7 above 1, so each is off by 2^-32 at most (they are below the type's least normal number)."""
    n, w = 32768, 1.5229979744712628e-08
    q = torch.zeros((1, 64, 1024, 128), dtype=dtype, device=device)
    k = torch.zeros((1, 1, n, 128), dtype=dtype, device=device)
    v = torch.ones((1, 1, n, 128), dtype=dtype, device=device)
    q[..., 0], k[:, :, at, 0], v[:, :, at] = 1.0, 18.0, 0.0
    got = prompt_attention(q, k.expand(1, 64, n, 128), v.expand(1, 64, n, 128), 1.0, causal=False)
    want = (n - 1) * w / (1 + (n - 1) * w)
    eps = torch.finfo(dtype).eps / 2
    tol = want * (2 * eps + 2 * 18 * 129 * 2.0 ** -24 + (n + 16) * 2.0 ** -23) + (n * 2.0 ** -32 + 2.0 ** -25 if dtype is F16 else 0)
    print(f"[prompt] small weights at {at} {dtype}: {got.double().sub(want).abs().max().item():.3g} of {tol:.3g}", flush=True)
    assert (got.double() - want).abs().max() <= tol


@pytest.mark.parametrize("last", [65536, 100])
def test_most_sequences(device, last):
    """65,536 sequences of a token, or as many of which most are empty: each token sees itself alone, whose weight
    is 1."""
    n = 65536
    q, k, v = make(device, F16, 1, 4, 2, n, n, seed=17)
    starts = torch.arange(n + 1, dtype=torch.int32, device=device).clamp(max=last)
    got = prompt_attention(q, k, v, SCALE, q_starts=starts, k_starts=starts)
    assert torch.equal(got[:, :, :last], v.repeat_interleave(2, 1)[:, :, :last]) and not got[:, :, last:].any()
    with pytest.raises(ValueError, match="at most 65536"):
        more = torch.zeros(n + 2, dtype=torch.int32, device=device)
        prompt_attention(q, k, v, SCALE, q_starts=more, k_starts=more)
