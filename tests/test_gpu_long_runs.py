"""Prompts and drafted trees of many workgroups: what the small cases of test_gpu_prompt.py and
test_gpu_tree.py leave out, with their bounds.

* The 256-row prompt kernel, which is chosen where its workgroups fill the GPU: thousands of rows, long runs of
  keys, causal and not, packed, with what is masked not finite.
* Trees whose workgroups take several pages each, the last one fewer: 64 (batch, head) rows share the GPU."""

import numpy as np
import pytest
import torch

import oracle
from common import ATOL, RTOL_L2, rel_l2
from test_gpu_prompt import BF16, F16, SCALE, close, make, reference, starts_of
from test_gpu_tree import EPS, draft, filled, random_parents
from turbopolar_amd import DraftTree
from turbopolar_amd.kernels import fp16_scale, prompt_attention

pytestmark = pytest.mark.gpu

LONG = [
    # B, hq, hkv, tq, tk: units x ceil(tq hq / hkv / 256) is 256 or more in each
    (1, 32, 8, 2111, 2111), (1, 28, 4, 2400, 2400), (4, 8, 8, 2049, 2049), (1, 32, 8, 2060, 3333), (2, 16, 16, 2100, 130),
    (16, 4, 4, 1100, 1100),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", LONG)
def test_long_prompts(device, shape, causal, dtype):
    q, k, v = make(device, dtype, *shape, seed=sum(shape))
    close(prompt_attention(q, k, v, SCALE, causal=causal), *reference(q, k, v, SCALE, causal), f"{shape} {causal} {dtype}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_long_packed(device, dtype, causal):
    """Sequences of many tiles beside ones of a token, an empty one, and rows behind the last."""
    lengths, rest = [700, 3, 1200, 1, 0, 131], 80
    starts = starts_of(lengths)
    q, k, v = make(device, dtype, 1, 32, 8, starts[-1] + rest, starts[-1] + rest, seed=5)
    k[:, :, starts[-1]:], v[:, :, starts[-1]:] = float("nan"), float("inf")
    want, tol = torch.zeros(q.shape, dtype=torch.float64, device=device), torch.zeros_like(q, dtype=torch.float64)
    for a, b in zip(starts, starts[1:]):
        want[:, :, a:b], tol[:, :, a:b] = reference(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], SCALE, causal)
    got = prompt_attention(q, k, v, SCALE, causal=causal, q_starts=starts, k_starts=starts)
    close(got, want, tol, f"packed {causal} {dtype}")
    assert not got[:, :, starts[-1]:].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("at", [0, 63, 1500, 2110])
def test_long_prompts_keep_what_is_masked_out(device, at, bad, dtype):
    """An infinite or NaN value at one key reaches the queries that see it, in its dimension alone; keys that are NaN
    from there on reach none before."""
    q, k, v = make(device, dtype, 1, 32, 8, 2111, 2111, seed=6)
    want, tol = reference(q, k, v, SCALE, True)
    v2 = v.clone()
    v2[:, :, at, 5] = bad
    got = prompt_attention(q, k, v2, SCALE)
    assert not torch.isfinite(got[:, :, at:, 5]).any()
    others = [d for d in range(128) if d != 5]
    close(got[..., others], want[..., others], tol[..., others], "other dimensions")
    close(got[:, :, :at], want[:, :, :at], tol[:, :, :at], "before")
    k2 = k.clone()
    k2[:, :, at:] = bad
    close(prompt_attention(q, k2, v, SCALE)[:, :, :at], want[:, :, :at], tol[:, :, :at], "before, keys")


def unit_history(rt, b, h):
    """Every token held of one (batch, head) row in float64: the oracle's decode of its pages, and the tail."""
    S, ks, vs = rt.k_storage.block_count, rt.k_storage, rt.v_storage
    host = lambda t: None if t is None else t[b:b + 1, h:h + 1, :S].cpu().numpy()  # noqa: E731
    k = oracle.decode_block(host(ks.radii), host(ks.radii_scales), host(ks.angle_codes_l1), host(ks.angle_codes_deep),
                            ks.metadata)[0, 0]
    v = oracle.dequantize_block(host(vs.codes)[:, :, :, 0], host(vs.scales)[:, :, :, 0])[0, 0].reshape(k.shape)
    tail = lambda t: t[b, h, : rt._tail_len].cpu().numpy()  # noqa: E731
    return (np.concatenate((k, tail(rt._tail_k))).astype(np.float64), np.concatenate((v, tail(rt._tail_v))).astype(np.float64))


PAGES = 41
# Nodes of four heads a group: rows 32, 64, 128, 256, and 320 in two blocks; 3, 6, 6 or 11, and 11 pages a workgroup.
@pytest.mark.parametrize("n", [8, 16, 32, 64, 80])
@pytest.mark.parametrize("layout", ["default", "fast", "deep2", "l1_8bit", "odd_split"])
def test_trees_of_many_pages_a_workgroup(device, layout, n):
    B, hkv, g, tokens = 8, 8, 4, 64 * PAGES + 20
    print(f"[tree] {layout} {n} nodes", flush=True)
    cache = filled(device, layout, B, hkv * g, hkv, tokens, seed=n, kind="loguniform")
    q, dk, dv = draft(device, B, hkv * g, hkv, n, seed=n)
    tree = DraftTree(random_parents(n, n))
    scale = fp16_scale(cache.config.attention_scale)
    got = cache.tree_attention(q, dk, dv, tree, cache.config.attention_scale).double().cpu().numpy()
    assert np.isfinite(got).all()
    seen = np.zeros((n, n), dtype=bool)
    for i in range(n):
        seen[i, tree.path_to(i)] = True
    for b, h in [(0, 0), (3, 5), (7, 7)]:
        k, v = unit_history(cache.runtime, b, h)
        k = np.concatenate((k, dk[b, h].double().cpu().numpy()))
        v = np.concatenate((v, dv[b, h].double().cpu().numpy()))
        q64 = q[b, h * g:(h + 1) * g].double().cpu().numpy().reshape(g * n, 128)
        s = q64 @ k.T * scale
        s[:, tokens:][~np.tile(seen, (g, 1))] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want, mine = p @ v, got[b, h * g:(h + 1) * g].reshape(g * n, 128)
        off = np.abs(mine - want)
        print(f"[tree] ({b}, {h}): max-abs {off.max():.3g}, rel L2 {rel_l2(mine, want):.3g}", flush=True)
        assert np.all(off <= ATOL + EPS * np.abs(want)) and rel_l2(mine, want) <= RTOL_L2
