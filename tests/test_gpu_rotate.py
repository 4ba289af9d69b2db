"""Rotated appends (tp_rotate_tokens) against the rotation in float64, and the caches they fill.

A result is the rounding of the exact sum x_a cos_a -+ x_b sin_a to fp32 and then to fp16.  Products of 24-bit
numbers are exact in float64 and their sum is rounded there by 2^-53, so float64 -> float32 -> float16 gives the same
number but where that rounding moves an fp32 tie (2^-29 of the cases): results are compared bit for bit.  Against
the exact value they are off by half an fp16 step (2^-11 of the value, 2^-25 below the normal range) and half an
fp32 step."""

import numpy as np
import pytest
import torch

from common import LAYOUTS, PAGE
from turbopolar_amd import TurboPolarConfig, TurboPolarFastCache
from turbopolar_amd.kernels import rotate_tokens

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def config(layout="default", hq=8, hkv=2):
    int8, l1, deep, split = LAYOUTS[layout]
    return TurboPolarConfig(num_q_heads=hq, num_kv_heads=hkv, use_int8_radii=int8, k_angle_bits_level1=l1,
                            k_angle_bits_deep=deep, split_dim=split)


def tables(device, start, T, columns, interleaved, dtype, batch=None):
    at = torch.arange(start, start + T, dtype=torch.float64)
    if batch:
        at = at + 17 * torch.arange(batch, dtype=torch.float64)[:, None]
    angle = at[..., None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    if columns == 128:
        angle = angle.repeat_interleave(2, -1) if interleaved else torch.cat((angle, angle), -1)
    return angle.cos().to(dtype).to(device), angle.sin().to(dtype).to(device)


def draw(device, B, hq, hkv, T, dtype, seed, spread=2.0):
    """Queries, keys and values as projections leave them, token by token; the channels' sizes spread by e^spread."""
    g = torch.Generator(device=device).manual_seed(seed)

    def one(h):
        x = torch.randn((B, T, h, 128), generator=g, device=device)
        return (x * torch.exp(spread * torch.randn((128,), generator=g, device=device))).to(dtype).transpose(1, 2)

    return one(hq), one(hkv), one(hkv)


def turned64(x, cos, sin, interleaved):
    """[B, H, T, 128] turned in float64."""
    x, c, s = (t.double().cpu().numpy() for t in (x, cos, sin))
    if c.ndim == 2:
        c, s = c[None], s[None]
    if c.shape[-1] == 64:
        c, s = ((np.repeat(t, 2, -1) if interleaved else np.concatenate((t, t), -1)) for t in (c, s))
    c, s = c[:, None], s[:, None]
    y = np.empty(x.shape)
    a, b = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, 64), slice(64, 128))
    y[..., a] = x[..., a] * c[..., a] - x[..., b] * s[..., a]
    y[..., b] = x[..., b] * c[..., b] + x[..., a] * s[..., b]
    return y


def check(got, want64, what):
    with np.errstate(over="ignore"):
        want = want64.astype(np.float32).astype(np.float16)
    assert got.dtype is torch.float16
    got = got.cpu().numpy()
    assert np.array_equal(got, want), (what, int((got != want).sum()))
    # And against the exact value.
    off = np.abs(got.astype(np.float64) - want64)
    assert np.all(off <= np.abs(want64) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25), what


@pytest.mark.parametrize("dtype,table", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("columns", [128, 64])
def test_rotation(device, dtype, table, interleaved, columns):
    """One token, an odd number of them, and many; one table for all rows and one each; the largest positions."""
    for B, hq, hkv, T, start, own in ((1, 32, 8, 1, 299, False), (3, 5, 5, 7, 131071, True), (2, 28, 4, 130, 0, False),
                                      (1, 1, 1, 3, 10 ** 6, False), (5, 40, 2, 1, 0, True)):
        print(f"[rotate] {dtype} {table} {interleaved} {columns} {B} {hq} {hkv} {T}", flush=True)
        q, k, v = draw(device, B, hq, hkv, T, TYPES[dtype], seed=T + B)
        cos, sin = tables(device, start, T, columns, interleaved, TYPES[table], B if own else None)
        q16, k16, v16 = rotate_tokens(q, k, v, cos, sin, interleaved)
        check(q16, turned64(q, cos, sin, interleaved), "q")
        check(k16, turned64(k, cos, sin, interleaved), "k")
        assert torch.equal(v16, v.half())
        assert k16.is_contiguous() and v16.is_contiguous() and q16.transpose(1, 2).is_contiguous()


def test_unequal_columns_and_other_table_types(device):
    """Each of 128 columns is used for its own dimension; tables of a third type are taken in float32."""
    q, k, v = draw(device, 2, 4, 2, 9, torch.float16, 1)
    cos, sin = (torch.randn(9, 128, device=device).bfloat16() for _ in range(2))
    for inter in (False, True):
        q16, k16, _ = rotate_tokens(q, k, v, cos, sin, inter)
        check(q16, turned64(q, cos, sin, inter), "q")
        check(k16, turned64(k, cos, sin, inter), "k")


def test_strides(device):
    """Slices of one projection, padded rows, broadcast and misaligned inputs, tables out of a larger one."""
    B, hq, hkv, T = 2, 6, 3, 5
    g = torch.Generator(device=device).manual_seed(3)
    both = torch.randn((B, T, (hq + 2 * hkv) * 128 + 8), generator=g, device=device).half()
    q = both[..., : hq * 128].view(B, T, hq, 128).transpose(1, 2)
    k = both[..., hq * 128:(hq + hkv) * 128].view(B, T, hkv, 128).transpose(1, 2)
    v = both[..., (hq + hkv) * 128:(hq + 2 * hkv) * 128].view(B, T, hkv, 128).transpose(1, 2)
    cos, sin = tables(device, 40, 64, 128, False, torch.float32)
    rows = torch.arange(3, 3 + T)
    for name, args in {
        "slices": (q, k, v, cos[3:3 + T], sin[3:3 + T]),
        "copies": (q.contiguous(), k.contiguous(), v.contiguous(), cos[rows], sin[rows].clone()),
        "broadcast": (q, k[:, :1].expand(-1, hkv, -1, -1), v[:1].expand(B, -1, -1, -1), cos[None, 3:3 + T], sin[None, 3:3 + T]),
        "one table row": (q, k, v, cos[:1].expand(T, -1), sin[:1].expand(T, -1)),
        "unlike tables": (q, k, v, cos[3:3 + T], sin.t().contiguous().t()[3:3 + T]),
        "misaligned": tuple(torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape).copy_(t) for t in (
            q, k, v, cos[3:3 + T], sin[3:3 + T])),
        "dims reversed": (q.flip(3).flip(3).contiguous().transpose(2, 3).contiguous().transpose(2, 3), k, v, cos[3:3 + T],
                          sin[3:3 + T]),
    }.items():
        q16, k16, v16 = rotate_tokens(*args)
        check(q16, turned64(args[0], args[3], args[4], False), name)
        check(k16, turned64(args[1], args[3], args[4], False), name)
        assert torch.equal(v16, args[2]), name
    assert rotate_tokens(q[:, :, :0], k[:, :, :0], v[:, :, :0], cos[:0], sin[:0])[0].shape == (B, hq, 0, 128)


def contents(cache):
    rt = cache.runtime
    key, value, tail_k, tail_v, _, n = rt.get_fused_attention_inputs()
    out = [n, rt.get_io_telemetry()]
    if key is not None:
        out += [key.radii, key.radii_scales, key.angle_codes_l1, key.angle_codes_deep, value.codes, value.scales]
    return out + [tail_k, tail_v]


def bits(t):
    """Bit patterns: keys past 256 overflow the codec's fp16 squares, and their pages hold infinities and NaN."""
    return t.view(torch.int16) if t.dtype is torch.float16 else t


def same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert torch.equal(bits(x), bits(y)) if isinstance(x, torch.Tensor) else x == y


@pytest.mark.parametrize("layout", ["default", "fast", "odd_split"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_appends(device, layout, dtype):
    """Appends of one token to several pages, into a new cache, up to a full page and past it: what the cache holds is
    what an append of the turned keys leaves, bit for bit, and updates return the same history."""
    for B in (1, 3):
        one, two = (TurboPolarFastCache(config(layout)) for _ in range(2))
        start = 0
        for i, T in enumerate((1, 5, 57, 1, 1, 63, 64, 1, 200, 7, 130)):
            q, k, v = draw(device, B, 8, 2, T, TYPES[dtype], seed=100 * B + i)
            cos, sin = tables(device, start, T, 128, bool(i & 1), torch.float32)
            q16, k16, v16 = rotate_tokens(q, k, v, cos, sin, bool(i & 1))
            assert torch.equal(one.append_rotated(q, k, v, cos, sin, bool(i & 1)), q16)
            two.runtime.append(k16, v16)
            start += T
            same(contents(one), contents(two))
        q, k, v = draw(device, B, 8, 2, 70, TYPES[dtype], seed=9)
        cos, sin = tables(device, start, 70, 64, False, torch.float32)
        got = one.update_rotated(q, k, v, cos, sin)
        q16, k16, v16 = rotate_tokens(q, k, v, cos, sin)
        same(got, (q16, *two.update_and_fetch(k16, v16)))
        same(contents(one), contents(two))


def test_batches_with_more_tokens_than_report_lines(device):
    """The verdict of a launch of many workgroups, with and without a line for each."""
    for B, T in ((64, 1), (2, 60), (1, 33), (40, 7)):
        cache = TurboPolarFastCache(config())
        q, k, v = draw(device, B, 8, 2, T, torch.float16, B)
        cos, sin = tables(device, 0, T, 128, False, torch.float16)
        cache.append_rotated(q, k, v, cos, sin)
        assert torch.equal(cache.runtime.partial_k, rotate_tokens(q, k, v, cos, sin)[1])
        held = cache.runtime.partial_k
        at = (B - 1, 1, T - 1, 100)
        bad = v.clone()
        bad[at] = float("inf")
        for _ in range(2):
            with pytest.raises(ValueError, match="finite"):
                cache.append_rotated(q[:, :, -1:], k[:, :, -1:], bad[:, :, -1:], cos[-1:], sin[-1:])
            assert cache.offset == T and torch.equal(cache.runtime.partial_k, held)
            cache.append_rotated(q[:, :, -1:], k[:, :, -1:], v[:, :, -1:], cos[-1:], sin[-1:])
            cache.truncate(T)


@pytest.mark.parametrize("T", [1, 40, 150])
def test_refused_appends_leave_the_cache(device, T):
    """Keys that a rotation or the cast takes past fp16, NaN and infinities, in a new cache and in a filled one."""
    for filled in (0, 30):
        cache = TurboPolarFastCache(config())
        if filled:
            cache.runtime.append(*(t.contiguous() for t in draw(device, 2, 8, 2, filled, torch.float16, 5)[1:]))
        before = contents(cache)
        q, k, v = draw(device, 2, 8, 2, T, torch.float32, 6)
        cos, sin = tables(device, filled, T, 128, False, torch.float32)
        for name, value in (("k", float("nan")), ("k", 1e5), ("k", float("-inf")), ("v", float("nan")), ("v", 7e4)):
            x = {"k": k.clone(), "v": v.clone()}
            x[name][1, 1, T - 1, 70] = value
            x[name][1, 1, T - 1, 6] = value
            with pytest.raises(ValueError, match="finite"):
                cache.append_rotated(q, x["k"], x["v"], cos, sin)
            assert cache.offset == filled
            if filled:
                same(contents(cache), before)
        with pytest.raises(ValueError, match="KV head"):
            cache.append_rotated(q, k[:, :1], v[:, :1], cos, sin)
        if filled:
            with pytest.raises(ValueError, match="batch size changed"):
                cache.append_rotated(q[:1], k[:1], v[:1], cos, sin)
        q[0, 0, 0, 0] = float("nan")  # queries are not checked, as decode_attention does not
        cache.append_rotated(q, k, v, cos, sin)
        assert cache.offset == filled + T


def test_float32_caches_and_gradients_are_refused(device):
    cache = TurboPolarFastCache(config())
    q, k, v = draw(device, 1, 8, 2, 3, torch.float32, 1)
    cos, sin = tables(device, 0, 3, 128, False, torch.float32)
    cache.runtime.append(k.contiguous(), v.contiguous())
    with pytest.raises(ValueError, match="dtype changed"):
        cache.append_rotated(q, k, v, cos, sin)
    fresh = TurboPolarFastCache(config())
    with pytest.raises(ValueError, match="no gradients"):
        fresh.append_rotated(q.requires_grad_(), k, v, cos, sin)
    with pytest.raises(ValueError, match="at least one token"):
        fresh.append_rotated(q[:, :, :0].detach(), k[:, :, :0], v[:, :, :0], cos[:0], sin[:0])
    assert fresh.offset == 0


def test_decode_rotated(device):
    """A rotated step is decode_attention of the turned token, with its verdict now or later."""
    one, two = (TurboPolarFastCache(config("fast", 32, 8)) for _ in range(2))
    scale = one.config.attention_scale
    for i in range(70):
        q, k, v = draw(device, 1, 32, 8, 1, torch.bfloat16, seed=i)
        cos, sin = tables(device, i, 1, 128, False, torch.bfloat16)
        got = one.decode_rotated(q, k, v, cos, sin, scale, defer_check=bool(i % 3))
        q16, k16, v16 = rotate_tokens(q, k, v, cos, sin)
        same([got], [two.decode_attention(q16, k16, v16, scale)])
    one.runtime.resolve_deferred_check()
    same(contents(one), contents(two))
    with pytest.raises(NotImplementedError, match="batch size 1"):
        one.decode_rotated(q.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1), cos, sin, scale)


def test_streams_and_graphs(device):
    """On another stream; captured and replayed over changing inputs."""
    q, k, v = draw(device, 2, 8, 2, 5, torch.float16, 8)
    cos, sin = tables(device, 0, 5, 128, False, torch.float16)
    want = rotate_tokens(q, k, v, cos, sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotate_tokens(q, k, v, cos, sin)
        cache = TurboPolarFastCache(config())
        cache.append_rotated(q, k, v, cos, sin)
    side.synchronize()
    same(got, want)
    assert torch.equal(cache.runtime.partial_k, want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotate_tokens(q, k, v, cos, sin)
    for seed in (11, 12, 13):
        for t, new in zip((q, k, v), draw(device, 2, 8, 2, 5, torch.float16, seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        same(out, rotate_tokens(q, k, v, cos, sin))
