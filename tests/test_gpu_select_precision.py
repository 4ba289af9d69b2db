"""What tp_selected_attention keeps that one fp16 number for a key, a value or a weight would lose: each test's inputs make
that loss more than the bound (4 to 12 times it, but 1.13 for the keys of deep2 and 12 heads, whose few angles all have
cosines of one size), which is asserted of the oracle with the rounding planted in it.

Against float64 over the pages' own codes: angles in fp32 as the decoder's contract has them, radii, cosines and products
in float64, values code times scale exactly."""

import numpy as np
import pytest
import torch

from common import LAYOUTS, PAGE, rel_l2
from oracle import turbopolar as oracle
from test_gpu_select import bridge_call
from test_gpu_tree import config
from turbopolar_amd import TurboPolarFastCache
from turbopolar_amd.kernels import fp16_scale

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -11
F16 = np.float16


def filled(device, layout, hq, hkv, k, v):
    cache = TurboPolarFastCache(config(layout, hq, hkv))
    cache.runtime.append(torch.from_numpy(k).to(device), torch.from_numpy(v).to(device))
    return cache


def exact_pages(cache):
    """Keys and values of the stored pages, and both as one fp16 number each: a key the product of a rounded radius and
    a rounded cosine."""
    key, value, *_ = cache.runtime.get_fused_attention_inputs()
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    norm = oracle._angle_norms(host(key.angle_codes_l1), host(key.angle_codes_deep), key.metadata, 128)
    angle = (norm * oracle.F32_TWO_PI - oracle.F32_PI).astype(np.float64)
    r = host(key.radii).astype(np.float64)
    if key.radii_scales is not None:
        r = np.exp(r * host(key.radii_scales).astype(np.float64).reshape(*r.shape[:3], 1, 1))
    cs = np.stack([np.cos(angle), np.sin(angle)], -1)
    shape = (*r.shape[:2], -1, 128)
    one = r.astype(F16)[..., None] * cs.astype(F16)
    codes, scales = host(value.codes).astype(np.float64).reshape(shape), host(value.scales).astype(np.float64)
    v = codes * np.repeat(scales.reshape(*shape[:2], -1, 4), 32, axis=-1)
    return [(r[..., None] * cs).reshape(shape), v], [one.astype(np.float64).reshape(shape), v.astype(F16).astype(np.float64)]


def attended(q, k, v, selected, scale16):
    """The result, its weights and the scores' products, one batch row."""
    g = q.shape[1] // k.shape[1]
    out, weights, sizes = [], [], []
    for h in range(q.shape[1]):
        at = (selected[0, h // g][:, None] * PAGE + np.arange(PAGE)).ravel()
        keys = k[0, h // g, at]
        s = keys @ q[0, h].astype(np.float64) * scale16
        w = np.exp(s - s.max())
        w /= w.sum()
        out.append(w @ v[0, h // g, at])
        weights.append(w)
        sizes.append(abs(scale16) * np.sqrt((keys ** 2 @ q[0, h].astype(np.float64) ** 2).max()))
    return np.array(out), weights, max(sizes)


def run(device, cache, q, n):
    out, selected = bridge_call(cache, torch.from_numpy(q).to(device), cache.runtime.page_bounds(), n, 0, 0)
    return out[0].double().cpu().numpy(), selected.cpu().numpy()


SHAPES = [(layout, g) for layout in sorted(LAYOUTS) for g in (4, 12)]  # query heads a kv head: at most 8 and more


@pytest.mark.parametrize("layout,g", SHAPES)
def test_keys_in_two_parts(device, layout, g):
    """Neighbouring pairs of a key are of one angle and of radii within 5 % of each other, and a query's of opposite
    signs: a score is the small difference of large products, whose roundings do not cancel.

    Relative L2: weights, records and the result are rounded once, each error uniform in half a step, which is at most
    2^-11 of the value: 2^-11 / sqrt(3) each, 2^-11 together.  A key is off by 2^-21 of itself, a score by the root of the
    products' squares times that, a weight by twice as much (its own and the sum's)."""
    hkv, pages, n = 2, 24, 16
    rng = np.random.default_rng(g)
    r = 8 * np.exp(rng.uniform(-0.05, 0.05, (1, hkv, pages * PAGE, 32, 2)))
    a = rng.uniform(-np.pi, np.pi, (1, hkv, pages * PAGE, 32, 1))
    k = np.stack([r * np.cos(a), r * np.sin(a)], -1).reshape(1, hkv, pages * PAGE, 128).astype(F16)
    v = rng.standard_normal(k.shape).astype(F16)
    x = 4 * rng.standard_normal((1, hkv * g, 32, 1, 2))
    q = np.concatenate([x, -x], 3).reshape(1, hkv * g, 128).astype(F16)
    cache = filled(device, layout, hkv * g, hkv, k, v)
    scale = fp16_scale(cache.config.attention_scale)
    got, selected = run(device, cache, q, n)
    (k64, v64), (k_one, _) = exact_pages(cache)
    want, _, size = attended(q, k64, v64, selected, scale)
    planted = rel_l2(attended(q, k_one, v64, selected, scale)[0], want)
    bound = EPS + 2 * 2.0 ** -21 * size
    off = rel_l2(got, want)
    print(f"[precision] keys {layout} g={g}: {off:.3g} of {bound:.3g}, one part {planted:.3g}", flush=True)
    assert planted > bound and off <= bound


@pytest.mark.parametrize("layout,g", SHAPES)
def test_values_in_two_parts(device, layout, g):
    """A query of zeros weighs all tokens alike, and every other one's values are the others' negated, 1.003 times as
    large: the mean is 0.0015 of them, and their roundings do not cancel.

    An element is rounded twice at most (a record and the result, 2^-11 of itself each); the sums are of two products a
    token, each addition off by at most 2^-23 of the values' mean size."""
    hkv, n = 2, 2
    rng = np.random.default_rng(g)
    x = rng.uniform(0.5, 1.5, (1, hkv, 1, 128)) * rng.choice([-1, 1], (1, hkv, 1, 128))
    v = np.where(np.arange(3 * PAGE)[:, None] % 2, -1.003 * x, x).astype(F16)
    k = rng.standard_normal(v.shape).astype(F16)
    cache = filled(device, layout, hkv * g, hkv, k, v)
    got, selected = run(device, cache, np.zeros((1, hkv * g, 128), F16), n)
    assert (selected == np.arange(n)).all()
    (_, v64), (_, v_one) = exact_pages(cache)
    mean = lambda x: np.repeat(x[0, :, :n * PAGE].mean(1), g, axis=0)  # noqa: E731
    want = mean(v64)
    bound = 2 * EPS * np.abs(want) + (2 * n * PAGE + 16) * 2.0 ** -23 * mean(np.abs(v64))
    off, planted = np.abs(got - want), np.abs(mean(v_one) - want)
    print(f"[precision] values {layout} g={g}: {(off / bound).max():.3g} of the bound, one part {(planted / bound).max():.3g}",
          flush=True)
    assert (planted > bound).mean() > 0.5 and np.all(off <= bound)


@pytest.mark.parametrize("layout,g", SHAPES)
def test_small_weights(device, layout, g):
    """A page's first token takes nearly all of the weight and has values of 0; the others weigh 2^-28 of it, which is
    0 in fp16 (half its smallest step is 2^-25), and give the whole result.

    Weights are held times 2^7: each is off by half a step of 2^-24, 2^-32 of the first token's; a record and the result
    are rounded once; a score as in the keys' test."""
    hkv, n = 2, 4
    rng = np.random.default_rng(g)
    k = np.zeros((1, hkv, 6 * PAGE, 128), F16)
    k[:, :, ::PAGE] = rng.uniform(1, 2, (1, hkv, 1, 128)).astype(F16)
    v = rng.uniform(500, 1500, k.shape).astype(F16)
    v[:, :, ::PAGE] = 0
    cache = filled(device, layout, hkv * g, hkv, k, v)
    scale = fp16_scale(cache.config.attention_scale)
    (k64, v64), _ = exact_pages(cache)
    q = np.repeat(k64[:, :, 0], g, axis=1) * rng.uniform(0.5, 1.5, (1, hkv * g, 128))
    of_first = np.einsum("bhd,bhd->bh", q, np.repeat(k64[:, :, 0] - k64[:, :, 1], g, axis=1)) * scale
    q = (q * (28 * np.log(2) / of_first)[..., None]).astype(F16)
    got, selected = run(device, cache, q, n)
    want, weights, size = attended(q, k64, v64, selected, scale)
    top = max(w.max() for w in weights)
    small = np.array([w[w < top / 2] for w in weights]) / top
    assert small.shape[1] == n * (PAGE - 1) and 2.0 ** -29 < small.min() and small.max() < 2.0 ** -27
    bound = n * (PAGE - 1) * 2.0 ** -32 * top * v64.max() + (2 * EPS + np.expm1(2 * 2.0 ** -21 * size) + 2.0 ** -14) * want
    print(f"[precision] weights {layout} g={g}: {(np.abs(got - want) / bound).max():.3g} of the bound, "
          f"without the factor {(want / bound).min():.3g}", flush=True)
    assert np.all(want > 4 * bound) and np.all(np.abs(got - want) <= bound)
