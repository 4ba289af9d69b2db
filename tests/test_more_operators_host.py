"""Rotated appends, shared prefixes and selected pages: what their entry points refuse, and the bookkeeping that
needs no GPU."""

import ctypes

import pytest
import torch

from turbopolar_amd import SharedPrefixCache, TurboPolarConfig, TurboPolarFastCache, _lib
from turbopolar_amd.kernels import check_selection, rotate_tokens

P = 4096  # aligned, never dereferenced: validation fails before any device access
NAN = float("nan")


def pages(capacity=8):
    return _lib.TPPages(P, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P, capacity)


DEFAULT = _lib.make_layout(False, 4, 4, 64)


def rotate(**kw):
    a = dict(q=P, k=P, v=P, dtype=0, batch=1, hq=4, hkv=2, tokens=3, strides=[0] * 9, cos=P, sin=P, table=0, columns=128,
             tstrides=[0, 128], inter=0, q_out=P, ostrides=[1536, 128, 512], k_out=P, v_out=P, out_tokens=64, pos=0,
             check=0, flag=None, words=0, epoch=0)
    a.update(kw)
    array = lambda x: None if x is None else (ctypes.c_int64 * len(x))(*x)  # noqa: E731
    st = _lib.lib().tp_rotate_tokens(
        a["q"], a["k"], a["v"], a["dtype"], a["batch"], a["hq"], a["hkv"], a["tokens"], array(a["strides"]), a["cos"],
        a["sin"], a["table"], a["columns"], array(a["tstrides"]), a["inter"], a["q_out"], array(a["ostrides"]), a["k_out"],
        a["v_out"], a["out_tokens"], a["pos"], a["check"], a["flag"], a["words"], a["epoch"], None)
    return st, _lib.lib().tp_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(table=2), "dtype"), (dict(dtype=1, table=0), "dtype"),
    (dict(batch=0), "shape"), (dict(hq=0), "shape"), (dict(hkv=0), "shape"), (dict(tokens=-1), "shape"),
    (dict(batch=2 ** 30, tokens=3), "2\\^31"), (dict(columns=32), "columns"), (dict(columns=256), "columns"),
    (dict(pos=62), "do not fit"), (dict(pos=-1), "do not fit"), (dict(out_tokens=2), "do not fit"),
    (dict(check=2), "check"), (dict(check=1, flag=P, words=16), "check"), (dict(check=2, flag=P, words=16, epoch=3), "check"),
    (dict(check=2, flag=P, words=0, epoch=2), "check"), (dict(q=None), "aligned"), (dict(v=P + 8), "aligned"),
    (dict(sin=P + 2), "aligned"), (dict(k_out=None), "aligned"), (dict(strides=None), "strides"),
    (dict(tstrides=None), "strides"), (dict(ostrides=None), "strides"), (dict(strides=[4] + [0] * 8), "multiples"),
    (dict(strides=[-8] + [0] * 8), "multiples"), (dict(tstrides=[0, 12]), "multiples"), (dict(ostrides=[0, 4, 8]), "multiples"),
])
def test_rotate_refusals(change, message):
    import re

    st, text = rotate(**change)
    assert st == _lib.TP_ERR_INVALID and re.search(message, text), (st, text)


def test_rotate_of_no_tokens():
    assert rotate(tokens=0)[0] == _lib.TP_OK


def shared(**kw):
    a = dict(q=P, out=P, batch=2, hq=4, hkv=2, layout=DEFAULT, prefix=pages(), prefix_pages=4, ptk=None, ptv=None,
             prefix_tail=0, pstride=0, pages=pages(), n_pages=2, tk=None, tv=None, tail=0, tstride=0,
             strides=[512, 128, 512, 128], scale=0.1, ws=None, wsb=0)
    a.update(kw)
    s = a["strides"]
    st = _lib.lib().tp_shared_attention(
        a["q"], a["out"], a["batch"], a["hq"], a["hkv"], ctypes.byref(a["layout"]), ctypes.byref(a["prefix"]),
        a["prefix_pages"], a["ptk"], a["ptv"], a["prefix_tail"], a["pstride"], ctypes.byref(a["pages"]), a["n_pages"],
        a["tk"], a["tv"], a["tail"], a["tstride"], None if s is None else (ctypes.c_int64 * 4)(*s), a["scale"], a["ws"],
        a["wsb"], None)
    return st, _lib.lib().tp_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(hq=5), "multiple"), (dict(batch=0), "shape"), (dict(hkv=0), "shape"), (dict(batch=2 ** 40), "shape"),
    (dict(prefix_pages=9), "prefix: n_pages"), (dict(n_pages=9), "own tokens: n_pages"), (dict(n_pages=-1), "own tokens"),
    (dict(prefix=_lib.TPPages(P, None, P, P, None, P, 8)), "prefix: page buffers missing"),
    (dict(pages=_lib.TPPages(P + 8, None, P, P, P, P, 8)), "own tokens: page buffers are not aligned"),
    (dict(prefix_tail=64, ptk=P, ptv=P, pstride=64), "prefix: tail_len"), (dict(tail=3, tk=P, tv=P, tstride=2), "tail buffers"),
    (dict(tail=3, tk=None, tv=P, tstride=64), "tail buffers"), (dict(prefix_tail=3, ptk=P + 8, ptv=P, pstride=64), "tail buffers"),
    (dict(prefix_pages=0, n_pages=0), "nothing to attend"), (dict(q=None), "q and out"), (dict(out=P + 8), "q and out"),
    (dict(strides=None), "strides"), (dict(strides=[512, 100, 512, 128]), "multiples"), (dict(scale=NAN), "finite"),
    (dict(scale=float("inf")), "finite"),
])
def test_shared_refusals(change, message):
    st, text = shared(**change)
    assert st == _lib.TP_ERR_INVALID and message in text, (st, text)


def test_shared_layout_and_workspace():
    assert shared(layout=_lib.make_layout(False, 3, 4, 64))[0] == _lib.TP_ERR_UNSUPPORTED
    st, text = shared()
    assert st == _lib.TP_ERR_WORKSPACE and "workspace" in text
    size = _lib.lib().tp_shared_workspace_bytes
    lay = ctypes.byref(DEFAULT)
    assert size(2, 4, 2, lay, 0, 5, 0, 0) == 0  # one tile: one record, none kept
    assert size(2, 4, 2, lay, 4, 0, 2, 0) > 0
    assert size(0, 4, 2, lay, 4, 0, 2, 0) == 0 and size(2, 5, 2, lay, 4, 0, 2, 0) == 0
    # Every shape's records: what a row takes times the tiles at most.
    for batch, hq, hkv, prefix, own in ((1, 1, 1, 1, 1), (64, 64, 8, 500, 8), (3, 28, 4, 2048, 0), (7, 40, 2, 0, 100)):
        assert size(batch, hq, hkv, lay, prefix, 0, own, 9) <= batch * hq * (prefix + own + 1) * 264


def select(**kw):
    a = dict(q=P, batch=1, hq=4, hkv=2, bounds=P, cap=8, n=8, first=1, last=1, count=4, scale=0.1, out=P, ws=P, wsb=65536 + 128)
    a.update(kw)
    st = _lib.lib().tp_select_pages(a["q"], a["batch"], a["hq"], a["hkv"], a["bounds"], a["cap"], a["n"], a["first"],
                                    a["last"], a["count"], a["scale"], a["out"], a["ws"], a["wsb"], None)
    return st, _lib.lib().tp_last_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(hq=5), "multiple"), (dict(batch=0), "shape"), (dict(batch=40000), "65535"), (dict(n=0), "n_pages"),
    (dict(n=9), "n_pages"), (dict(count=0, first=0, last=0), "cannot select"), (dict(count=9), "cannot select"),
    (dict(first=-1), "cannot select"), (dict(last=-1), "cannot select"), (dict(first=3, last=2), "cannot select"),
    (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), "cannot select"), (dict(scale=NAN), "finite"), (dict(q=None), "non-NULL"),
    (dict(bounds=P + 8), "non-NULL"), (dict(out=None), "non-NULL"), (dict(out=P + 2), "non-NULL"),
])
def test_select_refusals(change, message):
    st, text = select(**change)
    assert st == _lib.TP_ERR_INVALID and message in text, (st, text)


def test_select_workspace():
    assert select(wsb=65536 + 127)[0] == select(ws=None)[0] == select(ws=P + 8)[0] == _lib.TP_ERR_WORKSPACE
    size = _lib.lib().tp_select_workspace_bytes
    assert size(1, 4, 2, 8) == 65536 + 128 and size(0, 4, 2, 8) == 0 and size(3, 10, 5, 100) == 65536 + 12000


def test_bounds_refusals():
    f, lay = _lib.lib().tp_page_bounds, ctypes.byref(DEFAULT)
    p = ctypes.byref(pages())
    assert f(ctypes.byref(_lib.make_layout(False, 4, 3, 64)), p, 2, 0, 4, P, 8, None) == _lib.TP_ERR_UNSUPPORTED
    assert f(lay, p, 2, 0, 0, None, 0, None) == _lib.TP_OK
    bad = [(0, 0, 4, P, 8), (70000, 0, 4, P, 8), (2, -1, 4, P, 8), (2, 0, -1, P, 8), (2, 5, 4, P, 16), (2, 0, 4, P, 3),
           (2, 0, 4, None, 8), (2, 0, 4, P + 8, 8), (2, 2 ** 31 - 1, 4, P, 8)]
    for bh, begin, n, out, cap in bad:
        assert f(lay, p, bh, begin, n, out, cap, None) == _lib.TP_ERR_INVALID, (bh, begin, n, out, cap)
    int8 = ctypes.byref(_lib.make_layout(True, 4, 8, 0))
    assert f(int8, ctypes.byref(_lib.TPPages(P, None, None, P, None, None, 8)), 2, 0, 4, P, 8, None) == _lib.TP_ERR_INVALID


def test_selected_attention_refusals():
    def call(selected=P, count=3, n=4, scale=0.1, out=P, store=pages(), tail=0, tk=None, stride=0, ws=None, wsb=0, hq=4):
        st = _lib.lib().tp_selected_attention(P, 1, hq, 2, ctypes.byref(DEFAULT), ctypes.byref(store), n, selected, count, tk,
                                              tk, tail, stride, scale, ws, wsb, out, None)
        return st, _lib.lib().tp_last_error().decode()

    for kw in (dict(selected=None), dict(selected=P + 2), dict(count=0), dict(n=0), dict(n=9), dict(count=5), dict(scale=NAN),
               dict(out=None), dict(tail=64, tk=P, stride=64), dict(tail=3, tk=None, stride=64), dict(hq=5)):
        assert call(**kw)[0] == _lib.TP_ERR_INVALID, kw
    assert call(count=40, n=40, store=pages(64))[0] == _lib.TP_ERR_WORKSPACE


# ---- host layer ---------------------------------------------------------------------


def test_check_selection():
    check_selection(1, 0, 0)
    check_selection(5, 2, 3)
    for bad in ((0, 0, 0), (4, -1, 1), (4, 1, -1), (4, 3, 2)):
        with pytest.raises(ValueError, match="cannot select"):
            check_selection(*bad)
    for bad in ((True, 0, 0), (4.0, 1, 1), (4, 1.0, 1), (4, 1, None)):
        with pytest.raises(TypeError, match="must be an int"):
            check_selection(*bad)


def inputs(B=1, hq=4, hkv=2, T=3, dtype=torch.float16, columns=128):
    z = lambda *s: torch.zeros(s, dtype=dtype)  # noqa: E731
    return [z(B, hq, T, 128), z(B, hkv, T, 128), z(B, hkv, T, 128), z(T, columns), z(T, columns)]


@pytest.mark.parametrize("at,value,message", [
    (0, torch.zeros(1, 4, 128), "q must be"), (1, torch.zeros(1, 2, 3, 64), "k must be"), (2, None, "v must be"),
    (1, torch.zeros(1, 2, 3, 128), "one type"), (1, torch.zeros(1, 2, 4, 128).half(), "do not match"),
    (2, torch.zeros(1, 1, 3, 128).half(), "do not match"), (0, torch.zeros(2, 4, 3, 128).half(), "do not match"),
    (0, torch.zeros(1, 5, 3, 128).half(), "multiple"), (3, torch.zeros(3, 32).half(), "cos must be"),
    (3, torch.zeros(2, 128).half(), "cos must be"), (4, torch.zeros(2, 3, 128).half(), "sin must be"),
    (4, torch.zeros(3, 64).half(), "differ"), (4, torch.zeros(3, 128), "differ"), (3, torch.zeros(3, 128).int(), "float tensor"),
    (4, [0.0], "float tensor"),
])
def test_rotate_tokens_refusals(at, value, message):
    x = inputs()
    x[at] = value
    with pytest.raises(ValueError, match=message):
        rotate_tokens(*x)


def test_rotate_tokens_needs_a_gpu_and_no_gradients():
    with pytest.raises(RuntimeError, match="HIP device"):
        rotate_tokens(*inputs())
    with pytest.raises(ValueError, match="one type"):
        rotate_tokens(*inputs(dtype=torch.float64))


def small(**kw):
    return TurboPolarFastCache(TurboPolarConfig(**{"num_q_heads": 4, "num_kv_heads": 2, **kw}))


def kv(B, T, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((B, 2, T, 128), generator=g).half() for _ in range(2)]


def test_shared_prefix_refusals():
    prefix = small()
    prefix.runtime.append(*kv(1, 20))
    with pytest.raises(TypeError, match="TurboPolarFastCache"):
        SharedPrefixCache(prefix.runtime)
    with pytest.raises(TypeError, match="TurboPolarFastCache"):
        SharedPrefixCache(prefix, 3)
    with pytest.raises(ValueError, match="own cache"):
        SharedPrefixCache(prefix, prefix)
    two = small()
    two.runtime.append(*kv(2, 5))
    with pytest.raises(ValueError, match="batch 1"):
        SharedPrefixCache(two)
    for other in (small(k_angle_bits_deep=8), small(use_int8_radii=True), small(num_kv_heads=4), small(split_dim=32)):
        with pytest.raises(ValueError, match="one layout"):
            SharedPrefixCache(prefix, other)


def test_shared_prefix_bookkeeping():
    prefix = small()
    prefix.runtime.append(*kv(1, 20))
    cache = SharedPrefixCache(prefix)
    assert cache.offset == 20
    cache.append(*kv(3, 7, 1))
    assert cache.offset == 27 and prefix.offset == 20
    cache.select_rows([2, 0])
    assert cache.own.runtime._batch_size == 2
    assert torch.equal(cache.own.runtime.partial_k[0], kv(3, 7, 1)[0][2])
    branch = cache.fork(rows=[1, 1, 0])
    branch.append(*kv(3, 1, 2))
    assert (branch.offset, cache.offset, branch.prefix is prefix) == (28, 27, True)
    cache.truncate(22)
    assert cache.offset == 22
    for bad in (19, 23, -1):
        with pytest.raises(ValueError, match="cannot keep"):
            cache.truncate(bad)
    with pytest.raises(TypeError, match="int"):
        cache.truncate(21.0)
    cache.truncate(20)
    assert cache.offset == 20
    q = torch.zeros(2, 4, 1, 128).half()
    with pytest.raises(ValueError, match="HIP device"):
        cache.attention(q, 0.1)
    for bad in (q[:, :, 0], q.int(), torch.zeros(2, 4, 2, 128).half(), torch.zeros(2, 3, 1, 128).half()):
        with pytest.raises(ValueError):
            cache.attention(bad, 0.1)
    prefix.truncate(10)
    with pytest.raises(ValueError, match="held 20 tokens"):
        cache.attention(q, 0.1)
    with pytest.raises(ValueError, match="held 20 tokens"):
        cache.fork()
    with pytest.raises(ValueError, match="nothing to attend"):
        SharedPrefixCache(small()).attention(q, 0.1)


def test_a_prefix_of_other_tokens_is_refused():
    """Cut below its length and filled up to it again, or emptied: the length alone does not tell."""
    q = torch.zeros(2, 4, 1, 128).half()

    def shared_cache():
        prefix = small()
        prefix.runtime.append(*kv(1, 20))
        return prefix, SharedPrefixCache(prefix)

    prefix, cache = shared_cache()
    prefix.truncate(12)
    prefix.runtime.append(*kv(1, 8, 3))
    assert prefix.offset == 20
    for call in (lambda: cache.attention(q, 0.1), cache.fork, lambda: cache.decode_attention(q, *kv(2, 1), 0.1)):
        with pytest.raises(ValueError, match="tokens are others"):
            call()
    again = SharedPrefixCache(prefix)  # of the tokens held now
    with pytest.raises(ValueError, match="HIP device"):
        again.attention(q, 0.1)
    prefix.runtime.append(*kv(1, 9, 4))  # longer, and back: the same tokens
    prefix.truncate(25)
    prefix.truncate(20)
    assert again.fork().offset == 20
    prefix.select_rows([0])
    assert again.fork().offset == 20
    with pytest.raises(ValueError, match="tokens are others"):
        cache.fork()
    prefix.runtime.reset()
    prefix.runtime.append(*kv(1, 20))
    with pytest.raises(ValueError, match="tokens are others"):
        again.fork()
    prefix, cache = shared_cache()
    branch = prefix.fork()
    branch.truncate(3)
    assert cache.fork().offset == 20  # a branch's cuts are its own
    prefix.runtime = branch.runtime
    branch.runtime.append(*kv(1, 17))
    with pytest.raises(ValueError, match="tokens are others"):
        cache.fork()


def test_selected_attention_host_refusals():
    cache = small()
    q = torch.zeros(1, 4, 1, 128).half()
    with pytest.raises(ValueError, match="no tokens"):
        cache.selected_attention(q, 0.1, 4)
    with pytest.raises(ValueError, match="no pages"):
        cache.runtime.page_bounds()
    cache.runtime.append(*kv(1, 20))
    with pytest.raises(ValueError, match="HIP device"):
        cache.selected_attention(q, 0.1, 4)
    with pytest.raises(ValueError, match="batch of q"):
        cache.selected_attention(q.expand(2, -1, -1, -1), 0.1, 4)
    with pytest.raises(ValueError, match="multiple"):
        cache.selected_attention(q[:, :3], 0.1, 4)
    with pytest.raises(ValueError, match="q must be"):
        cache.selected_attention(q[:, :, 0], 0.1, 4)
    with pytest.raises(ValueError, match="float tensor"):
        cache.selected_attention(q.int(), 0.1, 4)


def test_append_rotated_host_refusals():
    cache = small()
    with pytest.raises(RuntimeError, match="HIP device"):
        cache.append_rotated(*inputs())
    assert cache.offset == 0 and not cache.runtime._initialized
