"""Refusals and host logic of the serving operators, none of which reaches a GPU."""

import ctypes

import pytest
import torch

from turbopolar_amd import DraftTree, TurboPolarConfig, TurboPolarFastCache, TurboPolarKVCacheRuntime, _lib, wire
from turbopolar_amd.kernels import _no_grad, _overlaps, _starts, prompt_attention

H = torch.float16


def x(*shape, dtype=H):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("q,k,v,message", [
    (x(4, 3, 128), x(1, 2, 3, 128), x(1, 2, 3, 128), "q must be"),
    (x(1, 4, 3, 64), x(1, 2, 3, 128), x(1, 2, 3, 128), "q must be"),
    (x(1, 4, 3, 128), x(1, 2, 3, 128), x(1, 2, 4, 128), "do not match"),
    (x(1, 4, 3, 128), x(2, 2, 3, 128), x(2, 2, 3, 128), "do not match"),
    (x(1, 4, 3, 128), x(1, 3, 3, 128), x(1, 3, 3, 128), "not a multiple"),
    (x(1, 4, 3, 128), x(1, 0, 3, 128), x(1, 0, 3, 128), "not a multiple"),
    (x(1, 4, 3, 128, dtype=torch.float32), x(1, 2, 3, 128), x(1, 2, 3, 128), "must all be float16"),
    (x(1, 4, 3, 128), x(1, 2, 3, 128, dtype=torch.bfloat16), x(1, 2, 3, 128), "must all be float16"),
])
def test_prompt_shapes(q, k, v, message):
    with pytest.raises(ValueError, match=message):
        prompt_attention(q, k, v, 0.1)


def test_prompt_needs_a_device():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        prompt_attention(x(1, 4, 3, 128), x(1, 2, 3, 128), x(1, 2, 3, 128), 0.1)


@pytest.mark.parametrize("starts", [[0], [1, 2], [0, 3, 2], [0, 9], torch.tensor([0, 4, 1])])
def test_starts(starts):
    with pytest.raises(ValueError, match="must ascend"):
        _starts(starts, "q_starts", 8, torch.device("cpu"))


def test_overlap():
    base = x(4, 4, 4, 128)
    assert not _overlaps(base) and not _overlaps(base.transpose(1, 2)) and not _overlaps(base[:, ::2])
    assert _overlaps(x(1, 1, 4, 128).expand(1, 3, 4, 128))
    assert _overlaps(x(2000).as_strided((1, 1, 3, 128), (0, 0, 64, 1)))


STRIDES = (ctypes.c_int64 * 12)(*[128] * 12)


def prompt_call(**change):
    a = dict(q=4096, k=8192, v=12288, out=16384, dtype=0, batch=1, hq=4, hkv=2, tq=3, tk=5, strides=STRIDES, causal=1,
             q_starts=None, k_starts=None, n_seq=0, keep=0, scale=0.1, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    return _lib.lib().tp_prompt_attention(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), b"dtype"), (dict(hkv=3), b"multiple"), (dict(batch=0), b"bad shape"), (dict(tq=-1), b"bad shape"),
    (dict(tq=2 ** 31), b"2^31"), (dict(tk=2 ** 31 - 1), b"2^31"), (dict(batch=2 ** 31), b"2^31"),
    (dict(q=4100), b"16-byte"), (dict(v=None), b"16-byte"), (dict(out=None), b"16-byte"), (dict(strides=None), b"strides"),
    (dict(strides=(ctypes.c_int64 * 12)(*[129] * 12)), b"strides"),
    (dict(strides=(ctypes.c_int64 * 12)(*[-128] * 12)), b"strides"),
    (dict(n_seq=2), b"packed"), (dict(n_seq=1, batch=2, q_starts=4096, k_starts=4096), b"packed"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"),
])
def test_prompt_abi(change, message):
    assert prompt_call(**change) == _lib.TP_ERR_INVALID and message in _lib.lib().tp_last_error()


def test_prompt_abi_workspace():
    L = _lib.lib()
    assert prompt_call(tq=0) == 0  # nothing to do
    need = L.tp_prompt_workspace_bytes(1, 4, 2, 1, 100000, 0)
    assert need > 0 and L.tp_prompt_workspace_bytes(1, 4, 2, 100000, 100000, 0) == 0
    st = prompt_call(tq=1, tk=100000, ws=4096, ws_bytes=need - 1)
    assert st == _lib.TP_ERR_WORKSPACE and b"workspace" in L.tp_last_error()
    st = prompt_call(tq=1, tk=100000, ws=4096 + 16, ws_bytes=need)
    assert st == _lib.TP_ERR_WORKSPACE


def tree_call(**change):
    lay = _lib.make_layout(False, 4, 4, 64)
    pages = _lib.TPPages(4096, 8192, 12288, 16384, 20480, 24576, 8)
    a = dict(q=4096, out=8192, batch=1, hq=4, hkv=2, nodes=3, layout=ctypes.byref(lay), pages=ctypes.byref(pages),
             n_pages=1, tail_k=4096, tail_v=4096, tail_len=3, tail_stride=64, dk=4096, dv=4096, strides=STRIDES,
             mask=4096, mask_stride=0, scale=0.1, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    return _lib.lib().tp_tree_attention(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(hkv=3), b"multiple"), (dict(nodes=0), b"nodes"), (dict(nodes=257), b"nodes"), (dict(n_pages=9), b"capacity"),
    (dict(n_pages=-1), b"capacity"), (dict(tail_len=64), b"tail_len"), (dict(tail_k=None), b"tail"),
    (dict(tail_stride=2), b"tail"), (dict(q=4104), b"16-byte"), (dict(mask=None), b"mask"), (dict(dk=None), b"draft"),
    (dict(strides=None), b"strides"), (dict(strides=(ctypes.c_int64 * 12)(*[4] * 12)), b"strides"),
    (dict(scale=float("inf")), b"scale"),
])
def test_tree_abi(change, message):
    assert tree_call(**change) == _lib.TP_ERR_INVALID and message in _lib.lib().tp_last_error()


def test_tree_abi_workspace():
    assert tree_call(n_pages=8) == _lib.TP_ERR_WORKSPACE
    assert _lib.lib().tp_tree_workspace_bytes(1, 4, 2, 3, 8) > 0 == _lib.lib().tp_tree_workspace_bytes(1, 4, 2, 3, 1)


def test_copy_abi():
    L = _lib.lib()
    buf = _lib.TPPageCopy(4096, 8192, 512)
    call = lambda **c: L.tp_copy_pages(*{**dict(  # noqa: E731
        bufs=ctypes.byref(buf), n=1, batch=1, heads=2, batch_in=1, rows=None, src=8, dst=4, stored=4, index=None, keep=4,
        host=0, tk=None, tv=None, tko=None, tvo=None, tail=0, row=0, stream=None), **c}.values())
    for change, message in [
        (dict(n=9), b"up to"), (dict(batch=40000), b"up to"), (dict(batch=2), b"row index"), (dict(keep=5), b"do not fit"),
        (dict(stored=9), b"do not fit"), (dict(keep=3, stored=2), b"do not fit"), (dict(tail=8, row=16), b"tails"),
        (dict(tail=32, row=16), b"tails"), (dict(tail=16, row=16), b"tails"), (dict(rows=4097), b"aligned"),
    ]:
        assert call(**change) == _lib.TP_ERR_INVALID and message in L.tp_last_error(), change
    for rows, pages, message in [([1], None, b"batch row 1"), (None, [0, 4, 1, 2], b"page 4"), (None, [0, -1, 1, 2], b"page -1")]:
        held = [None if x is None else (ctypes.c_int32 * len(x))(*x) for x in (rows, pages)]
        at = [None if x is None else ctypes.addressof(x) for x in held]
        assert call(rows=at[0], index=at[1], host=1) == _lib.TP_ERR_INVALID and message in L.tp_last_error()
    many = (ctypes.c_int32 * 769)()
    assert call(dst=1024, keep=769, index=ctypes.addressof(many), host=1) == _lib.TP_ERR_INVALID
    assert b"at most 768" in L.tp_last_error()
    none = _lib.TPPageCopy(None, 8192, 512)
    assert call(bufs=ctypes.byref(none)) == _lib.TP_ERR_INVALID and b"missing" in L.tp_last_error()


def test_take_abi():
    L = _lib.lib()
    index = (ctypes.c_int32 * 3)(0, 2, 1)
    strides = (ctypes.c_int64 * 6)(*[128] * 6)
    call = lambda **c: L.tp_take_tokens(*{**dict(  # noqa: E731
        k=4096, v=8192, dtype=0, batch=1, heads=2, tokens=3, strides=strides, index=index, n=3, per=0, ok=4096, ov=4096,
        out_tokens=64, pos=0, check=0, flag=None, epoch=0, stream=None), **c}.values())
    for change, message in [
        (dict(dtype=2), b"in_dtype"), (dict(k=None), b"bad input"), (dict(n=0), b"index must"), (dict(tokens=2), b"outside"),
        (dict(index=(ctypes.c_int32 * 3)(0, -1, 1)), b"outside"), (dict(pos=62), b"do not fit"), (dict(check=2), b"check"),
        (dict(check=1), b"check"), (dict(k=4097), b"aligned"), (dict(strides=(ctypes.c_int64 * 6)(*[4] * 6)), b"strides"),
        (dict(n=1025, index=(ctypes.c_int32 * 1025)()), b"index must"),
    ]:
        assert call(**change) == _lib.TP_ERR_INVALID and message in L.tp_last_error(), change


# ---- drafts -------------------------------------------------------------------------


def test_tree_masks_and_paths():
    tree = DraftTree([-1, 0, 0, 1, -1, 4])
    bits = [m[0] for m in tree._mask[0].tolist()]
    assert bits == [0b1, 0b11, 0b101, 0b1011, 0b10000, 0b110000]
    assert tree.depths() == [0, 1, 1, 2, 0, 1] and tree.path_to(3) == [0, 1, 3] and tree.path_to(4) == [4]
    with pytest.raises(IndexError):
        tree.path_to(6)
    long = DraftTree(list(range(-1, 199)))
    words = long._mask[0, 199].tolist()
    assert words == [-1, -1, -1, 2 ** 8 - 1] and long._mask[0, 63].tolist() == [-1, 0, 0, 0]


def test_padded_trees():
    tree = DraftTree([[-1, 0, 1], [-1]])
    assert (tree.nodes, tree.batch) == (3, 2) and tree._mask[1].tolist() == [[1], [0], [0]]


@pytest.mark.parametrize("parents,error", [
    ([], ValueError), ([0], ValueError), ([-1, 1], ValueError), ([-1, -2], ValueError), ([-1, 0.0], TypeError),
    ([-1, True], TypeError), (list(range(-1, 256)), ValueError), ([[-1], 0], TypeError), ([[]], ValueError),
])
def test_bad_trees(parents, error):
    with pytest.raises(error):
        DraftTree(parents)


def cache():
    return TurboPolarFastCache(TurboPolarConfig(num_q_heads=4, num_kv_heads=2))


@pytest.mark.parametrize("q,k,v,message", [
    (x(1, 4, 3, 128), x(1, 2, 2, 128), x(1, 2, 2, 128), "do not match"),
    (x(1, 4, 2, 128), x(1, 2, 2, 128), x(1, 2, 2, 128), "does not match"),
    (x(1, 4, 3, 128), x(1, 3, 3, 128), x(1, 3, 3, 128), "not a multiple"),
    (x(4, 3, 128), x(1, 2, 3, 128), x(1, 2, 3, 128), "q must be"),
    (x(1, 4, 3, 128, dtype=torch.int32), x(1, 2, 3, 128), x(1, 2, 3, 128), "float tensor"),
])
def test_draft_shapes(q, k, v, message):
    with pytest.raises(ValueError, match=message):
        cache().tree_attention(q, k, v, DraftTree([-1, 0, 0]), 0.1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cache().tree_attention(x(1, 4, 3, 128), x(1, 2, 3, 128), x(1, 2, 3, 128), DraftTree([-1, 0, 0]), 0.1)


# ---- a cache without pages, on the host ------------------------------------------------


def host_cache(B=2, T=20, dtype=H):
    torch.manual_seed(0)
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=4, num_kv_heads=2))
    k, v = torch.randn(2, B, 2, T, 128).to(dtype)
    rt.append(k, v)
    return rt, k, v


def test_host_fork_truncate_accept():
    rt, k, v = host_cache()
    other = rt.fork(tokens=7, rows=[1, 1, 0])
    assert other.actual_seq_len == 7 and torch.equal(other.partial_k, k[[1, 1, 0], :, :7])
    rt.truncate(9)
    assert torch.equal(rt.partial_v, v[:, :, :9]) and rt.actual_seq_len == 9
    dk, dv = torch.randn(2, 2, 2, 6, 128).half()
    rt.accept(dk, dv, [0, 4])
    assert torch.equal(rt.partial_k, torch.cat((k[:, :, :9], dk[:, :, [0, 4]]), 2)) and rt.actual_seq_len == 11
    rt.accept(dk, dv, [[5], [1]])
    assert torch.equal(rt.partial_k[0, :, -1], dk[0, :, 5]) and torch.equal(rt.partial_v[1, :, -1], dv[1, :, 1])
    rt.accept(dk, dv, [])
    rt.select_rows([1])
    assert rt.actual_seq_len == 12 and rt.partial_k.shape[0] == 1
    assert torch.equal(other.partial_k, k[[1, 1, 0], :, :7])  # a copy
    rt.append(k[:1], v[:1])
    assert rt.actual_seq_len == 32


def test_host_refusals():
    rt, k, v = host_cache()
    for bad, error in [(21, ValueError), (-1, ValueError), (2.0, TypeError), (True, TypeError)]:
        with pytest.raises(error):
            rt.truncate(bad)
        with pytest.raises(error):
            rt.fork(tokens=bad)
    for rows, error in [([2], IndexError), ([-1], IndexError), ([], ValueError), ([0.5], TypeError),
                        (torch.tensor([0.0]), ValueError), (torch.tensor([[0]]), ValueError)]:
        with pytest.raises(error):
            rt.fork(rows=rows)
    with pytest.raises(IndexError):
        rt.fork(pages=[0])
    with pytest.raises(ValueError, match="not both"):
        rt.fork(tokens=1, pages=[])
    d = torch.randn(2, 2, 6, 128).half()
    for path, error in [([6], IndexError), ([-1], IndexError), ([[0]], ValueError), ([[0], [0, 1]], ValueError),
                        ([1.5], TypeError)]:
        with pytest.raises(error):
            rt.accept(d, d, path)
    with pytest.raises(ValueError, match="batch size"):
        rt.accept(d[:1], d[:1], [0])
    with pytest.raises(ValueError, match="dtype"):
        rt.accept(d.float(), d.float(), [0])
    bad = d.clone()
    bad[0, 0, 1, 3] = float("nan")
    with pytest.raises(ValueError, match="finite"):
        rt.accept(bad, d, [1])
    assert rt.actual_seq_len == 20 and torch.equal(rt.partial_k, k)
    rt.accept(bad, d, [0, 2])  # a node that is not taken may hold anything
    assert rt.actual_seq_len == 22


def test_empty_cache():
    rt = TurboPolarKVCacheRuntime(TurboPolarConfig(num_q_heads=4, num_kv_heads=2))
    assert rt.fork().actual_seq_len == 0 and rt.fork(tokens=0).actual_seq_len == 0
    rt.truncate(0)
    with pytest.raises(IndexError):
        rt.fork(rows=[0])
    with pytest.raises(ValueError):
        rt.truncate(1)


def emptied(B=2):
    """A cache that was cut to nothing and holds no buffers, as a fork of no tokens does on a device."""
    rt, _, _ = host_cache(B)
    rt.truncate(0)
    rt = wire.load_state_dict(*wire.state_dict(rt), "cpu")
    assert rt._initialized and rt._tail_k is None and rt.k_storage.radii is None
    return rt


def test_branches_of_a_cache_without_buffers():
    rt = emptied()
    for other, B in ((rt.fork(), 2), (rt.fork(tokens=0), 2), (rt.fork(pages=[]), 2), (rt.fork(rows=[1, 0, 0]), 3)):
        assert other.actual_seq_len == 0 and other._batch_size == B and other._initialized
        k = torch.randn(B, 2, 3, 128).half()
        other.append(k, k)
        assert torch.equal(other.fork().partial_k, k)
    rt.select_rows([1])
    rt.keep_pages([])
    with pytest.raises(ValueError, match="batch size"):
        rt.append(k, k)
    rt.append(k[:1], k[:1])
    assert rt.actual_seq_len == 3


@pytest.mark.parametrize("scale,error", [(float("nan"), ValueError), (float("inf"), ValueError), (1e300, ValueError),
                                         (None, TypeError)])
def test_prompt_scale_is_checked_first(scale, error):
    """Before the device, and so before the append."""
    c = cache()
    with pytest.raises(error, match="scale|float"):
        c.prompt_attention(x(1, 4, 3, 128), x(1, 2, 3, 128), x(1, 2, 3, 128), scale)
    assert c.offset == 0


def test_replaced_stores_are_let_go():
    for use in (lambda c: c.select_rows([0, 1]), lambda c: c.keep_pages([])):
        c = cache()
        c.runtime.append(x(2, 2, 5, 128), x(2, 2, 5, 128))
        c._store = (x(1), x(1), None)  # as a call on the store leaves it
        use(c)
        assert c._store is None and c.offset == 5


def test_no_grad_sees_tangents():
    """Forward-mode duals are refused, with gradients recorded or not; plain tensors beside them are not."""
    import torch.autograd.forward_ad as fw

    a, b = x(3), x(3)
    _no_grad(a, b)
    with pytest.raises(ValueError, match="no gradients"):
        _no_grad(a, b.clone().requires_grad_())
    with torch.no_grad():
        _no_grad(a, b.clone().requires_grad_())
    with fw.dual_level():
        _no_grad(a, b)
        dual = fw.make_dual(b, a)
        with pytest.raises(ValueError, match="no gradients"):
            _no_grad(a, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="no gradients"):
            _no_grad(dual, a)
    with pytest.raises(ValueError, match="no gradients"):
        torch.func.jvp(lambda t: (_no_grad(t), t)[1], (a,), (b,))
    with torch.inference_mode():
        _no_grad(a, b, x(2))


def test_prompt_counts_stay_in_32_bits():
    """Sequences whose tiles, empty ones among them, would be counted past 2^31 rows, and more than a call takes."""
    packed = dict(q_starts=4096, k_starts=4096)
    for change, message in [(dict(n_seq=65537), b"at most 65536"), (dict(n_seq=10_000_000), b"at most 65536"),
                            (dict(n_seq=65536, tq=(2 ** 31 - 513) // 2), b"too many tiles")]:
        assert prompt_call(**packed, **change) == _lib.TP_ERR_INVALID and message in _lib.lib().tp_last_error(), change
