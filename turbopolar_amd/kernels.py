"""Launch wrappers: torch tensors -> the C ABI of libturbopolar_hip.so.

All device memory is owned by torch; the library never allocates.  Each call is
enqueued on the current torch stream of the tensors' device.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import TPPages, call_on, check, lib, on_device, ptr, require_hip, stream_handle
from .payload import PolarKeyBlock, QuantizedVBlock, layout_from_metadata

PAGE = 64
HEAD_DIM = 128
PAIRS = 64
V_GROUPS = 4


def fp16_scale(scale) -> float:
    """The attention scale as the reference kernels receive it: a 0-d fp16
    array (rfsn_v11/kernels/turbo_polar/metal.py:518,692,774).  ``scale`` is
    anything that NumPy converts; only plain non-zero floats, which nobody can
    change, are looked up (0.2 us against 0.7; 0.0 and -0.0 are one key)."""
    if type(scale) is float and scale:
        return _fp16_of_float(scale)
    return float(np.float16(scale))


@lru_cache(maxsize=64)
def _fp16_of_float(scale: float) -> float:
    return float(np.float16(scale))


# --------------------------------------------------------------------------
# page stores
# --------------------------------------------------------------------------

def _head_stride_pages(t: torch.Tensor, page_elems: int) -> Optional[int]:
    """Page slots between consecutive (batch, head) rows of a page tensor
    ``[B, H, S, ...]``; None when only one (batch, head) exists."""
    B, H = t.shape[0], t.shape[1]
    if H > 1:
        if B > 1 and t.stride(0) != H * t.stride(1):
            return -1
        st = t.stride(1)
    elif B > 1:
        st = t.stride(0)
    else:
        return None
    if st % page_elems:
        return -1
    return st // page_elems


def _inner_ok(t: torch.Tensor, inner_shape: Tuple[int, ...]) -> bool:
    """Dims 2.. are a dense run of pages of ``inner_shape``."""
    expect = 1
    for d in range(t.dim() - 1, 2, -1):
        if t.shape[d] > 1 and t.stride(d) != expect:
            return False
        expect *= t.shape[d]
    if t.shape[2] > 1 and t.stride(2) != expect:
        return False
    return tuple(t.shape[3:]) == inner_shape


def _fresh(t: torch.Tensor) -> torch.Tensor:
    out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    out.copy_(t)
    return out


class PageSet:
    """Device pointers (``tp_pages``) of a run of S pages per (batch, kv head),
    taken from 5-D page views (``[B, H, S, 64, .]``).  Views into a larger
    capacity buffer are used in place; anything else is copied once into a
    dense buffer, as the reference's ``_ensure_contiguous`` does."""

    def __init__(self, block: Optional[PolarKeyBlock], quant_v: Optional[QuantizedVBlock], head_dim: int = HEAD_DIM):
        self.keep = []
        tensors = {}
        if block is not None:
            int8, l1b, deepb, split, l1_row, deep_row = layout_from_metadata(block.metadata, head_dim)
            self.layout = _lib.make_layout(int8, l1b, deepb, split)
            self.l1_row, self.deep_row = l1_row, deep_row
            radii = block.radii
            if radii.dim() == 4:
                radii = radii.unsqueeze(2)
            if int8 and radii.dtype != torch.int8:
                raise ValueError(f"unsupported radii dtype: {radii.dtype}")
            if not int8 and radii.dtype != torch.float16:
                raise ValueError(f"unsupported radii dtype: {radii.dtype}")
            if int8 and block.radii_scales is None:
                raise ValueError("int8 radii require radii_scales")
            self.B, self.H, self.S = radii.shape[0], radii.shape[1], radii.shape[2]
            if radii.shape[3] != PAGE:
                raise ValueError(f"pages must hold {PAGE} tokens, got {radii.shape[3]}")
            tensors["radii"] = (radii, (PAGE, PAIRS))
            l1 = block.angle_codes_l1
            deep = block.angle_codes_deep
            if l1.dim() == 4:
                l1 = l1.unsqueeze(2)
                deep = deep.unsqueeze(2)
            tensors["angle_l1"] = (l1, (PAGE, l1_row))
            tensors["angle_deep"] = (deep, (PAGE, deep_row))
            if int8:
                rs = block.radii_scales
                if rs.dim() == 4:
                    rs = rs.unsqueeze(2)
                tensors["radii_scales"] = (rs.reshape(rs.shape[0], rs.shape[1], rs.shape[2], 1, 1), (1, 1))
        if quant_v is not None:
            codes, scales = quant_v.codes, quant_v.scales
            if codes.dim() == 4:
                codes = codes.unsqueeze(2)
                scales = scales.unsqueeze(2)
            if quant_v.group_size != 32 or codes.shape[-1] != HEAD_DIM:
                raise ValueError("quantised V must use groups of 32 over head_dim 128")
            if block is None:
                self.B, self.H, self.S = codes.shape[0], codes.shape[1], codes.shape[2]
            elif tuple(codes.shape[:3]) != (self.B, self.H, self.S):
                raise ValueError(f"K pages {(self.B, self.H, self.S)} and V pages {tuple(codes.shape[:3])} differ")
            tensors["v_codes"] = (codes, (PAGE, HEAD_DIM))
            tensors["v_scales"] = (scales, (PAGE, V_GROUPS))
        # Whether every buffer is used in place (changes to it are seen by later launches).
        self.in_place = True
        caps = set()
        for name, (t, inner) in tensors.items():
            require_hip(t, name)
            elems = int(np.prod(inner))
            if elems == 0:
                continue
            cap = _head_stride_pages(t, elems)
            if cap == -1 or not _inner_ok(t, inner) or (cap is not None and cap < self.S):
                t = _fresh(t)
                self.in_place = False
                tensors[name] = (t, inner)
                cap = _head_stride_pages(t, elems)
            caps.add(cap)
        caps.discard(None)
        if len(caps) > 1:
            # Buffers disagree on capacity: copy everything dense.
            self.in_place = False
            for name, (t, inner) in list(tensors.items()):
                if int(np.prod(inner)):
                    tensors[name] = (_fresh(t), inner)
            caps = {self.S}
        self.capacity = caps.pop() if caps else self.S
        self.tensors = {k: v[0] for k, v in tensors.items()}
        self.keep = list(self.tensors.values())
        self.pages = TPPages(
            ptr(self.tensors.get("radii")),
            ptr(self.tensors.get("radii_scales")),
            ptr(self.tensors.get("angle_l1")),
            ptr(self.tensors.get("angle_deep")),
            ptr(self.tensors.get("v_codes")),
            ptr(self.tensors.get("v_scales")),
            int(self.capacity),
        )

    def plan(self, bufs) -> Optional[tuple]:
        """What ``of_plan`` takes to describe other key buffers of the same forms as
        ``bufs`` (radii, level-1 codes, deep codes, scales), or None if one of
        these was copied."""
        used = [self.tensors.get(n) for n in ("radii", "angle_l1", "angle_deep", "radii_scales")]
        if not self.in_place or any(u is not None and u.data_ptr() != t.data_ptr() for u, t in zip(used, bufs)):
            return None
        return self.layout, self.l1_row, self.deep_row, self.B, self.H, self.S, self.capacity, used[3] is not None

    @classmethod
    def of_plan(cls, plan: tuple, bufs) -> "PageSet":
        """The PageSet of key buffers used in place, by a ``plan`` of their forms."""
        self = cls.__new__(cls)
        self.layout, self.l1_row, self.deep_row, self.B, self.H, self.S, self.capacity, scaled = plan
        self.in_place = True
        radii, l1, deep, scales = bufs
        self.tensors = {"radii": radii, "angle_l1": l1, "angle_deep": deep}
        if scaled:
            self.tensors["radii_scales"] = scales
        self.keep = list(bufs)
        self.pages = TPPages(radii.data_ptr(), scales.data_ptr() if scaled else None, l1.data_ptr(), deep.data_ptr(),
                             None, None, self.capacity)
        return self


# --------------------------------------------------------------------------
# kernel calls
# --------------------------------------------------------------------------

def encode_pages(
    k: Optional[torch.Tensor],
    v: Optional[torch.Tensor],
    token_begin: int,
    n_tokens: int,
    layout,
    pages: TPPages,
    page_begin: int,
) -> None:
    """tp_encode_pages over ``k``/``v`` of shape ``[B, H, T, 128]`` (contiguous,
    fp16 or fp32)."""
    ref = k if k is not None else v
    require_hip(ref, "k/v")
    if ref.dtype not in (torch.float16, torch.float32):
        raise ValueError(f"only float16 and float32 inputs are supported, got {ref.dtype}")
    for t in (k, v):
        if t is not None and (not t.is_contiguous() or t.dtype != ref.dtype or t.shape != ref.shape):
            raise ValueError("k and v must be contiguous tensors of one dtype and shape")
    B, H, T, D = ref.shape
    if D != HEAD_DIM:
        raise ValueError(f"head_dim must be {HEAD_DIM}, got {D}")
    in_dtype = 1 if ref.dtype == torch.float32 else 0
    with on_device(ref.device):
        st = lib().tp_encode_pages(
            ptr(k), ptr(v), in_dtype, B * H, T, int(token_begin), int(n_tokens),
            ctypes.byref(layout), ctypes.byref(pages), int(page_begin), stream_handle(ref.device),
        )
    check(st, "tp_encode_pages")


def decode_pages_into(layout, pages: TPPages, bh: int, page_begin: int, n_pages: int,
                      k_out: Optional[torch.Tensor], v_out: Optional[torch.Tensor], out_offset: int) -> None:
    """tp_decode_pages_into: pages [page_begin, page_begin + n_pages) of every
    (batch, head) row into tokens [out_offset, out_offset + 64 n_pages) of
    ``k_out`` / ``v_out`` (fp16 ``[B, H, T, 128]``, contiguous)."""
    ref = k_out if k_out is not None else v_out
    for t in (k_out, v_out):
        if t is not None and (t.dtype != torch.float16 or not t.is_contiguous() or t.shape != ref.shape):
            raise ValueError("k_out / v_out must be contiguous fp16 tensors of one shape")
    dev = ref.device
    with on_device(dev):
        st = lib().tp_decode_pages_into(
            ctypes.byref(layout), ctypes.byref(pages), int(bh), int(page_begin), int(n_pages), ptr(k_out), ptr(v_out),
            int(ref.shape[2]), int(out_offset), stream_handle(dev),
        )
    check(st, "tp_decode_pages_into")


def decode_pages_gather(layout, pages: TPPages, B: int, H: int, n_stored: int, page_index: torch.Tensor,
                        want_k: bool = True, want_v: bool = False):
    """tp_decode_pages_gather: the stored pages ``page_index`` (a device int32
    tensor, every entry in [0, n_stored)) of every (batch, head) row, in that
    order, as dense fp16 ``[B, H, len(page_index)*64, 128]`` K and/or V."""
    if page_index.dtype != torch.int32 or page_index.dim() != 1 or not page_index.is_contiguous():
        raise ValueError("page_index must be a contiguous 1-D int32 tensor")
    require_hip(page_index, "page_index")
    n = int(page_index.shape[0])
    dev = page_index.device
    shape = (B, H, n * PAGE, HEAD_DIM)
    k_out = torch.empty(shape, dtype=torch.float16, device=dev) if want_k else None
    v_out = torch.empty(shape, dtype=torch.float16, device=dev) if want_v else None
    with on_device(dev):
        st = lib().tp_decode_pages_gather(
            ctypes.byref(layout), ctypes.byref(pages), B * H, int(n_stored), ptr(page_index), n, ptr(k_out),
            ptr(v_out), stream_handle(dev),
        )
    check(st, "tp_decode_pages_gather")
    return k_out, v_out


def decode_pages(pageset: PageSet, want_k: bool = True, want_v: bool = True):
    """tp_decode_pages -> dense fp16 ``[B, H, S*64, 128]`` K and/or V."""
    B, H, S = pageset.B, pageset.H, pageset.S
    dev = next(iter(pageset.tensors.values())).device
    k_out = torch.empty((B, H, S * PAGE, HEAD_DIM), dtype=torch.float16, device=dev) if want_k else None
    v_out = torch.empty((B, H, S * PAGE, HEAD_DIM), dtype=torch.float16, device=dev) if want_v else None
    layout = getattr(pageset, "layout", _lib.make_layout(False, 4, 4, 64))
    with on_device(dev):
        st = lib().tp_decode_pages(
            ctypes.byref(layout), ctypes.byref(pageset.pages), B * H, 0, S, ptr(k_out), ptr(v_out), stream_handle(dev)
        )
    check(st, "tp_decode_pages")
    return k_out, v_out


def _q16(q: torch.Tensor) -> torch.Tensor:
    require_hip(q, "q")
    if q.dim() != 3 or q.shape[-1] != HEAD_DIM:
        raise ValueError(f"q must be [B, H_q, {HEAD_DIM}], got {tuple(q.shape)}")
    if q.dtype is torch.float16 and q.is_contiguous():
        return q
    return q.to(torch.float16).contiguous()


def fused_qk(q: torch.Tensor, pageset: PageSet, scale: float, qjl=None) -> torch.Tensor:
    """tp_fused_qk -> fp16 scores ``[B, H_q, S*64]``; with ``qjl`` (a
    ``qjl.QJLPages``) tp_fused_qk_qjl, which adds the QJL correction."""
    q16 = _q16(q)
    B, Hq, _ = q16.shape
    if B != pageset.B or Hq % pageset.H:
        raise ValueError(f"q heads {Hq} / batch {B} do not match kv pages {pageset.B}x{pageset.H}")
    dev = q16.device
    scores = torch.empty((B, Hq, pageset.S * PAGE), dtype=torch.float16, device=dev)
    common = (q16.data_ptr(), B, Hq, pageset.H, ctypes.byref(pageset.layout), ctypes.byref(pageset.pages), pageset.S)
    if qjl is None:
        st = call_on(dev, lib().tp_fused_qk, *common, float(scale), ptr(scores), stream_handle(dev))
    else:
        qjl.check_against(pageset.B, pageset.H, pageset.S, Hq)
        st = call_on(dev, lib().tp_fused_qk_qjl, *common, ctypes.byref(qjl.desc), float(scale), ptr(scores),
                     stream_handle(dev))
    check(st, "tp_fused_qk_qjl" if qjl is not None else "tp_fused_qk")
    return scores


class _Workspace:
    """Per-(device, stream) split-K workspace, grown on demand; its counter area
    starts zeroed and every kernel call leaves it zeroed."""

    _bufs: dict = {}

    @classmethod
    def get(cls, device: torch.device, nbytes: int, stream: Optional[int] = None) -> torch.Tensor:
        key = (device.index, stream_handle(device) if stream is None else stream)
        buf = cls._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            cls._bufs[key] = buf
        return buf


def _zeroed_workspace(nbytes: int, device: torch.device, stream: int) -> torch.Tensor:
    """The split-K workspace of the stream; one of its own inside a captured graph, whose replays may run beside
    those of another graph or eager calls."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return _Workspace.get(device, nbytes, stream)


@lru_cache(maxsize=1024)
def _workspace_bytes(B: int, Hq: int, Hkv: int, n_pages: int, pps: int) -> int:
    """tp_decode_workspace_bytes (its size does not depend on the tail)."""
    return int(lib().tp_decode_workspace_bytes(B, Hq, Hkv, n_pages, 0, pps))


def decode_attention(
    q: torch.Tensor,
    pageset: Optional[PageSet],
    tail_k: Optional[torch.Tensor],
    tail_v: Optional[torch.Tensor],
    actual_seq_len: int,
    scale: float,
    num_kv_heads: Optional[int] = None,
    pages_per_split: int = 0,
    out: Optional[torch.Tensor] = None,
    qjl=None,
) -> torch.Tensor:
    """tp_decode_attention -> fp16 ``[B, H_q, 128]``.

    ``tail_k``/``tail_v``: ``[B, H_kv, T_tail, 128]`` (T_tail < 64, any float
    dtype; converted to fp16 as metal.py:744 does).  ``qjl`` (a
    ``qjl.QJLPages`` of the pages): tp_decode_attention_qjl."""
    q16 = _q16(q)
    B, Hq, _ = q16.shape
    tail_len = 0 if tail_k is None else int(tail_k.shape[2])
    if pageset is not None:
        Hkv, n_pages = pageset.H, pageset.S
        if pageset.B != B:
            raise ValueError(f"batch of q ({B}) and pages ({pageset.B}) differ")
    else:
        if tail_len == 0:
            raise ValueError("nothing to attend: no pages and no tail")
        Hkv, n_pages = int(tail_k.shape[1]), 0
    if num_kv_heads is not None and num_kv_heads != Hkv:
        raise ValueError(f"expected {num_kv_heads} kv heads, got {Hkv}")
    if Hq % Hkv:
        raise ValueError(f"H_q={Hq} is not a multiple of H_kv={Hkv}")
    tk = tv = None
    tail_stride = 0
    if tail_len:
        require_hip(tail_k, "tail_k")
        if tail_k.shape != tail_v.shape or tuple(tail_k.shape[:2]) != (B, Hkv) or tail_k.shape[3] != HEAD_DIM:
            raise ValueError(f"tail shape {tuple(tail_k.shape)} does not match [B={B}, H_kv={Hkv}, T, {HEAD_DIM}]")
        tk, tv, tail_stride = _tail_pair(tail_k, tail_v)
    layout = pageset.layout if pageset is not None else _DEFAULT_LAYOUT
    pages = pageset.pages if pageset is not None else _NO_PAGES
    if qjl is not None:
        qjl.check_against(B, Hkv, n_pages, Hq)
    return _launch_decode(q16, Hkv, layout, pages, n_pages, tk, tv, tail_len, tail_stride, actual_seq_len, scale,
                          pages_per_split, out, qjl)


_DEFAULT_LAYOUT = _lib.make_layout(False, 4, 4, 64)
_NO_PAGES = TPPages()


def _launch_decode(q16, Hkv, layout, pages, n_pages, tk, tv, tail_len, tail_stride, seq_len, scale, pps, out,
                   qjl=None, own_workspace=False):
    B, Hq, _ = q16.shape
    dev = q16.device
    if out is None:
        out = torch.empty((B, Hq, HEAD_DIM), dtype=torch.float16, device=dev)
    L = lib()
    pps = int(pps)  # 0: the library's default
    stream = stream_handle(dev)
    nbytes = _workspace_bytes(B, Hq, Hkv, n_pages, pps)
    ws = _zeroed_workspace(nbytes, dev, stream) if own_workspace else _Workspace.get(dev, nbytes, stream)
    head = (ptr(q16), B, Hq, Hkv, ctypes.byref(layout), ctypes.byref(pages), n_pages)
    rest = (None if tk is None else tk.data_ptr(), None if tv is None else tv.data_ptr(), tail_len, tail_stride,
            int(seq_len), float(scale), pps, ws.data_ptr(), ws.numel(), ptr(out), stream)
    if qjl is None:
        st = call_on(dev, L.tp_decode_attention, *head, *rest)
    else:
        st = call_on(dev, L.tp_decode_attention_qjl, *head, ctypes.byref(qjl.desc), *rest)
    check(st, "tp_decode_attention_qjl" if qjl is not None else "tp_decode_attention")
    return out


def decode_attention_dense_v(
    q: torch.Tensor,
    pageset: PageSet,
    v_dense: torch.Tensor,
    actual_seq_len: int,
    scale: float,
    pages_per_split: int = 0,
    out: Optional[torch.Tensor] = None,
    qjl=None,
) -> torch.Tensor:
    """tp_decode_attention_dense_v -> fp16 ``[B, H_q, 128]``: attention over
    the compressed K pages of ``pageset`` (its V fields are not read) and dense
    V ``v_dense`` ``[B, H_kv, S, 64, 128]`` or ``[B, H_kv, S * 64, 128]`` (any
    float dtype; converted to fp16), the reference's
    execute_online_attention_dense_v (metal.py:586-649).  ``qjl``: a
    ``qjl.QJLPages`` of the pages (use_qjl=True)."""
    q16 = _q16(q)
    B, Hq, _ = q16.shape
    Hkv, n_pages = pageset.H, pageset.S
    if pageset.B != B:
        raise ValueError(f"batch of q ({B}) and pages ({pageset.B}) differ")
    if Hq % Hkv:
        raise ValueError(f"H_q={Hq} is not a multiple of H_kv={Hkv}")
    require_hip(v_dense, "v_dense")
    if v_dense.ndim == 5:
        if tuple(v_dense.shape[:2]) != (B, Hkv) or v_dense.shape[3] != PAGE or v_dense.shape[4] != HEAD_DIM:
            raise ValueError(f"v_dense shape {tuple(v_dense.shape)} does not match [B={B}, H_kv={Hkv}, S, "
                             f"{PAGE}, {HEAD_DIM}]")
        v_cap = int(v_dense.shape[2])
    elif v_dense.ndim == 4:
        if tuple(v_dense.shape[:2]) != (B, Hkv) or v_dense.shape[3] != HEAD_DIM or v_dense.shape[2] % PAGE:
            raise ValueError(f"v_dense shape {tuple(v_dense.shape)} does not match [B={B}, H_kv={Hkv}, S * {PAGE}, "
                             f"{HEAD_DIM}]")
        v_cap = int(v_dense.shape[2]) // PAGE
    else:
        raise ValueError(f"v_dense must be 4-D or 5-D, got shape {tuple(v_dense.shape)}")
    if v_cap < n_pages:
        raise ValueError(f"v_dense holds {v_cap} pages, the key block {n_pages}")
    v16 = v_dense.to(torch.float16).contiguous()
    if qjl is not None:
        qjl.check_against(B, Hkv, n_pages, Hq)
    dev = q16.device
    if out is None:
        out = torch.empty((B, Hq, HEAD_DIM), dtype=torch.float16, device=dev)
    L = lib()
    pps = int(pages_per_split)
    ws = _Workspace.get(dev, _workspace_bytes(B, Hq, Hkv, n_pages, pps))
    with on_device(dev):
        st = L.tp_decode_attention_dense_v(
            ptr(q16), B, Hq, Hkv, ctypes.byref(pageset.layout), ctypes.byref(pageset.pages), n_pages,
            ctypes.byref(qjl.desc) if qjl is not None else None, ptr(v16), v_cap, int(actual_seq_len),
            float(scale), pps, ws.data_ptr(), ws.numel(), ptr(out), stream_handle(dev),
        )
    check(st, "tp_decode_attention_dense_v")
    return out


def decode_attention_store(q: torch.Tensor, layout, pages: TPPages, n_pages: int, num_kv_heads: int,
                           tail_k: Optional[torch.Tensor], tail_v: Optional[torch.Tensor], seq_len: int,
                           scale: float, own_workspace: bool = False) -> torch.Tensor:
    """A cache's decode step: ``tp_decode_attention`` over the first ``n_pages``
    slots of a page store used in place (``pages`` carries its capacity) and a
    dense tail given as ``[B, H_kv, T, 128]`` views of a token-major buffer
    (``T`` < 64).  ``q`` is ``[B, H_q, 128]``.  ``own_workspace``: inside a captured
    graph the workspace is the graph's (``_zeroed_workspace``)."""
    q16 = _q16(q)
    tail_len = 0 if tail_k is None else int(tail_k.shape[2])
    tk = tv = None
    tail_stride = 0
    if tail_len:
        tk, tv, tail_stride = _tail_pair(tail_k, tail_v)
    if pages is None:
        pages, n_pages = _NO_PAGES, 0
    return _launch_decode(q16, num_kv_heads, layout, pages, n_pages, tk, tv, tail_len, tail_stride, seq_len, scale,
                          0, None, own_workspace=own_workspace)


@lru_cache(maxsize=1024)
def step_flag_words(B: int, Hq: int, Hkv: int) -> int:
    """Words of tp_decode_step's flag with check 4: a 64-byte line for the verdict and
    one per unit (batch row, kv head, head block of 16)."""
    return 16 * (1 + B * Hkv * -(-(Hq // Hkv) // 16))


def decode_step(q: torch.Tensor, layout, pages: Optional[TPPages], n_pages: int, new_k: torch.Tensor,
                new_v: torch.Tensor, tail_k: torch.Tensor, tail_v: torch.Tensor, tail_len: int, scale: float,
                check_mode: int, flag: torch.Tensor, epoch: int) -> torch.Tensor:
    """tp_decode_step: the token ``new_k`` / ``new_v`` ``[B, H_kv, 1, 128]``
    (contiguous fp16) joins the ``tail_len`` tokens of the tail buffers
    ``[B, H_kv, 64, 128]`` and ``q`` ``[B, H_q, 128]`` attends all of it in one
    launch.  Raises the append's ValueError when the launch reports a non-finite
    value (``check_mode`` 2 and 4; with 4 ``new_k`` and ``new_v`` are no longer read
    when this returns, and ``flag`` holds ``step_flag_words`` words)."""
    q16 = _q16(q)
    B, Hq, _ = q16.shape
    Hkv = new_k.shape[1]
    dev = q16.device
    out = torch.empty((B, Hq, HEAD_DIM), dtype=torch.float16, device=dev)
    stream = stream_handle(dev)
    ws = _Workspace.get(dev, _workspace_bytes(B, Hq, Hkv, n_pages, 0), stream)
    st = call_on(
        dev, lib().tp_decode_step,
        q16.data_ptr(), B, Hq, Hkv, ctypes.byref(layout), ctypes.byref(pages if pages is not None else _NO_PAGES),
        n_pages, new_k.data_ptr(), new_v.data_ptr(), tail_k.data_ptr(), tail_v.data_ptr(), tail_len, PAGE, scale, 0,
        ws.data_ptr(), ws.numel(), out.data_ptr(), check_mode, flag.data_ptr(), epoch, stream,
    )
    if st == _lib.TP_ERR_NONFINITE:
        raise ValueError("append() inputs must contain finite values")
    check(st, "tp_decode_step")
    return out


def _tail_view(t: torch.Tensor):
    """(tensor, token stride) such that rows are dense 128-element fp16 rows and
    (batch, head) planes are ``stride`` rows apart."""
    B, H, T, D = t.shape
    s0, s1, s2, s3 = t.stride()
    ok = s3 == 1 and (T == 1 or s2 == D)
    if ok:
        if H > 1:
            plane = s1
            ok = plane % D == 0 and (B == 1 or s0 == H * plane)
        elif B > 1:
            plane = s0
            ok = plane % D == 0
        else:
            plane = T * D
        if ok:
            stride = plane // D
            if stride >= T:
                return t, stride
    t = _fresh(t)
    return t, T


def _tail_pair(tail_k: torch.Tensor, tail_v: torch.Tensor):
    """fp16 K and V tails and the token stride they share (``_tail_view``)."""
    tk, stride = _tail_view(tail_k if tail_k.dtype is torch.float16 else tail_k.to(torch.float16))
    tv, stride_v = _tail_view(tail_v if tail_v.dtype is torch.float16 else tail_v.to(torch.float16))
    if stride_v != stride:
        tk, tv, stride = _fresh(tk), _fresh(tv), tk.shape[2]
    return tk, tv, stride


# --------------------------------------------------------------------------
# prompts and drafts
# --------------------------------------------------------------------------

_Strides12, _Strides6 = ctypes.c_int64 * 12, ctypes.c_int64 * 6


def _no_grad(*tensors: torch.Tensor) -> None:
    """Refuses tensors whose gradient is recorded, and those that carry a forward-mode tangent."""
    if (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) or (
        # A look at a level costs less than one at each tensor: 0.1 us against 2.
        getattr(forward_ad, "_current_level", 0) >= 0
        and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    ):
        raise ValueError("the TurboPolar kernels compute no gradients; call them under torch.no_grad()")


def _strided(t: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, int, int]]:
    """``t`` ``[B, H, T, 128]`` as a kernel reads it in place, and its (batch, head, token)
    strides: rows of 128 contiguous elements, 16 bytes aligned, tokens less than 2^23
    elements apart.  Anything else is copied."""
    B, H, T, _ = t.shape
    s0, s1, s2, s3 = t.stride()
    s0, s1, s2 = s0 if B > 1 else 0, s1 if H > 1 else 0, s2 if T > 1 else 0
    if s3 != 1 or (s0 | s1 | s2) & 7 or s2 >= 1 << 23 or t.data_ptr() & 15:
        t = _fresh(t)
        s0, s1, s2, _ = t.stride()
    return t, (s0, s1, s2)


def _token_major(B: int, H: int, T: int, dtype, device) -> torch.Tensor:
    """An output ``[B, H, T, 128]`` that lies token by token, as the output projection reads it."""
    return torch.empty_strided((B, H, T, HEAD_DIM), (T * H * HEAD_DIM, HEAD_DIM, H * HEAD_DIM, 1), dtype=dtype, device=device)


def _scratch(nbytes: int, device) -> Optional[torch.Tensor]:
    """Workspace of one call.  Not kept: its content is any, and the caching allocator orders its
    reuse on the stream, inside a captured graph too (graphs never share it)."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


@lru_cache(maxsize=1024)
def _prompt_workspace(B: int, Hq: int, Hkv: int, Tq: int, Tk: int, n_seq: int) -> int:
    return int(lib().tp_prompt_workspace_bytes(B, Hq, Hkv, Tq, Tk, n_seq))


def _starts(starts, name: str, tokens: int, device: torch.device) -> torch.Tensor:
    """Starts of packed sequences as a device int32 array.  A device tensor is taken as it is
    (its values are not read here); a host one or a sequence of ints is checked and copied."""
    if isinstance(starts, torch.Tensor) and starts.is_cuda:
        if starts.dtype is not torch.int32 or starts.dim() != 1 or not starts.is_contiguous() or starts.shape[0] < 2:
            raise ValueError(f"{name} must be a contiguous 1-D int32 tensor of at least 2 starts")
        if starts.device != device:
            raise ValueError(f"{name} is on {starts.device}, q on {device}")
        return starts
    values = [int(x) for x in (starts.tolist() if isinstance(starts, torch.Tensor) else starts)]
    if len(values) < 2 or values[0] != 0 or any(b < a for a, b in zip(values, values[1:])) or values[-1] > tokens:
        raise ValueError(f"{name} must ascend from 0 to at most {tokens} tokens, got {values[:8]}")
    return torch.tensor(values, dtype=torch.int32).to(device)


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float,
    causal: bool = True,
    q_starts=None,
    k_starts=None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """tp_prompt_attention: attention of ``q`` ``[B, H_q, Tq, 128]`` over ``k`` / ``v`` ``[B, H_kv,
    Tk, 128]``, all float16 or all bfloat16, any strides with contiguous rows of 128 (others are
    copied).  ``causal``: the queries are the last ``Tq`` of the ``Tk`` positions.  A query that
    sees no key gives 0.

    ``q_starts`` / ``k_starts`` (together, batch 1): packed sequences, at most 65,536, the ``n + 1``
    ascending token positions between them, as sequences of ints or host tensors, which are checked, or as
    int32 device tensors, which are not read here (values out of order give unspecified rows).
    Query rows behind the last sequence are 0, or left as they are where ``out`` is given.
    ``out`` shares no memory with k or v, nor with q unless it is q.

    Returns ``out``, or a new ``[B, H_q, Tq, 128]`` of q's type that lies token by token."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[-1] != HEAD_DIM:
            raise ValueError(f"{name} must be [B, H, T, {HEAD_DIM}], got {tuple(getattr(t, 'shape', ()))}")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"q, k and v must all be float16 or all bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, Hq, Tq, _ = q.shape
    Hkv, Tk = int(k.shape[1]), int(k.shape[2])
    if v.shape != k.shape or k.shape[0] != B:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match each other and q's batch of {B}")
    if B < 1 or Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"H_q={Hq} is not a multiple of H_kv={Hkv}, or the batch is empty")
    require_hip(q, "q")
    dev = q.device
    if k.device != dev or v.device != dev:
        raise ValueError(f"q is on {dev}, k on {k.device}, v on {v.device}")
    _no_grad(q, k, v)
    n_seq = 0
    if (q_starts is None) != (k_starts is None):
        raise ValueError("q_starts and k_starts come together")
    if q_starts is not None:
        if B != 1:
            raise ValueError(f"packed sequences take a batch of 1, got {B}")
        same = k_starts is q_starts and Tq == Tk
        q_starts = _starts(q_starts, "q_starts", Tq, dev)
        k_starts = q_starts if same else _starts(k_starts, "k_starts", Tk, dev)
        if q_starts.shape != k_starts.shape:
            raise ValueError(f"{q_starts.shape[0]} q_starts, {k_starts.shape[0]} k_starts")
        n_seq = int(q_starts.shape[0]) - 1
    keep_rest = out is not None
    if out is None:
        out = _token_major(B, Hq, Tq, q.dtype, dev)
    else:
        if out.shape != q.shape or out.dtype is not q.dtype or out.device != dev:
            raise ValueError(f"out must be {tuple(q.shape)} {q.dtype} on {dev}")
        _no_grad(out)
        view, strides = _strided(out)
        if view is not out or _overlaps(out):
            raise ValueError("out must have distinct, contiguous rows of 128 elements, 16 bytes aligned")
    if Tq == 0:
        return out
    (q, qs), (k, ks), (v, vs), (_, os_) = _strided(q), _strided(k), _strided(v), _strided(out)
    L = lib()
    ws = _scratch(_prompt_workspace(B, Hq, Hkv, Tq, Tk, n_seq), dev)
    st = call_on(
        dev, L.tp_prompt_attention, q.data_ptr(), ptr(k), ptr(v), out.data_ptr(), 1 if q.dtype is torch.bfloat16 else 0,
        B, Hq, Hkv, Tq, Tk, _Strides12(*qs, *ks, *vs, *os_), 1 if causal else 0, ptr(q_starts), ptr(k_starts), n_seq,
        1 if keep_rest else 0, float(scale), ptr(ws), 0 if ws is None else ws.numel(), stream_handle(dev),
    )
    check(st, "tp_prompt_attention")
    return out


def _overlaps(t: torch.Tensor) -> bool:
    """Whether two rows of ``t`` share memory (sizes and strides sorted, each step past the last)."""
    dims = sorted((s, n) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1)
    reach = t.shape[-1]
    for s, n in dims:
        if s < reach:
            return True
        reach = s * (n - 1) + reach
    return False


@lru_cache(maxsize=1024)
def _tree_workspace(B: int, Hq: int, Hkv: int, nodes: int, n_pages: int) -> int:
    return int(lib().tp_tree_workspace_bytes(B, Hq, Hkv, nodes, n_pages))


def tree_attention(q: torch.Tensor, layout, pages: Optional[TPPages], n_pages: int,
                   tail_k: Optional[torch.Tensor], tail_v: Optional[torch.Tensor], draft_k: torch.Tensor,
                   draft_v: torch.Tensor, tree, scale: float) -> torch.Tensor:
    """tp_tree_attention: the drafted tokens ``draft_k`` / ``draft_v`` ``[B, H_kv, T, 128]`` of a
    ``DraftTree`` and their queries ``q`` ``[B, H_q, T, 128]`` over the first ``n_pages`` slots of a
    page store and a dense tail ``[B, H_kv, < 64, 128]`` (None for none).  Float types other than
    float16 are converted to it, as the cache and the decode step do.  Returns fp16 ``[B, H_q, T,
    128]`` that lies token by token."""
    _check_draft(q, draft_k, draft_v, tree)
    return _tree_attention(q, layout, pages, n_pages, tail_k, tail_v, draft_k, draft_v, tree, scale)


def _tree_attention(q, layout, pages, n_pages, tail_k, tail_v, draft_k, draft_v, tree, scale) -> torch.Tensor:
    """``tree_attention`` of a checked draft."""
    B, Hq, T, _ = q.shape
    Hkv = int(draft_k.shape[1])
    dev = q.device
    tk = tv = None
    tail_len = tail_stride = 0
    if tail_k is not None and tail_k.shape[2]:
        if tail_k.shape != tail_v.shape or tuple(tail_k.shape[:2]) != (B, Hkv) or tail_k.shape[3] != HEAD_DIM:
            raise ValueError(f"tail shape {tuple(tail_k.shape)} does not match [B={B}, H_kv={Hkv}, T, {HEAD_DIM}]")
        tail_len = int(tail_k.shape[2])
        tk, tv, tail_stride = _tail_pair(tail_k, tail_v)
    (q, qs), (dk, ks), (dv, vs) = (_strided(t if t.dtype is torch.float16 else t.to(torch.float16))
                                   for t in (q, draft_k, draft_v))
    mask = tree.mask_on(dev)
    out, os_ = _token_major(B, Hq, T, torch.float16, dev), (T * Hq * HEAD_DIM, HEAD_DIM, Hq * HEAD_DIM)
    if pages is None:
        pages, n_pages = _NO_PAGES, 0
    ws = _scratch(_tree_workspace(B, Hq, Hkv, T, n_pages), dev)
    st = call_on(
        dev, lib().tp_tree_attention, q.data_ptr(), out.data_ptr(), B, Hq, Hkv, T, ctypes.byref(layout),
        ctypes.byref(pages), n_pages, ptr(tk), ptr(tv), tail_len, tail_stride, dk.data_ptr(), dv.data_ptr(),
        _Strides12(*qs, *ks, *vs, *os_), mask.data_ptr(), 0 if tree.shared else mask.stride(0), float(scale), ptr(ws),
        0 if ws is None else ws.numel(), stream_handle(dev),
    )
    check(st, "tp_tree_attention")
    return out


def _check_draft(q, draft_k, draft_v, tree) -> None:
    """The checks of a draft's tensors against each other and its tree."""
    for name, t in (("q", q), ("k", draft_k), ("v", draft_v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[-1] != HEAD_DIM:
            raise ValueError(f"{name} must be [B, H, T, {HEAD_DIM}], got {tuple(getattr(t, 'shape', ()))}")
        if not t.is_floating_point():
            raise ValueError(f"{name} must be a float tensor, got {t.dtype}")
    B, Hq, T, _ = q.shape
    if draft_k.shape != draft_v.shape or draft_k.shape[0] != B or draft_k.shape[2] != T:
        raise ValueError(f"drafted k {tuple(draft_k.shape)} and v {tuple(draft_v.shape)} do not match q {tuple(q.shape)}")
    Hkv = int(draft_k.shape[1])
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError(f"H_q={Hq} is not a multiple of H_kv={Hkv}")
    if tree.nodes != T or (tree.batch is not None and tree.batch != B):
        raise ValueError(f"a tree of {tree.nodes} nodes for {tree.batch or 'every'} batch rows does not match q {tuple(q.shape)}")
    require_hip(q, "q")
    if draft_k.device != q.device or draft_v.device != q.device:
        raise ValueError(f"q is on {q.device}, k on {draft_k.device}, v on {draft_v.device}")
    _no_grad(q, draft_k, draft_v)


def take_tokens(k: torch.Tensor, v: torch.Tensor, index: Union[Sequence[int], Sequence[Sequence[int]]], n: int,
                out_k: torch.Tensor, out_v: torch.Tensor, out_pos: int, flag: Optional[torch.Tensor] = None,
                epoch: int = 0) -> None:
    """tp_take_tokens: tokens ``index`` of ``k`` / ``v`` ``[B, H, T, 128]`` (fp16 or fp32; one list of
    ``n`` for every batch row, or one each) into rows ``[out_pos, out_pos + n)`` of ``out_k`` /
    ``out_v`` ``[B, H, tokens, 128]`` of the same type, contiguous.  With ``flag`` and ``epoch`` (as for
    an append) the call waits for the verdict and raises the append's ValueError."""
    B, H, T, _ = k.shape
    per_batch = isinstance(index[0], (list, tuple))
    flat = [i for row in index for i in row] if per_batch else list(index)
    (k, ks), (v, vs) = _strided(k), _strided(v)
    dev = k.device
    st = call_on(
        dev, lib().tp_take_tokens, k.data_ptr(), v.data_ptr(), 1 if k.dtype is torch.float32 else 0, B, H, T,
        _Strides6(*ks, *vs), (ctypes.c_int32 * len(flat))(*flat), n, 1 if per_batch else 0, out_k.data_ptr(),
        out_v.data_ptr(), int(out_k.shape[2]), out_pos, 0 if flag is None else 2, ptr(flag), epoch, stream_handle(dev),
    )
    if st == _lib.TP_ERR_NONFINITE:
        raise ValueError("append() inputs must contain finite values")
    check(st, "tp_take_tokens")


# --------------------------------------------------------------------------
# rotated appends
# --------------------------------------------------------------------------

_Strides2, _Strides3, _Strides9 = ctypes.c_int64 * 2, ctypes.c_int64 * 3, ctypes.c_int64 * 9
_ROTATE_TYPES = {torch.float16: 0, torch.float32: 1, torch.bfloat16: 2}


def _check_rotated(q, k, v, cos, sin) -> None:
    """The checks of ``rotate_tokens``'s tensors against each other."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[-1] != HEAD_DIM:
            raise ValueError(f"{name} must be [B, H, T, {HEAD_DIM}], got {tuple(getattr(t, 'shape', ()))}")
    if q.dtype not in _ROTATE_TYPES or k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError(f"q, k and v must be of one type, float16, bfloat16 or float32, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, Hq, T, _ = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[2] != T:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match each other and q {tuple(q.shape)}")
    if B < 1 or Hq < 1 or k.shape[1] < 1 or Hq % int(k.shape[1]):
        raise ValueError(f"H_q={Hq} is not a multiple of H_kv={k.shape[1]}, or the batch is empty")
    for name, t in (("cos", cos), ("sin", sin)):
        if not isinstance(t, torch.Tensor) or not t.is_floating_point():
            raise ValueError(f"{name} must be a float tensor")
        if t.dim() not in (2, 3) or t.shape[-2] != T or t.shape[-1] not in (HEAD_DIM // 2, HEAD_DIM) or (
                t.dim() == 3 and t.shape[0] not in (1, B)):
            raise ValueError(f"{name} must be [T, C] or [1 or B, T, C] for T={T} tokens of B={B} rows, C {HEAD_DIM} or "
                             f"{HEAD_DIM // 2}, got {tuple(t.shape)}")
    if cos.shape != sin.shape or cos.dtype is not sin.dtype:
        raise ValueError(f"cos {tuple(cos.shape)} {cos.dtype} and sin {tuple(sin.shape)} {sin.dtype} differ")
    require_hip(q, "q")
    for name, t in (("k", k), ("v", v), ("cos", cos), ("sin", sin)):
        if t.device != q.device:
            raise ValueError(f"q is on {q.device}, {name} on {t.device}")
    _no_grad(q, k, v, cos, sin)


def _table(t: torch.Tensor, dtype) -> Tuple[torch.Tensor, int, int]:
    """A table as the kernel reads it, and its batch and token strides."""
    if t.dtype is not dtype and t.dtype is not torch.float32:
        t = t.to(torch.float32)
    b, tok = (t.stride(0) if t.dim() == 3 and t.shape[0] > 1 else 0), (t.stride(-2) if t.shape[-2] > 1 else 0)
    if t.stride(-1) != 1 or (b | tok) & 7 or t.data_ptr() & 15:
        t = _fresh(t)
        b, tok = (t.stride(0) if t.dim() == 3 and t.shape[0] > 1 else 0), t.stride(-2)
    return t, b, tok


def rotate_tokens(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                  interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """tp_rotate_tokens: ``q`` ``[B, H_q, T, 128]`` and ``k`` ``[B, H_kv, T, 128]`` turned by their positions and
    ``v`` cast, each fp16: q token by token, k and v contiguous, as an append takes them.  q, k and v are float16,
    bfloat16 or float32, any strides with contiguous rows (others are copied).

    ``cos`` / ``sin``: ``[T, C]`` or ``[1 or B, T, C]``, as a model's rotary embedding gives them: C = 128, a column a
    dimension, or 64, a column a pair; of q's type or float32 (others are taken in float32).  Pairs are (d, d + 64), or
    (2d, 2d + 1) where ``interleaved``."""
    _check_rotated(q, k, v, cos, sin)
    B, H, T, _ = k.shape
    k_out, v_out = (torch.empty((B, H, T, HEAD_DIM), dtype=torch.float16, device=q.device) for _ in range(2))
    return _rotate_tokens(q, k, v, cos, sin, interleaved, k_out, v_out, 0), k_out, v_out


def _rotate_tokens(q, k, v, cos, sin, interleaved, k_out, v_out, pos, flag=None, epoch=0) -> torch.Tensor:
    """``rotate_tokens`` of checked inputs into rows ``[pos, pos + T)`` of ``k_out`` / ``v_out`` ``[B, H, tokens, 128]``
    (contiguous fp16); with ``flag`` and ``epoch`` (as for an append) the call waits for the verdict and raises the
    append's ValueError.  Returns q turned."""
    B, Hq, T, _ = q.shape
    dev, kind = q.device, _ROTATE_TYPES[q.dtype]
    out = _token_major(B, Hq, T, torch.float16, dev)
    if T == 0:
        return out
    (q, qs), (k, ks), (v, vs) = _strided(q), _strided(k), _strided(v)
    (cos, *table), (sin, *other) = _table(cos, q.dtype), _table(sin, q.dtype)
    if table != other:
        cos, sin = _fresh(cos), _fresh(sin)
        table = [cos.stride(0) if cos.dim() == 3 and cos.shape[0] > 1 else 0, cos.stride(-2)]
    st = call_on(
        dev, lib().tp_rotate_tokens, q.data_ptr(), k.data_ptr(), v.data_ptr(), kind, B, Hq, int(k.shape[1]), T,
        _Strides9(*qs, *ks, *vs), cos.data_ptr(), sin.data_ptr(), _ROTATE_TYPES[cos.dtype], int(cos.shape[-1]),
        _Strides2(*table), 1 if interleaved else 0, out.data_ptr(), _Strides3(T * Hq * HEAD_DIM, HEAD_DIM, Hq * HEAD_DIM),
        k_out.data_ptr(), v_out.data_ptr(), int(k_out.shape[2]), pos, 0 if flag is None else 2, ptr(flag),
        0 if flag is None else flag.numel(), epoch, stream_handle(dev),
    )
    if st == _lib.TP_ERR_NONFINITE:
        raise ValueError("append() inputs must contain finite values")
    check(st, "tp_rotate_tokens")
    return out


# --------------------------------------------------------------------------
# shared prefixes
# --------------------------------------------------------------------------

_Strides4 = ctypes.c_int64 * 4


def tail_args(tail_k: Optional[torch.Tensor], tail_v: Optional[torch.Tensor], tokens: int) -> tuple:
    """The first ``tokens`` rows of a cache's tail buffers ``[B, H, 64, 128]`` as an attention call takes them: (keys,
    values, tokens, tokens between rows), pointers or, where the buffers are not fp16, converted tensors."""
    if not tokens:
        return None, None, 0, 0
    if tail_k.dtype is torch.float16:  # contiguous, as the runtime makes them
        return tail_k.data_ptr(), tail_v.data_ptr(), tokens, int(tail_k.shape[2])
    k, v, stride = _tail_pair(tail_k[:, :, :tokens], tail_v[:, :, :tokens])
    return k, v, tokens, stride


def _pointer(x):
    return x.data_ptr() if isinstance(x, torch.Tensor) else x


@lru_cache(maxsize=1024)
def _shared_workspace(B: int, Hq: int, Hkv: int, layout: tuple, prefix_pages: int, prefix_tail: bool, n_pages: int,
                      tail: bool) -> int:
    return int(lib().tp_shared_workspace_bytes(B, Hq, Hkv, ctypes.byref(_lib.make_layout(*layout)), prefix_pages,
                                               int(prefix_tail), n_pages, int(tail)))


def _step_query(q: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """A step's queries ``[B, H_q, 1, 128]`` as a kernel reads them in place, and their batch and head strides."""
    if q.dtype is not torch.float16:
        q = q.to(torch.float16)
    s0, s1, _, s3 = q.stride()
    if s3 != 1 or (s0 | s1) & 7 or q.data_ptr() & 15:
        q = _fresh(q)
        s0, s1, _, _ = q.stride()
    return q, s0, s1


def shared_attention(q: torch.Tensor, layout, num_kv_heads: int, prefix, own, scale: float) -> torch.Tensor:
    """tp_shared_attention: ``q`` ``[B, H_q, 1, 128]`` over a prefix that every row shares and each row's own tokens.
    ``prefix`` and ``own`` are (store's descriptor or None, stored pages, ``tail_args``): of one batch row, and of B.
    Returns fp16 ``[B, H_q, 128]``."""
    q, q_b, q_h = _step_query(q)
    B, Hq, _, _ = q.shape
    dev = q.device
    (pages0, n0, (k0, v0, tail0, stride0)), (pages1, n1, (k1, v1, tail1, stride1)) = prefix, own
    out = torch.empty((B, Hq, HEAD_DIM), dtype=torch.float16, device=dev)
    form = layout.int8_radii, layout.l1_bits, layout.deep_bits, layout.split_dim
    ws = _scratch(_shared_workspace(B, Hq, num_kv_heads, form, n0, tail0 > 0, n1, tail1 > 0), dev)
    st = call_on(
        dev, lib().tp_shared_attention, q.data_ptr(), out.data_ptr(), B, Hq, num_kv_heads, ctypes.byref(layout),
        ctypes.byref(_NO_PAGES if pages0 is None else pages0), n0, _pointer(k0), _pointer(v0), tail0, stride0,
        ctypes.byref(_NO_PAGES if pages1 is None else pages1), n1, _pointer(k1), _pointer(v1), tail1, stride1,
        _Strides4(q_b, q_h, Hq * HEAD_DIM, HEAD_DIM), float(scale), None if ws is None else ws.data_ptr(),
        0 if ws is None else ws.numel(), stream_handle(dev),
    )
    check(st, "tp_shared_attention")
    return out


# --------------------------------------------------------------------------
# selected pages
# --------------------------------------------------------------------------

def page_bounds_into(layout, pages: TPPages, bh: int, page_begin: int, n_pages: int, bounds: torch.Tensor) -> None:
    """tp_page_bounds: pages [page_begin, page_begin + n_pages) of every (batch, head) row into their places of
    ``bounds`` (fp16 ``[B, H, capacity, 2, 128]``, contiguous)."""
    dev = bounds.device
    st = call_on(dev, lib().tp_page_bounds, ctypes.byref(layout), ctypes.byref(pages), bh, page_begin, n_pages,
                 ptr(bounds), int(bounds.shape[2]), stream_handle(dev))
    check(st, "tp_page_bounds")


def _bounds_view(bounds: torch.Tensor, B: int, H: int, S: int, device) -> Tuple[torch.Tensor, int]:
    """``bounds`` ``[B, H, S, 2, 128]`` as the kernel reads them, and the pages between its rows."""
    if isinstance(bounds, torch.Tensor) and bounds.shape == (B, H, S, 2, HEAD_DIM) and bounds.dtype is torch.float16 and (
            bounds.device == device and bounds.is_contiguous() and not bounds.data_ptr() & 15):
        return bounds, S
    if not isinstance(bounds, torch.Tensor) or tuple(bounds.shape) != (B, H, S, 2, HEAD_DIM) or bounds.dtype is not torch.float16:
        raise ValueError(f"bounds must be float16 [{B}, {H}, {S}, 2, {HEAD_DIM}], got "
                         f"{getattr(bounds, 'dtype', None)} {tuple(getattr(bounds, 'shape', ()))}")
    if bounds.device != device:
        raise ValueError(f"q is on {device}, bounds on {bounds.device}")
    cap = _head_stride_pages(bounds, 2 * HEAD_DIM)
    if cap == -1 or not _inner_ok(bounds, (2, HEAD_DIM)) or (cap is not None and cap < S) or bounds.data_ptr() & 15:
        bounds = _fresh(bounds)
        bounds = bounds if bounds.is_contiguous() else bounds.contiguous()
        cap = S
    return bounds, S if cap is None else cap


def check_selection(pages: int, first: int, last: int) -> None:
    for name, x in (("pages", pages), ("first", first), ("last", last)):
        if isinstance(x, bool) or not isinstance(x, int):
            raise TypeError(f"{name} must be an int, got {type(x).__name__}")
    if pages < 1 or first < 0 or last < 0 or first + last > pages:
        raise ValueError(f"cannot select {pages} pages, the first {first} and the last {last} among them")


@lru_cache(maxsize=1024)
def _selection_workspace(B: int, Hq: int, Hkv: int, n_pages: int, count: int) -> int:
    """What tp_select_pages and tp_selected_attention take, one after the other."""
    return max(int(lib().tp_select_workspace_bytes(B, Hq, Hkv, n_pages)), _workspace_bytes(B, Hq, Hkv, count, 0))


def selected_attention(q: torch.Tensor, layout, pages: TPPages, n_pages: int, num_kv_heads: int, bounds: torch.Tensor,
                       capacity: int, tail: tuple, scale: float, count: int, first: int,
                       last: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """tp_select_pages and tp_selected_attention: ``q`` ``[B, H_q, 128]`` over ``count`` of the ``n_pages`` stored
    pages, each kv head its own, and the dense tail (``tail_args``).  ``bounds``: fp16 ``[B, H_kv, n_pages, 2, 128]``,
    rows ``capacity`` pages apart.  Returns fp16 ``[B, H_q, 128]`` and the pages, int32 ``[B, H_kv, count]``,
    ascending."""
    q16 = _q16(q)
    B, Hq, _ = q16.shape
    dev = q16.device
    tk, tv, tail_len, tail_stride = tail
    out = torch.empty((B, Hq, HEAD_DIM), dtype=torch.float16, device=dev)
    selected = torch.empty((B, num_kv_heads, count), dtype=torch.int32, device=dev)
    L, stream = lib(), stream_handle(dev)
    ws = _zeroed_workspace(_selection_workspace(B, Hq, num_kv_heads, n_pages, count), dev, stream)
    q_ptr, list_ptr, ws_ptr, ws_bytes, scale = q16.data_ptr(), selected.data_ptr(), ws.data_ptr(), ws.numel(), float(scale)
    st = call_on(dev, L.tp_select_pages, q_ptr, B, Hq, num_kv_heads, bounds.data_ptr(), capacity, n_pages, first, last,
                 count, scale, list_ptr, ws_ptr, ws_bytes, stream)
    check(st, "tp_select_pages")
    st = call_on(
        dev, L.tp_selected_attention, q_ptr, B, Hq, num_kv_heads, ctypes.byref(layout), ctypes.byref(pages), n_pages,
        list_ptr, count, _pointer(tk), _pointer(tv), tail_len, tail_stride, scale, ws_ptr, ws_bytes, out.data_ptr(), stream,
    )
    check(st, "tp_selected_attention")
    return out, selected


def copy_pages(buffers, batch: int, heads: int, batch_in: int, rows: Optional[list], src_capacity: int,
               dst_capacity: int, n_stored: int, page_index: Optional[list], keep: int,
               tails: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]], tail_tokens: int,
               device: torch.device) -> None:
    """tp_copy_pages: ``buffers`` is a list of (source, destination, bytes of a page), sources and
    destinations contiguous ``[batch, heads, capacity, ...]``; ``rows`` and ``page_index`` lists of
    ints (the caller has checked them); ``tails`` (k, v, their copies), each ``[batch, heads, 64,
    128]`` and contiguous, of which ``tail_tokens`` rows are copied."""
    bufs = (_lib.TPPageCopy * max(1, len(buffers)))(*[_lib.TPPageCopy(ptr(s), ptr(d), n) for s, d, n in buffers])
    tail_ptrs, tail_bytes, tail_row = (None,) * 4, 0, 0
    if tails is not None and tail_tokens:
        token = HEAD_DIM * tails[0].element_size()
        tail_ptrs, tail_bytes, tail_row = tuple(t.data_ptr() for t in tails), tail_tokens * token, PAGE * token
    # Short indices travel with the launch; longer ones are copied to the device first.
    on_host = len(rows or ()) + len(page_index or ()) <= 768
    held = [
        None if not x else (ctypes.c_int32 * len(x))(*x) if on_host else torch.tensor(x, dtype=torch.int32).to(device)
        for x in (rows, page_index)
    ]
    row_ptr, page_ptr = (x if x is None else ctypes.addressof(x) if on_host else x.data_ptr() for x in held)
    st = call_on(
        device, lib().tp_copy_pages, bufs, len(buffers), batch, heads, batch_in, row_ptr, src_capacity, dst_capacity,
        n_stored, page_ptr, keep, 1 if on_host else 0, *tail_ptrs, tail_bytes, tail_row, stream_handle(device),
    )
    check(st, "tp_copy_pages")
