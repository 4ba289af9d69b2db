"""``TurboPolarFastCache`` -- one decoder layer's compressed KV cache as a
generation loop drives it -- and ``make_turbo_caches``.

Interface of the reference's mlx_lm cache object
(benchmarks/turbopolar_fast_attention.py:20-229): the class, its attributes and
method names, the meaning of every argument, the validation messages of
``_validate_decode_shape`` (:89-104) and the layout ``make_turbo_caches``
builds (:207-229).  The mechanism is this library's own:

* ``decode_attention`` is one launch, which checks the token, copies it to the
  runtime's dense-tail buffer and attends it with the tail and the runtime's page
  store, used in place with its capacity as the page stride; a token that
  completes a page is appended first (staging, page encode) and then attended.
  The store's ``tp_pages`` descriptor is kept until the store moves (growth or
  reset).  A cache with no completed page attends the tail alone (the reference
  switches to dense MLX attention there, :150-159).
* ``update_and_fetch`` (prefill) appends, encodes the zero-padded tail as one
  page (the reference's ``_maybe_encode_partial``) and decodes the stored
  pages and that page side by side into one fp16 K and one fp16 V buffer
  (``tp_decode_pages_into``), returning views of its first ``offset`` tokens.
  Nothing the size of the cache is copied besides that output.
"""

from __future__ import annotations

import copy
import math
from ctypes import c_float
from typing import List, Optional, Sequence, Tuple

import torch

from .bridge import HipKernelBridge
from .codecs import GroupedVQuantizer, PolarQuantDecoder
from .config import TurboPolarConfig
from .draft import DraftTree
from .kernels import (
    HEAD_DIM, PAGE, _check_draft, _no_grad, _tree_attention, check_selection, decode_attention_store, decode_pages_into,
    fp16_scale, prompt_attention, rotate_tokens, selected_attention, tail_args,
)
from .runtime import TurboPolarKVCacheRuntime
from .storage import pages_of


class TurboPolarFastCache:
    def __init__(self, config: TurboPolarConfig):
        self.config = config
        self.runtime = TurboPolarKVCacheRuntime(config)
        # The reference's attributes: the kernel bridge (the decode step here
        # launches the kernel without it), the codecs, and no QJL encoder
        # (the config rejects QJL).
        self.bridge = HipKernelBridge()
        self.decoder = PolarQuantDecoder()
        self.v_dequantizer = GroupedVQuantizer(group_size=32)
        self.qjl_encoder = None
        self._store = None  # (radii buffer, V codes buffer, their tp_pages)

    @property
    def offset(self) -> int:
        """Tokens held (the position the next token's RoPE uses)."""
        return self.runtime.actual_seq_len

    def _store_pages(self):
        """tp_pages of the runtime's page store, rebuilt when its buffers move."""
        ks, vs = self.runtime.k_storage, self.runtime.v_storage
        hit = self._store
        if hit is None or hit[0] is not ks.radii or hit[1] is not vs.codes:
            hit = (ks.radii, vs.codes, pages_of(ks, vs))
            self._store = hit
        return hit[2]

    # ------------------------------------------------------------------ prefill
    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Append ``[B, H_kv, T, D]`` keys/values and return the whole history
        decompressed (turbopolar_fast_attention.py:56-86): the stored pages and
        the zero-padded tail page decoded exactly as the reference's
        ``decode_block`` / ``dequantize_block`` do, cut to ``offset`` tokens,
        in the dtype of ``keys``."""
        want = keys.dtype
        rt = self.runtime
        rt.append(keys.to(torch.float16), values.to(torch.float16))
        n_pages, tail = rt.k_storage.block_count, rt._tail_len
        if n_pages == 0 and tail == 0:
            raise RuntimeError("TurboPolar cache returned no blocks after append")
        B, H = rt._batch_size, rt._num_kv_heads
        slots = n_pages + (1 if tail else 0)
        dev = rt._tail_k.device
        k_out = torch.empty((B, H, slots * PAGE, HEAD_DIM), dtype=torch.float16, device=dev)
        v_out = torch.empty_like(k_out)
        layout = rt.polar_encoder.layout
        run = n_pages
        full = n_pages == rt.k_storage.capacity
        if run and full:  # the tail page has no free slot: the long launch goes first, the host's work runs under it
            decode_pages_into(layout, self._store_pages(), B * H, 0, run, k_out, v_out, 0)
        if tail:
            pages, slot, in_storage = rt._partial_page_store()
            if in_storage:  # the tail page sits in the store's next free slot
                run = n_pages + 1
            else:
                decode_pages_into(layout, pages, B * H, slot, 1, k_out, v_out, n_pages * PAGE)
        if run and not full:
            decode_pages_into(layout, self._store_pages(), B * H, 0, run, k_out, v_out, 0)
        k, v = k_out[:, :, : rt.actual_seq_len], v_out[:, :, : rt.actual_seq_len]
        if want != torch.float16:
            k, v = k.to(want), v.to(want)
        return k, v

    # ------------------------------------------------------------------ decode
    @staticmethod
    def _validate_decode_shape(q, k_new, v_new, config: TurboPolarConfig) -> None:
        """The reference's decode-shape contract (turbopolar_fast_attention.py:89-104):
        same checks, exception types and messages."""
        if any(t.ndim != 4 for t in (q, k_new, v_new)):
            raise ValueError("decode_attention inputs must be 4-D (B, H, T, D)")
        B, H_q, T, D = q.shape
        H_kv, T_k, T_v = k_new.shape[1], k_new.shape[2], v_new.shape[2]
        if B != 1:
            raise NotImplementedError("TurboPolar fused decode only supports batch size 1.")
        if (T, T_k, T_v) != (1, 1, 1):
            raise ValueError("decode_attention only supports a single query/key/value token")
        if D != 128:
            raise NotImplementedError("TurboPolar fused decode only supports head_dim == 128.")
        if D != config.head_dim:
            raise ValueError(f"decode_attention head_dim {D} does not match config {config.head_dim}")
        if H_q % H_kv != 0:
            raise ValueError(f"decode_attention requires GQA ratio to divide evenly, got {H_q} and {H_kv}")

    def decode_attention(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                         scale: float, defer_check: bool = False) -> torch.Tensor:
        """One decode step (turbopolar_fast_attention.py:106-188): append the
        token's K/V ``[1, H_kv, 1, 128]`` and attend ``q`` ``[1, H_q, 1, 128]``
        over every cached token with ``scale`` (taken as fp16, as the
        reference's kernels receive it).  Returns fp16 ``[1, H_q, 128]``.  The
        caller may overwrite or free ``k_new`` and ``v_new`` on any stream once the
        call is back (``q`` once its launch is through, and K and V too with
        ``defer_check``).

        ``defer_check``: the append's non-finite verdict is read later by
        ``runtime.resolve_deferred_check()`` instead of now (no stream drain
        per step; the transformers hook resolves every layer once per forward)."""
        self._validate_decode_shape(q, k_new, v_new, self.config)
        rt = self.runtime
        k_new, v_new = k_new.to(torch.float16), v_new.to(torch.float16)
        scale = fp16_scale(scale)
        layout = rt.polar_encoder.layout
        out = rt.append_and_attend(q[:, :, 0], k_new, v_new, scale,
                                   self._store_pages() if rt.k_storage.block_count else None, layout, defer_check)
        if out is not None:
            return out
        rt.append(k_new, v_new, defer_check=defer_check)
        n_pages = rt.k_storage.block_count
        tail_k, tail_v = rt._tail_views()
        pages = self._store_pages() if n_pages else None
        return decode_attention_store(q[:, :, 0], layout, pages, n_pages, rt._num_kv_heads, tail_k, tail_v,
                                      rt.actual_seq_len, scale)

    # ------------------------------------------------------------------ rotated appends
    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                       interleaved: bool = False) -> torch.Tensor:
        """Queries and keys turned by their positions, keys and values appended
        (``TurboPolarKVCacheRuntime.append_rotated``).  Returns the queries, fp16 ``[B, H_q, T, 128]``."""
        return self.runtime.append_rotated(q, k, v, cos, sin, interleaved)

    def update_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                       interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """``append_rotated`` of a prompt or a chunk, and the whole history decompressed, as ``update_and_fetch``
        returns it: (queries, keys, values), all fp16."""
        q, k, v = rotate_tokens(q, k, v, cos, sin, interleaved)
        return (q, *self.update_and_fetch(k, v))

    def decode_rotated(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, cos: torch.Tensor,
                       sin: torch.Tensor, scale: float, interleaved: bool = False,
                       defer_check: bool = False) -> torch.Tensor:
        """``decode_attention`` of a token whose query and key are still to be turned by its position (``cos`` /
        ``sin`` as for ``append_rotated``): two launches in all.  Returns fp16 ``[1, H_q, 128]``."""
        self._validate_decode_shape(q, k_new, v_new, self.config)
        q, k_new, v_new = rotate_tokens(q, k_new, v_new, cos, sin, interleaved)
        return self.decode_attention(q, k_new, v_new, scale, defer_check)

    # ------------------------------------------------------------------ selected pages
    def selected_attention(self, q: torch.Tensor, scale: float, pages: int, first: int = 1, last: int = 1) -> torch.Tensor:
        """One decode step's attention over part of the cache: the queries ``q`` ``[B, H_q, 1, 128]`` of the newest
        tokens (appended before) over ``pages`` stored pages and the dense tail.  Of the pages each kv head takes the
        first ``first``, the last ``last`` and those whose key bounds allow the largest scores to a query head of its
        group (tp_select_pages); a cache of no more pages is attended whole, as by ``decode_attention``.  ``scale`` is
        taken as fp16.  The bounds are kept with the cache (``runtime.page_bounds``).  Returns fp16 ``[B, H_q, 128]``."""
        check_selection(pages, first, last)
        _check_step_query(q, self)
        rt = self.runtime
        rt.resolve_deferred_check()
        n_pages, H = rt.k_storage.block_count, rt._num_kv_heads
        scale, layout = fp16_scale(scale), rt.polar_encoder.layout
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        stored = self._store_pages() if n_pages else None
        if n_pages <= pages:
            tail_k, tail_v = rt._tail_views()
            return decode_attention_store(q[:, :, 0], layout, stored, n_pages, H, tail_k, tail_v, rt.actual_seq_len, scale,
                                          own_workspace=True)
        bounds = rt.page_bounds()
        return selected_attention(q[:, :, 0], layout, stored, n_pages, H, bounds, int(rt._bounds.shape[2]),
                                  tail_args(rt._tail_k, rt._tail_v, rt._tail_len), scale, pages, first, last)[0]

    # ------------------------------------------------------------------ prompts, drafts, branches
    def prompt_attention(self, q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, scale: float,
                         causal: bool = True) -> torch.Tensor:
        """A prompt's, or a chunk's, attention without its score matrix: append ``keys`` /
        ``values`` ``[B, H_kv, T, 128]`` and attend the chunk's ``q`` ``[B, H_q, T, 128]`` over the
        whole history as ``update_and_fetch`` decompresses it (tp_prompt_attention in fp16, the
        cache's type, in which ``q`` is taken too; the scale in 32 bits, as the model's own attention
        takes it).  Returns ``[B, H_q, T, 128]`` of q's type.  No counterpart in the reference, which
        hands the history to the model's attention."""
        for name, t in (("q", q), ("keys", keys), ("values", values)):
            if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[-1] != HEAD_DIM:
                raise ValueError(f"{name} must be [B, H, T, {HEAD_DIM}], got {tuple(getattr(t, 'shape', ()))}")
            if t.dtype not in (torch.float16, torch.bfloat16, torch.float32):
                raise ValueError(f"{name} must be float16, bfloat16 or float32, got {t.dtype}")
        if keys.shape != values.shape or q.shape[0] != keys.shape[0] or q.shape[2] != keys.shape[2]:
            raise ValueError(f"q {tuple(q.shape)}, keys {tuple(keys.shape)} and values {tuple(values.shape)} differ")
        if q.shape[1] < 1 or keys.shape[1] < 1 or q.shape[1] % keys.shape[1]:
            raise ValueError(f"H_q={q.shape[1]} is not a multiple of H_kv={keys.shape[1]}")
        # Before the append: a refused call leaves the cache as it was.
        scale = float(scale)
        if not math.isfinite(c_float(scale).value):
            raise ValueError(f"scale must be finite in 32 bits, got {scale}")
        if not (q.device == keys.device == values.device and q.is_cuda):
            raise ValueError(f"q is on {q.device}, keys on {keys.device}, values on {values.device}; need one HIP device")
        _no_grad(q, keys, values)
        k, v = self.update_and_fetch(keys.to(torch.float16), values.to(torch.float16))
        return prompt_attention(q.to(torch.float16), k, v, scale, causal=causal).to(q.dtype)

    def tree_attention(self, q: torch.Tensor, k_draft: torch.Tensor, v_draft: torch.Tensor, tree: DraftTree,
                       scale: float) -> torch.Tensor:
        """Attention of a tree of drafted tokens: the queries ``q`` ``[B, H_q, T, 128]`` of its nodes
        over every cached token, their ancestors among the drafted ``k_draft`` / ``v_draft`` ``[B,
        H_kv, T, 128]`` and themselves (tp_tree_attention; ``scale`` taken as fp16, as for
        ``decode_attention``).  The cache does not change; ``accept`` takes the nodes that the
        verification keeps.  Returns fp16 ``[B, H_q, T, 128]``."""
        _check_draft(q, k_draft, v_draft, tree)
        rt = self.runtime
        rt.resolve_deferred_check()
        if int(k_draft.shape[1]) != self.config.num_kv_heads:
            raise ValueError(f"draft has {k_draft.shape[1]} KV heads but config expects {self.config.num_kv_heads}")
        if rt._initialized and q.shape[0] != rt._batch_size:
            raise ValueError(f"batch of q ({q.shape[0]}) and cache ({rt._batch_size}) differ")
        n_pages = rt.k_storage.block_count
        tail_k, tail_v = rt._tail_views()
        held = rt.k_storage.radii if n_pages else tail_k
        if held is not None and held.device != q.device:
            raise ValueError(f"q is on {q.device}, the cache on {held.device}")
        return _tree_attention(q, rt.polar_encoder.layout, self._store_pages() if n_pages else None, n_pages, tail_k,
                               tail_v, k_draft, v_draft, tree, fp16_scale(scale))

    def accept(self, k_draft: torch.Tensor, v_draft: torch.Tensor, path: Sequence) -> None:
        """Appends the drafted tokens ``path`` (node indices, root first; ``DraftTree.path_to``)."""
        self.runtime.accept(k_draft.to(torch.float16), v_draft.to(torch.float16), path)

    def truncate(self, tokens: int) -> None:
        """Keeps the first ``tokens`` tokens (``TurboPolarKVCacheRuntime.truncate``)."""
        self.runtime.truncate(tokens)

    def fork(self, tokens: Optional[int] = None, rows: Optional[Sequence[int]] = None,
             pages: Optional[Sequence[int]] = None) -> "TurboPolarFastCache":
        """An independent copy of this cache or a part of it (``TurboPolarKVCacheRuntime.fork``)."""
        other = copy.copy(self)
        other.runtime, other._store = self.runtime.fork(tokens, rows, pages), None
        return other

    def select_rows(self, rows: Sequence[int]) -> None:
        """Makes batch row i what row ``rows[i]`` was."""
        self.runtime.select_rows(rows)
        self._store = None  # holds the replaced buffers

    def keep_pages(self, pages: Sequence[int]) -> None:
        """Compacts the cache to the stored pages ``pages`` and the tail."""
        self.runtime.keep_pages(pages)
        self._store = None

    # ------------------------------------------------------------------ mlx_lm cache protocol
    def size(self) -> int:
        return self.offset

    @property
    def nbytes(self) -> int:
        return int(self.runtime.get_io_telemetry().get("actual_cache_bytes", 0))

    def empty(self) -> bool:
        return self.offset == 0


def _check_step_query(q, cache: TurboPolarFastCache) -> None:
    """The checks of a step's queries ``[B, H_q, 1, 128]`` against the tokens that ``cache`` holds."""
    rt = cache.runtime
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[2] != 1 or q.shape[-1] != HEAD_DIM:
        raise ValueError(f"q must be [B, H_q, 1, {HEAD_DIM}], got {tuple(getattr(q, 'shape', ()))}")
    if not q.is_floating_point():
        raise ValueError(f"q must be a float tensor, got {q.dtype}")
    if not rt.actual_seq_len:
        raise ValueError("nothing to attend: the cache holds no tokens")
    if q.shape[0] != rt._batch_size:
        raise ValueError(f"batch of q ({q.shape[0]}) and cache ({rt._batch_size}) differ")
    if q.shape[1] < 1 or q.shape[1] % rt._num_kv_heads:
        raise ValueError(f"H_q={q.shape[1]} is not a multiple of H_kv={rt._num_kv_heads}")
    held = rt.k_storage.radii if rt.k_storage.block_count else rt._tail_k
    if not q.is_cuda or held.device != q.device:
        raise ValueError(f"q is on {q.device}, the cache on {held.device}; need one HIP device")
    _no_grad(q)


def make_turbo_caches(num_layers: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                      use_qjl: bool = False) -> List[TurboPolarFastCache]:
    """One cache per layer in the benchmark layout of the reference
    (turbopolar_fast_attention.py:207-229): int8 log radii, split 0, 8-bit
    deep angles, quantised V, pages of 64."""
    if head_dim not in (64, 128):
        raise ValueError(f"TurboPolar only supports head_dim 64 or 128, got {head_dim}")
    config = TurboPolarConfig(
        num_q_heads=num_q_heads, num_kv_heads=num_kv_heads, head_dim=head_dim, block_size=64,
        qjl_proj_dim=32 if head_dim == 64 else 64, use_qjl=use_qjl, storage_mode="kv_quant",
        use_int8_radii=True, k_angle_bits_deep=8, split_dim=0,
    )
    return [TurboPolarFastCache(config) for _ in range(num_layers)]
