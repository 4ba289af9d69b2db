"""``SharedPrefixCache`` -- a batch of sequences behind one prefix that is stored once.

Samples of one prompt, requests behind one system prompt or questions about one document share their first
tokens.  ``TurboPolarFastCache.fork`` gives each of them a copy; here the prefix stays one cache of batch 1, which
attention reads and decodes once for the whole batch, and each sequence keeps only the tokens of its own (a cache of
batch B).  No counterpart in the reference, which keeps one line of tokens per cache.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from .fast_attention import TurboPolarFastCache
from .kernels import HEAD_DIM, _no_grad, fp16_scale, shared_attention, tail_args


def _layout_of(cache: TurboPolarFastCache) -> tuple:
    x = cache.runtime.polar_encoder.layout
    return x.int8_radii, x.l1_bits, x.deep_bits, x.split_dim


class SharedPrefixCache:
    """``prefix``: the cache of the common tokens, of batch 1; it is not copied and must not change while branches
    read it: where its length is another, or others took the place of tokens that were cut from it, calls raise.  ``own``:
    the sequences' own tokens, a cache of the same layout and heads (a new one by default, whose batch the first append
    fixes)."""

    def __init__(self, prefix: TurboPolarFastCache, own: Optional[TurboPolarFastCache] = None):
        for name, cache in (("prefix", prefix), ("own", own)):
            if cache is not None and not isinstance(cache, TurboPolarFastCache):
                raise TypeError(f"{name} must be a TurboPolarFastCache, got {type(cache).__name__}")
        if own is prefix:
            raise ValueError("the prefix cannot be the sequences' own cache")
        prefix.runtime.resolve_deferred_check()
        if prefix.runtime._initialized and prefix.runtime._batch_size != 1:
            raise ValueError(f"a shared prefix is a cache of batch 1, got {prefix.runtime._batch_size}")
        own = TurboPolarFastCache(prefix.config) if own is None else own
        if _layout_of(own) != _layout_of(prefix) or own.config.num_kv_heads != prefix.config.num_kv_heads:
            raise ValueError("the prefix and the sequences' own cache must have one layout and number of KV heads")
        self.prefix, self.own, self.config = prefix, own, prefix.config
        self.prefix_tokens = prefix.offset
        self._shared = prefix.runtime, prefix.runtime.mark()

    @property
    def offset(self) -> int:
        """Tokens of each sequence, the prefix's among them (the position that the next token takes)."""
        return self.prefix_tokens + self.own.offset

    # ------------------------------------------------------------------ the sequences' own tokens
    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Appends ``[B, H_kv, T, 128]``, T tokens to each sequence, in fp16."""
        self.own.runtime.append(k.to(torch.float16), v.to(torch.float16))

    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                       interleaved: bool = False) -> torch.Tensor:
        """``TurboPolarFastCache.append_rotated``, T tokens to each sequence (positions from ``offset`` on)."""
        return self.own.append_rotated(q, k, v, cos, sin, interleaved)

    def truncate(self, tokens: int) -> None:
        """Keeps the first ``tokens`` tokens of each sequence, at least the prefix."""
        if isinstance(tokens, bool) or not isinstance(tokens, int):
            raise TypeError(f"tokens must be an int, got {type(tokens).__name__}")
        if not self.prefix_tokens <= tokens <= self.offset:
            raise ValueError(f"cannot keep {tokens} of {self.offset} tokens, {self.prefix_tokens} of them the prefix")
        self.own.truncate(tokens - self.prefix_tokens)

    def select_rows(self, rows: Sequence[int]) -> None:
        """Makes sequence i what sequence ``rows[i]`` was; the prefix stays where it is."""
        if self.own.runtime._initialized:
            self.own.select_rows(rows)

    def fork(self, rows: Optional[Sequence[int]] = None) -> "SharedPrefixCache":
        """Branches of these sequences behind the same prefix (``TurboPolarFastCache.fork`` of their own tokens)."""
        self._check_prefix()
        return SharedPrefixCache(self.prefix, self.own.fork(rows=rows if self.own.runtime._initialized else None))

    # ------------------------------------------------------------------ attention
    def _check_prefix(self) -> None:
        if self.prefix.offset != self.prefix_tokens:
            raise ValueError(f"the prefix held {self.prefix_tokens} tokens when it was shared and holds "
                             f"{self.prefix.offset} now")
        runtime, mark = self._shared
        if self.prefix.runtime is not runtime or runtime.kept_since(mark) < self.prefix_tokens:
            raise ValueError("the prefix was cut and filled again after it was shared: its tokens are others")

    def attention(self, q: torch.Tensor, scale: float) -> torch.Tensor:
        """One decode step's attention: the queries ``q`` ``[B, H_q, 1, 128]`` over the prefix and each sequence's own
        tokens (tp_shared_attention; ``scale`` taken as fp16, as for ``TurboPolarFastCache.decode_attention``).
        Returns fp16 ``[B, H_q, 128]``."""
        scale = self._check_step(q, scale)
        if not self.offset:
            raise ValueError("nothing to attend: the prefix and the sequences hold no tokens")
        return self._attend(q, scale)

    def _attend(self, q: torch.Tensor, scale: float) -> torch.Tensor:
        parts = []
        for cache in (self.prefix, self.own):
            rt = cache.runtime
            n_pages, tokens = rt.k_storage.block_count, rt._tail_len
            parts.append((cache._store_pages() if n_pages else None, n_pages, tail_args(rt._tail_k, rt._tail_v, tokens)))
        return shared_attention(q, self.prefix.runtime.polar_encoder.layout, self.config.num_kv_heads, *parts, scale)

    def _check_step(self, q: torch.Tensor, scale: float) -> float:
        """The checks of a step's queries against what is held; ``scale`` in fp16."""
        if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.shape[2] != 1 or q.shape[-1] != HEAD_DIM:
            raise ValueError(f"q must be [B, H_q, 1, {HEAD_DIM}], got {tuple(getattr(q, 'shape', ()))}")
        if not q.is_floating_point():
            raise ValueError(f"q must be a float tensor, got {q.dtype}")
        B, Hq, heads = int(q.shape[0]), int(q.shape[1]), self.config.num_kv_heads
        if B < 1 or Hq < 1 or Hq % heads:
            raise ValueError(f"H_q={Hq} is not a multiple of H_kv={heads}, or the batch is empty")
        self._check_prefix()
        scale = fp16_scale(scale)
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        for name, cache, rows in (("prefix", self.prefix, 1), ("own cache", self.own, B)):
            rt = cache.runtime
            rt.resolve_deferred_check()
            if rt.actual_seq_len and rt._batch_size != rows:
                raise ValueError(f"batch of q ({B}) and of the {name} ({rt._batch_size}) do not match")
            held = rt.k_storage.radii if rt.k_storage.block_count else rt._tail_k
            if rt.actual_seq_len and (held.device != q.device or not q.is_cuda):
                raise ValueError(f"q is on {q.device}, the {name} on {held.device}; need one HIP device")
        _no_grad(q)
        return scale

    def decode_attention(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, scale: float) -> torch.Tensor:
        """Appends a token to each sequence (``[B, H_kv, 1, 128]``) and attends; a refused call leaves the sequences as
        they were."""
        if k_new.dim() != 4 or k_new.shape[2] != 1 or q.dim() != 4 or q.shape[0] != k_new.shape[0]:
            raise ValueError("decode_attention only supports a single query/key/value token")
        scale = self._check_step(q, scale)
        if k_new.device != q.device or not q.is_cuda:
            raise ValueError(f"q is on {q.device}, the new token on {k_new.device}; need one HIP device")
        self.append(k_new, v_new)
        return self._attend(q, scale)
