"""``DraftTree``: which drafted tokens see which.

A draft is a tree of tokens that continue a cache: node i hangs on node
``parents[i]``, or on the cache's last token where that is -1, and parents come
before their children.  A node's query attends everything that the cache holds, its
ancestors and itself.  The tree is validated and turned into ancestor bit masks once
(``include/turbopolar.h``, tp_tree_attention); a program that drafts the same shape at
every step keeps it.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import torch

from ._lib import stream_handle

MAX_NODES = 256


class DraftTree:
    """``parents``: one parent per node, or one such list per batch row.  Lists of
    different lengths are padded; a padding node's output row is 0.  ``device``: where
    the masks are put at once (otherwise at the first call on a device, by a copy that
    waits).  A captured graph reads the masks: keep the tree as long as the graph."""

    def __init__(self, parents: Sequence, device=None):
        rows = list(parents)
        self.shared = not rows or not isinstance(rows[0], (list, tuple))
        lists = [rows] if self.shared else rows
        self.parents: List[List[int]] = []
        for row in lists:
            if not isinstance(row, (list, tuple)):
                raise TypeError("DraftTree takes a list of parents, or one such list per batch row")
            for p in row:
                if isinstance(p, bool) or not isinstance(p, int):
                    raise TypeError(f"parents must be ints, got {type(p).__name__}")
            row = [int(p) for p in row]
            bad = [i for i, p in enumerate(row) if not -1 <= p < i]
            if bad:
                raise ValueError(f"node {bad[0]} hangs on {row[bad[0]]}: a parent is -1 or an earlier node")
            self.parents.append(row)
        self.nodes = max((len(row) for row in self.parents), default=0)
        if not 1 <= self.nodes <= MAX_NODES:
            raise ValueError(f"a draft holds 1 to {MAX_NODES} nodes, got {self.nodes}")
        #: Batch rows with a tree of their own (None: one tree for every row).
        self.batch: Optional[int] = None if self.shared else len(self.parents)
        words = -(-self.nodes // 64)
        table = []
        for row in self.parents:
            sees: List[int] = []
            for i, p in enumerate(row):
                sees.append((sees[p] if p >= 0 else 0) | (1 << i))
            sees += [0] * (self.nodes - len(sees))
            table.append([[_signed((s >> (64 * w)) & (2 ** 64 - 1)) for w in range(words)] for s in sees])
        self._mask = torch.tensor(table, dtype=torch.int64)  # [1 or batch, nodes, words]
        self._on: Dict[torch.device, Tuple[torch.Tensor, int]] = {}
        if device is not None:
            self.mask_on(torch.device(device))

    def mask_on(self, device: torch.device) -> torch.Tensor:
        """The masks on ``device``, int64 ``[1 or batch, nodes, words]``, for a call on its current
        stream."""
        hit = self._on.get(device)
        if hit is None:
            if device.type != "cuda":
                return self._mask
            if device.index is None:
                return self.mask_on(torch.device("cuda", torch.cuda.current_device()))
            hit = self._on[device] = (self._mask.to(device), stream_handle(device))
        mask, stream = hit
        if stream_handle(device) != stream and not torch.cuda.is_current_stream_capturing():
            # The tree may go while that call still reads.
            mask.record_stream(torch.cuda.current_stream(device))
        return mask

    def depths(self, row: int = 0) -> List[int]:
        """Tokens between the cache's last one and each node: node i sits at position
        ``cache.offset + depths()[i]``."""
        out: List[int] = []
        for p in self.parents[row]:
            out.append(out[p] + 1 if p >= 0 else 0)
        return out

    def path_to(self, node: int, row: int = 0) -> List[int]:
        """The nodes from the root to ``node``: what ``accept`` takes when ``node`` is the
        last accepted one."""
        parents = self.parents[row]
        if not 0 <= node < len(parents):
            raise IndexError(f"node {node} outside the {len(parents)} of the draft")
        path = []
        while node >= 0:
            path.append(node)
            node = parents[node]
        return path[::-1]


def _signed(word: int) -> int:
    return word - 2 ** 64 if word >= 2 ** 63 else word
