"""Rows of several tensors that are copied together: what a page (or a slot) is across all layers of a cache."""
import math
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch


class RowSet:
    """Tensors whose dimension 0 counts rows, all of them in step: row 7 is page 7 of every layer's keys and values.

    tensors      on one device; the rows of a tensor may lie apart, a row itself is contiguous
    token_axes   for each tensor the dimension that counts the places of tokens, which `copy_rows` may bound, or None for a
                 tensor whose rows are always copied whole; left out: None for all
    targets      the tensors that rows are copied to, of the same types and shapes but for the number of rows; left out: the
                 tensors themselves

    No two of them lie in the same memory, and none between another's first and last row: what is copied would depend on which is
    copied first.
    """

    def __init__(self, tensors: Sequence[torch.Tensor], token_axes: Optional[Sequence[Optional[int]]] = None,
                 targets: Optional[Sequence[torch.Tensor]] = None):
        self.tensors: List[torch.Tensor] = list(tensors)
        self.in_place = targets is None
        self.targets: List[torch.Tensor] = self.tensors if targets is None else list(targets)
        self.token_axes = [None] * len(self.tensors) if token_axes is None else list(token_axes)
        if not self.tensors:
            raise ValueError("a set of rows needs at least one tensor")
        if not len(self.tensors) == len(self.token_axes) == len(self.targets):
            raise ValueError(f"{len(self.tensors)} tensors, {len(self.token_axes)} token axes, {len(self.targets)} targets")
        self.device = self.tensors[0].device
        words, places, spans = [], set(), []
        for t, axis, to in zip(self.tensors, self.token_axes, self.targets):
            at, apart, shape, item = self._layout(t)
            to_at, to_apart, to_shape, _ = (at, apart, shape, item) if to is t else self._layout(to)
            if to.dtype != t.dtype or to_shape[1:] != shape[1:]:
                raise ValueError(f"rows of {t.dtype} {shape[1:]} cannot go to rows of {to.dtype} {to_shape[1:]}")
            row = math.prod(shape[1:]) * item
            if row >= 2 ** 31:
                raise ValueError(f"a row of {row} bytes is more than copy_rows takes (2 GiB)")
            if axis is None:
                run, inner, outer = row, 0, 1
            else:
                if not 0 < axis < len(shape):
                    raise ValueError(f"the token axis of a tensor of shape {shape} is one of 1 to {len(shape) - 1}, got {axis}")
                inner = math.prod(shape[axis + 1:]) * item
                run = shape[axis] * inner
                outer = row // run
                places.add(shape[axis])
            distances = at | to_at | run | (apart if shape[0] > 1 else 0) | (to_apart if to_shape[0] > 1 else 0)
            grain = next(g for g in (16, 4, 2, 1) if distances % g == 0 and (g == 16 or inner % g == 0))
            words.append((at, to_at, apart, to_apart, run, inner, outer, grain))
            spans.append((at, at + (shape[0] - 1) * apart + row))
            if not self.in_place:
                spans.append((to_at, to_at + (to_shape[0] - 1) * to_apart + row))
        spans.sort()
        if any(end > begin for (_, end), (begin, _) in zip(spans, spans[1:])):
            raise ValueError("two tensors of a set of rows share memory")
        if len(places) > 1:
            raise ValueError(f"the token axes of a set of rows are of one length, got {sorted(places)}")
        self.places: Optional[int] = places.pop() if places else None
        self.num_rows = min(t.shape[0] for t in self.tensors)
        self.num_target_rows = min(t.shape[0] for t in self.targets)
        self._rows = [tuple(w[4:7]) for w in words]
        self.row_bytes = self.bytes_of(-1)
        self._shapes = sorted({tuple(w[4:]) for w in words})
        self.words = np.array(words, dtype=np.int64)
        self.table = None                                  # the words on the device, put there by the backend

    def _layout(self, x: torch.Tensor):
        """(address, bytes from row to row, shape, bytes of an element), of rows that are what they have to be."""
        shape, strides, item = tuple(x.shape), x.stride(), x.element_size()
        if x.device != self.device:
            raise ValueError(f"the tensors of a set of rows lie on one device, got {self.device} and {x.device}")
        if not shape or 0 in shape:
            raise ValueError(f"a set of rows takes tensors with rows in them, got shape {shape}")
        count = 1
        for n, s in zip(shape[:0:-1], strides[:0:-1]):
            if n > 1 and s != count:
                raise ValueError("a row has to be contiguous")
            count *= n
        if shape[0] > 1 and strides[0] < count:
            raise ValueError("rows may not overlap")
        return x.data_ptr(), strides[0] * item, shape, item

    def bytes_of(self, tokens: int) -> int:
        """What is copied of a row that holds `tokens` tokens (below zero: all of it), in all tensors."""
        return sum((run if tokens < 0 or inner == 0 else min(run, tokens * inner)) * outer for run, inner, outer in self._rows)

    def units(self, tokens: int) -> int:
        """Pieces of at most 16 bytes in what is copied of the largest row where it holds `tokens` tokens (below zero: all)."""
        most = 0
        for run, inner, outer, grain in self._shapes:
            length = run if tokens < 0 or inner == 0 else min(run, tokens * inner)
            most = max(most, -(-length * outer // grain) if length == run else -(-length // grain) * outer)
        return most

    def pairs(self, sources: Sequence[int], targets: Sequence[int], tokens=None) -> List[Tuple[int, int, int]]:
        """(source, tokens, target), tokens -1 for all, ordered by them, and checked: rows there are, no target named twice, and
        within the same tensors no target that is a source."""
        src, dst = [int(s) for s in sources], [int(d) for d in targets]
        n = len(src)
        if len(dst) != n:
            raise ValueError(f"{n} sources and {len(dst)} targets")
        if n == 0:
            return []
        for what, rows, most in (("source", src, self.num_rows), ("target", dst, self.num_target_rows)):
            low, high = min(rows), max(rows)
            if low < 0 or high >= most:
                raise ValueError(f"{what} row {low if low < 0 else high} is outside the {most} rows there are")
        into = set(dst)
        if len(into) != n:
            raise ValueError("a target row is named twice")
        if self.in_place and not into.isdisjoint(src):
            raise ValueError("a row is both source and target")
        if tokens is None:
            held = [-1] * n
        else:
            if self.places is None:
                raise ValueError("no tensor of this set counts tokens")
            held = [int(tokens)] * n if isinstance(tokens, (int, np.integer)) else [int(t) for t in tokens]
            if len(held) != n:
                raise ValueError(f"{n} pairs of rows and {len(held)} numbers of tokens")
            if min(held) < 0 or max(held) > self.places:
                raise ValueError(f"a row holds 0 to {self.places} tokens, got {min(held)} to {max(held)}")
        return sorted(zip(src, held, dst))

    @staticmethod
    def groups(pairs: List[Tuple[int, int, int]]) -> Tuple[List[List[int]], List[int]]:
        """([source, tokens, first target, targets] of every source with its tokens, the targets)."""
        heads: List[List[int]] = []
        for i, (s, n, _) in enumerate(pairs):
            if heads and heads[-1][0] == s and heads[-1][1] == n:
                heads[-1][3] += 1
            else:
                heads.append([s, n, i, 1])
        return heads, [d for _, _, d in pairs]
