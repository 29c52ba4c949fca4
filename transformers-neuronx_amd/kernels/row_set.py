"""Rows of several tensors that are copied together: what a page (or a slot) is across all layers of a cache."""
from typing import List, Optional, Sequence

import numpy as np
import torch


class RowSet:
    """Tensors whose dimension 0 counts rows, all of them in step: row 7 is page 7 of every layer's keys and values.

    tensors      on one device; the rows of a tensor may lie apart, a row itself is contiguous
    token_axes   for each tensor the dimension that counts the places of tokens, which `copy_rows` may bound, or None for a
                 tensor whose rows are always copied whole; left out: None for all
    targets      the tensors that rows are copied to, of the same types and shapes but for the number of rows; left out: the
                 tensors themselves
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
        words, places = [], set()
        for t, axis, to in zip(self.tensors, self.token_axes, self.targets):
            for x in (t, to):
                if x.device != self.device:
                    raise ValueError(f"the tensors of a set of rows lie on one device, got {self.device} and {x.device}")
                if x.dim() < 1 or x.numel() == 0:
                    raise ValueError(f"a set of rows takes tensors with rows in them, got shape {tuple(x.shape)}")
                if not x[0].is_contiguous() or (x.shape[0] > 1 and x.stride(0) < x[0].numel()):
                    raise ValueError("a row has to be contiguous, and rows may not overlap")
            if to.dtype != t.dtype or to.shape[1:] != t.shape[1:]:
                raise ValueError(f"rows of {t.dtype} {tuple(t.shape[1:])} cannot go to rows of {to.dtype} {tuple(to.shape[1:])}")
            item, shape = t.element_size(), list(t.shape)
            row = int(np.prod(shape[1:], dtype=np.int64)) * item
            if row >= 2 ** 31:
                raise ValueError(f"a row of {row} bytes is more than copy_rows takes (2 GiB)")
            if axis is None:
                run, inner, outer = row, 0, 1
            else:
                if not 0 < axis < t.dim():
                    raise ValueError(f"the token axis of a tensor of shape {tuple(t.shape)} is one of 1 to {t.dim() - 1}, got {axis}")
                inner = int(np.prod(shape[axis + 1:], dtype=np.int64)) * item
                run = shape[axis] * inner
                outer = row // run
                places.add(shape[axis])
            distances = [t.data_ptr(), to.data_ptr(), run]
            distances += [x.stride(0) * item for x in (t, to) if x.shape[0] > 1]
            grain = next(g for g in (16, 4, 2, 1) if all(d % g == 0 for d in distances))
            words.append([t.data_ptr(), to.data_ptr(), t.stride(0) * item, to.stride(0) * item, run, inner, outer, grain])
        if len(places) > 1:
            raise ValueError(f"the token axes of a set of rows are of one length, got {sorted(places)}")
        self.places: Optional[int] = places.pop() if places else None
        self.num_rows = min(t.shape[0] for t in self.tensors)
        self.num_target_rows = min(t.shape[0] for t in self.targets)
        self.row_bytes = sum(w[4] * w[6] for w in words)
        self.largest = max(w[4] * w[6] for w in words)
        self.words = np.array(words, dtype=np.int64)
        self.table: Optional[torch.Tensor] = None          # the words on the device, put there by the backend

    def pairs(self, sources: Sequence[int], targets: Sequence[int], tokens=None) -> np.ndarray:
        """int32 `[n, 3]` (source, target, tokens; -1: all), checked: rows there are, no target named twice, and within the
        same tensors no target that is a source."""
        src, dst = np.asarray(sources, dtype=np.int64).reshape(-1), np.asarray(targets, dtype=np.int64).reshape(-1)
        n = src.size
        if dst.size != n:
            raise ValueError(f"{n} sources and {dst.size} targets")
        out = np.empty((n, 3), dtype=np.int32)
        if n == 0:
            return out
        for what, rows, most in (("source", src, self.num_rows), ("target", dst, self.num_target_rows)):
            if rows.min() < 0 or rows.max() >= most:
                bad = rows.min() if rows.min() < 0 else rows.max()
                raise ValueError(f"{what} row {int(bad)} is outside the {most} rows there are")
        if n > 1 and np.unique(dst).size != n:
            raise ValueError("a target row is named twice")
        if self.in_place and np.isin(dst, src).any():
            raise ValueError("a row is both source and target")
        out[:, 0], out[:, 1] = src, dst
        if tokens is None:
            out[:, 2] = -1
            return out
        if self.places is None:
            raise ValueError("no tensor of this set counts tokens")
        held = np.asarray(tokens, dtype=np.int64).reshape(-1)
        if held.size == 1:
            held = np.broadcast_to(held, (n,))
        if held.size != n:
            raise ValueError(f"{n} pairs of rows and {held.size} numbers of tokens")
        if held.min() < 0 or held.max() > self.places:
            raise ValueError(f"a row holds 0 to {self.places} tokens, got {int(held.min())} to {int(held.max())}")
        out[:, 2] = held
        return out
