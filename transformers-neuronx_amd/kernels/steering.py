"""What steers the choice of a batch's tokens: the histories that penalties go by, and the rules of each row."""
from typing import Dict, List, Optional, Sequence

import numpy as np
import torch


class TokenHistory:
    """The tokens of live sequences, one history a slot: its distinct tokens in the order of their first appearance.

    entries  int32 `[slots, capacity, 2]`: (token, twice the times it was chosen + 1 if the prompt has it)
    used     int32 `[slots]`: entries of each slot that count

    A vocabulary's worth of entries never fills up; fewer do where a sequence cannot hold as many tokens."""

    def __init__(self, entries: torch.Tensor, used: torch.Tensor):
        if entries.dim() != 3 or entries.shape[2] != 2 or entries.dtype != torch.int32 or not entries.is_contiguous():
            raise ValueError(f"entries are contiguous int32 [slots, capacity, 2], got {entries.dtype} {tuple(entries.shape)}")
        if used.dtype != torch.int32 or used.shape != entries.shape[:1] or used.device != entries.device or not used.is_contiguous():
            raise ValueError(f"used is int32 [{entries.shape[0]}] beside the entries, got {used.dtype} {tuple(used.shape)}")
        if entries.numel() == 0 or entries.data_ptr() % 8:
            raise ValueError("a history needs at least one slot and one entry, and begins on 8 bytes")
        self.entries, self.used = entries, used
        self.slots, self.capacity = entries.shape[0], entries.shape[1]

    @staticmethod
    def distinct(prompt: Sequence[int], output: Sequence[int] = ()) -> np.ndarray:
        """int32 `[n, 2]`: the entries of a sequence's tokens, those of the prompt and those chosen after it."""
        tokens = np.concatenate([np.asarray(prompt, dtype=np.int64).reshape(-1), np.asarray(output, dtype=np.int64).reshape(-1)])
        split = len(tokens) - len(output)
        if tokens.size == 0:
            return np.zeros((0, 2), dtype=np.int32)
        ids, first, which = np.unique(tokens, return_index=True, return_inverse=True)
        if ids[0] < 0 or ids[-1] >= 2 ** 31:
            raise ValueError(f"a token is a number from 0 to 2^31 - 1, got {int(ids[0] if ids[0] < 0 else ids[-1])}")
        times = np.bincount(which.reshape(-1)[split:], minlength=len(ids))
        order = np.argsort(first)
        out = np.empty((len(ids), 2), dtype=np.int32)
        out[:, 0], out[:, 1] = ids[order], (2 * times + (first < split))[order]
        return out


class LogitRules:
    """The rules of a batch's rows, checked and laid out in one array of 32-bit words: what `adjust_logits` takes. One stays good
    for as long as the rows keep their slots, their numbers and their masks' places; histories and masks may change under it.

    vocab        tokens a row has logits for
    slots        the slot of each row's history, below zero for a row that keeps none (left out: none does); no two rows share one
    repetition   a row's logits above zero are divided by it, others multiplied, for every token of its history (1: no change)
    presence     subtracted from the logit of every token that was chosen before (the prompt's do not count)
    frequency    subtracted as many times as the token was chosen
    biases       a row's {token: what is added to its logit} (-inf bars it), or None
    mask_rows    which of the masks says what a row may choose; below zero: anything
    """

    WORDS = 8

    def __init__(self, vocab: int, rows: int, slots: Optional[Sequence[int]] = None, repetition=None, presence=None, frequency=None,
                 biases: Optional[Sequence[Optional[Dict[int, float]]]] = None, mask_rows: Optional[Sequence[int]] = None):
        def column(name, values, default, dtype):
            a = np.full(rows, default, dtype=np.float64 if dtype == np.float32 else np.int64)
            if values is not None:
                if len(values) != rows:
                    raise ValueError(f"{name}: {len(values)} values for {rows} rows")
                a[:] = values
            if dtype == np.float32 and not (np.isfinite(a).all() and (np.abs(a) <= np.finfo(np.float32).max).all()):
                raise ValueError(f"{name} has to be a finite number")
            return a
        if vocab <= 0 or vocab >= 2 ** 31 or rows < 0:
            raise ValueError(f"bad sizes: {rows} rows of {vocab} logits")
        self.vocab, self.rows = vocab, rows
        self.slots = column("slots", slots, -1, np.int64)
        rho = column("repetition", repetition, 1.0, np.float32)
        if rows and not (rho.astype(np.float32) >= np.finfo(np.float32).tiny).all():
            raise ValueError("repetition has to be above zero")
        held = self.slots[self.slots >= 0]
        if np.unique(held).size != held.size:
            raise ValueError("two rows name one slot: a history is entered by one row at a time")
        masks = column("mask_rows", mask_rows, -1, np.int64)
        if rows and max(self.slots.max(), masks.max()) >= 2 ** 31:
            raise ValueError("a slot or a mask is out of range")
        self.most_slot = int(self.slots.max()) if rows else -1
        self.most_mask = int(masks.max()) if rows else -1
        if biases is not None and len(biases) != rows:
            raise ValueError(f"biases: {len(biases)} values for {rows} rows")
        starts = np.zeros(rows + 1, dtype=np.int64)
        if biases is not None:
            np.cumsum([len(row) if row else 0 for row in biases], out=starts[1:])
        ids, add = np.empty(starts[-1], dtype=np.int64), np.empty(starts[-1], dtype=np.float64)
        for i, row in enumerate(biases or ()):
            if row:
                a, b = starts[i], starts[i + 1]
                ids[a:b], add[a:b] = np.fromiter(row.keys(), np.int64, b - a), np.fromiter(row.values(), np.float64, b - a)
        if ids.size:
            if ids.min() < 0 or ids.max() >= vocab:
                bad = ids.min() if ids.min() < 0 else ids.max()
                raise ValueError(f"a bias names token {int(bad)}, outside the vocabulary of {vocab}")
            if np.isnan(add).any() or (add > np.finfo(np.float32).max).any() or (np.isfinite(add) & (add < -np.finfo(np.float32).max)).any():
                raise ValueError("a bias is a finite number, or -inf for a token that must not be chosen")
        n, self.num_biases = rows * self.WORDS, int(ids.size)
        flat = np.zeros(n + 2 * self.num_biases, dtype=np.int32)
        head = flat[:n].reshape(rows, self.WORDS)
        head[:, 0] = np.maximum(self.slots, -1)
        for at, a in ((1, rho), (2, column("presence", presence, 0.0, np.float32)), (3, column("frequency", frequency, 0.0, np.float32))):
            head[:, at] = a.astype(np.float32).view(np.int32)
        head[:, 4], head[:, 5] = starts[:-1], starts[1:]
        head[:, 6] = np.maximum(masks, -1)
        flat[n:n + self.num_biases] = ids
        flat[n + self.num_biases:] = add.astype(np.float32).view(np.int32)
        self.flat = flat
        self.mask_words = mask_words(vocab)
        self.tokens_at, self.values_at = 4 * n, 4 * (n + self.num_biases)      # bytes before the biases' tokens, and their values
        self.device_words = None                              # put there by the backend

    def pieces(self, words):
        """(rules, bias tokens, bias values) of the words, in whatever memory they lie."""
        n = self.rows * self.WORDS
        return words[:n], words[n:n + self.num_biases], words[n + self.num_biases:]


def mask_words(vocab: int) -> int:
    """32-bit words of a mask over `vocab` tokens."""
    return -(-vocab // 32)


def pack_mask(vocab: int, allowed) -> np.ndarray:
    """int32 `[mask_words(vocab)]`, bit t % 32 of word t // 32 set where token t may be chosen. `allowed`: the token ids, or a
    boolean for every token."""
    a = np.asarray(sorted(allowed) if isinstance(allowed, (set, frozenset)) else allowed)
    if a.dtype == bool:
        if a.shape != (vocab,):
            raise ValueError(f"a mask has a truth value for each of the {vocab} tokens, got shape {a.shape}")
        bits = a
    else:
        if a.size and a.dtype.kind not in "iu":
            raise ValueError(f"allowed tokens are whole numbers, or a truth value for each of the {vocab}, got {a.dtype}")
        ids = a.astype(np.int64).reshape(-1)
        if ids.size and (ids.min() < 0 or ids.max() >= vocab):
            bad = ids.min() if ids.min() < 0 else ids.max()
            raise ValueError(f"token {int(bad)} is outside the vocabulary of {vocab}")
        bits = np.zeros(vocab, dtype=bool)
        bits[ids] = True
    whole = np.zeros(mask_words(vocab) * 32, dtype=bool)
    whole[:vocab] = bits
    return np.packbits(whole, bitorder="little").view("<i4").astype(np.int32)
