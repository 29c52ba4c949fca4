"""Inputs for the tests of steered logits and scored tokens, and what comes of them in 64 bits, written out row by row."""
import numpy as np
import torch


def random_rules(rows, vocab, seen, biases, allowed, seed):
    """A batch's logits with some odd values among them, its rules, histories, masks and the tokens chosen last."""
    rng = np.random.default_rng(seed)
    slots = rows + 2
    logits = rng.normal(0, 3, (rows, vocab)).astype(np.float32)
    if vocab > 8:
        logits[:, rng.integers(0, vocab)] = -np.inf
        logits[rng.integers(0, rows), rng.integers(0, vocab)] = np.inf
        logits[0, 3] = 0.0
    seen = min(seen, vocab)
    used = rng.integers(0, seen + 1, slots).astype(np.int32)
    used[0] = seen
    entries = np.zeros((slots, vocab, 2), dtype=np.int32)          # a vocabulary's worth: never too few
    for s in range(slots):
        entries[s, :used[s], 0] = rng.choice(vocab, used[s], replace=False)
        entries[s, :used[s], 1] = rng.integers(1, 8, used[s])
    last = rng.integers(0, vocab, slots).astype(np.int32)
    last[rng.random(slots) < 0.3] = -1
    mine = rng.permutation(slots)[:rows]
    if rows > 2:
        mine[1] = -1
    rules = dict(slots=mine.tolist(), repetition=np.round(rng.uniform(0.5, 2, rows), 3).tolist(),
                 presence=np.round(rng.uniform(-1, 1, rows), 3).tolist(), frequency=np.round(rng.uniform(-1, 1, rows), 3).tolist())
    lists = []
    for _ in range(rows):
        ids = rng.choice(vocab, int(rng.integers(0, min(biases, vocab) + 1)), replace=False)
        lists.append({int(t): (-np.inf if rng.random() < 0.1 else float(np.float32(rng.normal(0, 4)))) for t in ids})
    rules["biases"] = lists
    kinds = max(1, rows - 1)
    bits = rng.random((kinds, -(-vocab // 32) * 32)) < allowed     # bits behind the vocabulary may be set
    masks = np.packbits(bits, axis=1, bitorder="little").view("<i4").astype(np.int32)
    rules["mask_rows"] = [-1 if allowed < 0 or (rows > 3 and i == 2) else i % kinds for i in range(rows)]
    case = dict(rows=rows, vocab=vocab, logits=logits, entries=entries, used=used, last=last, rules=rules, masks=masks)
    case["scale"] = np.abs(np.where(np.isfinite(logits), logits, 0)).astype(np.float64) * 2 + 20    # what a rounding is half a step of
    return case


def history_tensors(case, device):
    return torch.from_numpy(case["entries"].copy()).to(device), torch.from_numpy(case["used"].copy()).to(device)


def adjusted(case):
    """(logits in 64 bits, entries, used) behind the step."""
    x, entries, used, rules = case["logits"].astype(np.float64), case["entries"].copy(), case["used"].copy(), case["rules"]
    for r in range(case["rows"]):
        slot = rules["slots"][r]
        rho, presence, frequency = (np.float64(np.float32(rules[k][r])) for k in ("repetition", "presence", "frequency"))
        if slot >= 0:
            token = int(case["last"][slot])
            if token >= 0:
                for i in range(used[slot]):
                    if entries[slot, i, 0] == token:
                        entries[slot, i, 1] += 2
                        break
                else:
                    entries[slot, used[slot]] = token, 2
                    used[slot] += 1
            for i in range(used[slot]):
                t, times = int(entries[slot, i, 0]), int(entries[slot, i, 1]) // 2
                v = x[r, t] / rho if x[r, t] > 0 else x[r, t] * rho
                x[r, t] = v - frequency * times - (presence if times else 0.0)
        for t, b in rules["biases"][r].items():
            x[r, t] = -np.inf if b == -np.inf else x[r, t] + b
        if rules["mask_rows"][r] >= 0:
            words = case["masks"][rules["mask_rows"][r]]
            for t in range(case["vocab"]):
                if not (int(words[t // 32]) >> (t % 32)) & 1:
                    x[r, t] = -np.inf
    return x, entries, used


def log_probs_in_64(logits, tokens, top):
    """(log-probabilities of the tokens, the largest logits' tokens, theirs), by the rules for odd values."""
    rows, vocab = logits.shape
    out, ids, best = np.empty(rows), np.empty((rows, top), dtype=np.int32), np.empty((rows, top))
    for r in range(rows):
        x = np.where(np.isnan(logits[r]), -np.inf, logits[r].astype(np.float64))
        m = x.max()
        if m == -np.inf:
            lp = np.full(vocab, -np.inf)
        elif m == np.inf:
            lp = np.where(x == m, -np.log((x == m).sum()), -np.inf)
        else:
            lp = x - m - np.log(np.exp(x - m).sum())
        t = int(tokens[r])
        out[r] = lp[t] if 0 <= t < vocab else -np.inf
        order = sorted(range(vocab), key=lambda i: (-x[i], i))[:top] if top else []
        ids[r], best[r] = order, lp[order]
    return out, ids, best
