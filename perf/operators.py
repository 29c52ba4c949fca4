"""What is measured of the operators that let several answers share a prompt: pages copied, logits steered, answers scored.

Kinds of cases:

  copy    rows of all page tensors of a cache (every layer's keys and values) copied to other rows, whole or up to the tokens
          that a page holds: a request forked into several, a pool compacted
  rules   a decode step's logits under penalties for repeated tokens, biases and masks of allowed tokens, with the token that
          was chosen last entered into each row's history
  score   the log-probability of a token for every row of logits, with the best alternatives

Logits are float32, as the models give them. A history is the list of a sequence's distinct tokens in the order of their first
appearance, as pairs (token, twice the times it was chosen + 1 if the prompt has it).
"""
import math

import numpy as np
import torch

own = False

VOCAB = 50272
PAD = 384                      # bytes between one page and the next, as the engine leaves them


def listed():
    return [
        # one user, a short conversation with a mild repetition penalty: the launch is what counts
        dict(name="rules 1x50272 penalties", kind="rules", rows=1, vocab=VOCAB, seen=120, biases=0, allowed=-1.0),
        # eight requests that answer in a grammar: few tokens are allowed at each place, almost all of a row is barred
        dict(name="rules 8x50272 grammar", kind="rules", rows=8, vocab=VOCAB, seen=400, biases=0, allowed=0.002),
        # a full batch with everything at once: long histories, lists of biases, half of the tokens allowed
        dict(name="rules 64x50272 all", kind="rules", rows=64, vocab=VOCAB, seen=1500, biases=300, allowed=0.5),
        # rows of an odd vocabulary, which begin at any place in memory
        dict(name="rules 33x32001 all", kind="rules", rows=33, vocab=32001, seen=700, biases=17, allowed=0.93),
        # the chosen token of one user's step, with five alternatives
        dict(name="score 1x50272 top 5", kind="score", rows=1, vocab=VOCAB, top=5),
        # a full batch's tokens with twenty alternatives each
        dict(name="score 64x50272 top 20", kind="score", rows=64, vocab=VOCAB, top=20),
        # a prompt that fills the context, scored token by token
        dict(name="score 2048x50272", kind="score", rows=2048, vocab=VOCAB, top=0),
        # a text of odd length over an odd vocabulary, with a few alternatives
        dict(name="score 777x32001 top 3", kind="score", rows=777, vocab=32001, top=3),
        # a prompt at a small model forked into four answers: the page that is not full, in every layer
        dict(name="copy 350m 1 to 3", kind="copy", layers=24, heads=16, head=64, page=64, pages=24, sources=1, targets=3, tokens=36,
             dtype="bf16"),
        # eight prompts of the headline's model forked into four answers each
        dict(name="copy 6.7b 8 to 24", kind="copy", layers=32, heads=32, head=128, page=64, pages=48, sources=8, targets=24, tokens=45,
             dtype="bf16"),
        # a pool of the same model compacted: whole pages move to the front
        dict(name="copy 6.7b 20 whole", kind="copy", layers=32, heads=32, head=128, page=64, pages=48, sources=20, targets=20, tokens=64,
             dtype="bf16"),
        # the float32 engine, small pages and a head size that is no power of two
        dict(name="copy 2.7b f32 5 to 9", kind="copy", layers=32, heads=32, head=80, page=16, pages=40, sources=5, targets=9, tokens=7,
             dtype="f32"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rules", "score", "copy"])
    if kind == "rules":
        vocab = rng.choice([VOCAB, _log_int(rng, 500, 50000)])
        return dict(kind=kind, rows=_log_int(rng, 1, 64), vocab=vocab, seen=min(vocab // 2, _log_int(rng, 1, 2048)),
                    biases=rng.choice([0, _log_int(rng, 1, 300)]), allowed=rng.choice([-1.0, 0.001, round(rng.random(), 3), 0.98]))
    if kind == "score":
        return dict(kind=kind, rows=_log_int(rng, 1, 2048), vocab=rng.choice([VOCAB, _log_int(rng, 500, 50000)]),
                    top=rng.choice([0, 1, rng.randint(2, 20)]))
    heads, head = rng.choice([(16, 64), (32, 64), (32, 80), (32, 128)])
    page = rng.choice([16, 32, 64])
    sources = _log_int(rng, 1, 12)
    targets = sources * rng.choice([1, 1, 2, 3])
    return dict(kind=kind, layers=rng.choice([24, 32]), heads=heads, head=head, page=page, pages=sources + targets + rng.randint(0, 6),
                sources=sources, targets=targets, tokens=rng.choice([page, rng.randint(1, page)]), dtype=rng.choice(["bf16", "f32"]))


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ops(dtype):
    from transformers_neuronx_amd.kernels import make_ops
    return make_ops("hip", dtype, "cuda:0")


def _logits(g, rows, vocab):
    return torch.randn(rows, vocab, generator=g, device="cuda") * 2.5 - 1.0


def _prepare_copy(case, seed):
    g = _generator(seed)
    rng = np.random.default_rng(seed)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    heads, head, page, pages = case["heads"], case["head"], case["page"], case["pages"]
    count, pad = heads * head * page, PAD // (2 if dtype == torch.bfloat16 else 4)
    tensors = []
    for _ in range(case["layers"]):
        for shape in ((heads, page, head), (heads, head, page)):          # keys, and values turned inside a page
            whole = torch.randn(pages, count + pad, generator=g, device="cuda").to(dtype)
            tensors.append(whole[:, :count].view(pages, *shape))
    order = rng.permutation(pages)
    sources, targets = order[:case["sources"]], order[case["sources"]:case["sources"] + case["targets"]]
    named = np.repeat(sources, -(-case["targets"] // case["sources"]))[:case["targets"]]
    # pages that are not full hold unlike numbers of tokens, those of one source the same
    held = np.full(pages, case["tokens"])
    if case["tokens"] < page:
        held = np.maximum(1, case["tokens"] - rng.integers(0, 1 + case["tokens"] // 4, pages))
    state = dict(kind="copy", tensors=tensors, sources=named.tolist(), targets=targets.tolist(), tokens=held[named].tolist(),
                 whole=case["tokens"] == page, page=page)
    if own:
        state["ops"] = _ops(dtype)
        state["rows"] = state["ops"].row_set(tensors, [2, 3] * case["layers"])
    return state


def _prepare_rules(case, seed):
    g = _generator(seed)
    rng = np.random.default_rng(seed)
    rows, vocab, seen = case["rows"], case["vocab"], case["seen"]
    slots = rows + 3
    used = rng.integers(seen // 2, seen + 1, slots).astype(np.int32)
    if rows > 4:
        used[rng.integers(0, slots)] = 0                              # a request that has nothing yet
    entries = np.zeros((slots, seen + 8, 2), dtype=np.int32)
    for s in range(slots):
        entries[s, :used[s], 0] = rng.choice(vocab, used[s], replace=False)
        prompt = rng.random(used[s]) < 0.7
        entries[s, :used[s], 1] = 2 * np.where(prompt, rng.integers(0, 3, used[s]), rng.integers(1, 5, used[s])) + prompt
    # the token chosen last: for every other request one that it has had, for some none
    last = rng.integers(0, vocab, slots).astype(np.int32)
    again = (rng.random(slots) < 0.5) & (used > 0)
    last[again] = entries[again, rng.integers(0, np.maximum(used, 1))[again], 0]
    last[rng.random(slots) < 0.1] = -1
    row_slots = rng.permutation(slots)[:rows].astype(np.int32)
    repetition = np.round(rng.uniform(0.9, 1.5, rows), 3).astype(np.float32)
    presence = np.round(rng.uniform(-0.5, 1.0, rows), 3).astype(np.float32)
    frequency = np.round(rng.uniform(0.0, 1.0, rows), 3).astype(np.float32)
    if rows > 2:
        row_slots[rows // 2] = -1                                     # a row that keeps no history
    bias_tokens = np.full((rows, max(1, case["biases"])), vocab, dtype=np.int64)       # `vocab`: no bias in this place
    bias_values = np.zeros(bias_tokens.shape, dtype=np.float32)
    for r in range(rows):
        n = int(rng.integers((case["biases"] + 1) // 2, case["biases"] + 1))
        bias_tokens[r, :n] = rng.choice(vocab, n, replace=False)
        bias_values[r, :n] = np.round(rng.normal(0, 4, n), 3)
        if n > 3:
            bias_values[r, 0] = -np.inf                               # a token that must not come
    masks, mask_rows = None, np.full(rows, -1, dtype=np.int32)
    if case["allowed"] >= 0:
        kinds = max(1, rows // 2)                                     # requests in the same place of a grammar share its mask
        words = -(-vocab // 32)
        bits = torch.rand(kinds, words, 32, generator=g, device="cuda") < case["allowed"]
        masks = (bits.long() << torch.arange(32, device="cuda")).sum(-1)
        masks = torch.where(masks >= 2 ** 31, masks - 2 ** 32, masks).to(torch.int32).contiguous()
        mask_rows = (np.arange(rows) % kinds).astype(np.int32)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    state = dict(kind="rules", logits=_logits(g, rows, vocab), entries=dev(entries), used=dev(used), last=dev(last), masks=masks)
    if own:
        from transformers_neuronx_amd.kernels.hip import TokenHistory
        state["ops"] = _ops(torch.bfloat16)
        state["history"] = TokenHistory(state["entries"], state["used"])
        biases = [{int(t): float(v) for t, v in zip(bias_tokens[r], bias_values[r]) if t < vocab} for r in range(rows)]
        state["rules"] = state["ops"].logit_rules(
            vocab, slots=row_slots.tolist(), repetition=repetition.tolist(), presence=presence.tolist(), frequency=frequency.tolist(),
            biases=biases, mask_rows=mask_rows.tolist())
    else:
        state.update(slots=dev(row_slots).long(), repetition=dev(repetition), presence=dev(presence), frequency=dev(frequency),
                     bias_tokens=dev(bias_tokens), bias_values=dev(bias_values), mask_rows=dev(mask_rows).long())
    return state


def _prepare_score(case, seed):
    g = _generator(seed)
    logits = _logits(g, case["rows"], case["vocab"])
    # as a model that is sure of some of its answers gives them, with tokens that were barred before
    sure = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device="cuda")
    logits[torch.arange(case["rows"], device="cuda"), sure] += 12.0 * torch.rand(case["rows"], generator=g, device="cuda")
    logits[:, 1] = float("-inf")
    other = torch.randint(2, case["vocab"], (case["rows"],), generator=g, device="cuda")
    tokens = torch.where(torch.rand(case["rows"], generator=g, device="cuda") < 0.6, sure, other).to(torch.int32)
    state = dict(kind="score", logits=logits, tokens=tokens, top=case["top"])
    if own:
        state["ops"] = _ops(torch.bfloat16)
    return state


def prepare(case, seed):
    return {"copy": _prepare_copy, "rules": _prepare_rules, "score": _prepare_score}[case["kind"]](case, seed)


# ---------------------------------------------------------------- the plain forms

def _plain_copy_one(t, axis, sources, targets, filled):
    if filled is None:
        t[targets] = t[sources]
    else:
        shape = [1] * t.dim()
        shape[0], shape[axis] = filled.shape
        t[targets] = torch.where(filled.view(shape), t[sources], t[targets])


def _plain_copy(s):
    dev = s["tensors"][0].device
    sources, targets = torch.tensor(s["sources"], device=dev), torch.tensor(s["targets"], device=dev)
    filled = None
    if not s["whole"]:
        filled = torch.arange(s["page"], device=dev) < torch.tensor(s["tokens"], device=dev)[:, None]
    [_plain_copy_one(t, 2 + i % 2, sources, targets, filled) for i, t in enumerate(s["tensors"])]


def _plain_rules(s):
    logits, entries, used = s["logits"], s["entries"], s["used"]
    rows, vocab = logits.shape
    has = s["slots"] >= 0
    slots = s["slots"].clamp(min=0)
    mine, n = entries[slots], torch.where(has, used[slots], 0)
    token = torch.where(has, s["last"][slots], -1)
    place = torch.arange(entries.shape[1], device=logits.device)
    # the token chosen last, into the history
    hit = (place < n[:, None]) & (mine[..., 0] == token[:, None]) & (token >= 0)[:, None]
    new = ((token >= 0) & ~hit.any(1))[:, None] & (place == n[:, None])
    mine[..., 0] = torch.where(new, token[:, None], mine[..., 0])
    mine[..., 1] = torch.where(new, 2, mine[..., 1] + 2 * hit)
    n = n + new.any(1)
    own_slots = torch.where(has, slots, entries.shape[0])              # rows without a history write a row that is cut off
    entries.copy_(torch.cat([entries, entries[:1]]).index_copy(0, own_slots, mine)[:-1])
    used.copy_(torch.cat([used, used[:1]]).index_copy(0, own_slots, n.to(used.dtype))[:-1])
    # penalties, biases, the mask; column `vocab` takes what stands for nothing
    wide = torch.cat([logits, logits.new_zeros(rows, 1)], 1)
    at = torch.where(place < n[:, None], mine[..., 0], vocab).long()
    x = wide.gather(1, at)
    times = (mine[..., 1] >> 1).float()
    rho = s["repetition"][:, None]
    y = torch.where(x > 0, x / rho, x * rho)
    y = y - (s["frequency"][:, None] * times + torch.where(times > 0, s["presence"][:, None], 0.0))
    wide.scatter_(1, at, torch.where(place < n[:, None], y, 0.0))
    wide.scatter_add_(1, s["bias_tokens"], s["bias_values"])
    out = wide[:, :vocab]
    if s["masks"] is not None:
        bits = (s["masks"][s["mask_rows"].clamp(min=0)].unsqueeze(-1) >> torch.arange(32, device=logits.device, dtype=torch.int32)) & 1
        allowed = (bits.view(rows, -1)[:, :vocab] == 1) | (s["mask_rows"] < 0)[:, None]
        out = torch.where(allowed, out, float("-inf"))
    logits.copy_(out)


def _plain_score(s):
    x = torch.where(torch.isnan(s["logits"]), float("-inf"), s["logits"])
    m = x.max(dim=1, keepdim=True).values
    lp = x - m - torch.log(torch.exp(x - m).sum(1, keepdim=True))
    out = {"log_prob": lp.gather(1, s["tokens"].long()[:, None])[:, 0]}
    if s["top"]:
        # by the logits themselves: two of them may have one log-probability when it is rounded
        ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
        out["top_log_probs"], out["top_tokens"] = lp.gather(1, ids), ids.to(torch.int32)
    return out


def run(state):
    kind = state["kind"]
    if kind == "copy":
        if own:
            state["ops"].copy_rows(state["rows"], state["sources"], state["targets"], state["tokens"])
        else:
            _plain_copy(state)
        return state["tensors"]
    if kind == "rules":
        if own:
            state["ops"].adjust_logits(state["logits"], state["rules"], state["history"], state["last"], state["masks"])
        else:
            _plain_rules(state)
        return {"logits": state["logits"], "entries": state["entries"], "used": state["used"]}
    if own:
        log_prob, top_tokens, top_log_probs = state["ops"].log_probs(state["logits"], state["tokens"], state["top"])
        out = {"log_prob": log_prob}
        if state["top"]:
            out.update(top_log_probs=top_log_probs, top_tokens=top_tokens)
        return out
    return _plain_score(state)


def work(case):
    if case["kind"] == "copy":
        item = 2 if case["dtype"] == "bf16" else 4
        tokens = case["tokens"] if case["tokens"] == case["page"] else case["tokens"] * 0.875
        return {"bytes": (case["sources"] + case["targets"]) * tokens * 2 * case["layers"] * case["heads"] * case["head"] * item, "flops": 0}
    rows, vocab = case["rows"], case["vocab"]
    if case["kind"] == "score":
        return {"bytes": rows * (4 * vocab + 8 + 8 * case["top"]), "flops": 4.0 * rows * vocab}
    seen, biases = 0.75 * case["seen"] + 1, 0.75 * case["biases"]
    barred = 0.0 if case["allowed"] < 0 else 1.0 - case["allowed"]
    mask = 0.0 if case["allowed"] < 0 else max(1, rows // 2) * vocab / 8
    return {"bytes": mask + rows * (32 + seen * 8 + (1 - barred) * (seen + biases) * 8 + biases * 8 + barred * vocab * 4),
            "flops": rows * (5.0 * seen + biases)}


# ---------------------------------------------------------------- in 64 bits

def _exact_rules(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    h = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor)}
    logits, entries, used = h["logits"].astype(np.float64), h["entries"].copy(), h["used"].copy()
    rows, vocab = logits.shape
    for r in range(rows):
        slot = int(h["slots"][r])
        if slot >= 0:
            token, n = int(h["last"][slot]), int(used[slot])
            if token >= 0:
                found = np.nonzero(entries[slot, :n, 0] == token)[0]
                if len(found):
                    entries[slot, found[0], 1] += 2
                else:
                    entries[slot, n] = (token, 2)
                    used[slot] = n = n + 1
            ids, times = entries[slot, :n, 0], entries[slot, :n, 1] // 2
            x, rho = logits[r, ids], float(h["repetition"][r])
            x = np.where(x > 0, x / rho, x * rho)
            logits[r, ids] = x - float(h["frequency"][r]) * times - float(h["presence"][r]) * (times > 0)
        real = h["bias_tokens"][r] < vocab
        np.add.at(logits[r], h["bias_tokens"][r][real], h["bias_values"][r][real].astype(np.float64))
        if "masks" in h and h["mask_rows"][r] >= 0:
            words = h["masks"][h["mask_rows"][r]].astype("<i4")
            allowed = np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab].astype(bool)
            logits[r, ~allowed] = -np.inf
    return {"logits": logits, "entries": entries, "used": used}


def _exact_copy(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    got = []
    for i, t in enumerate(s["tensors"]):
        for a, b, n in zip(s["sources"], s["targets"], s["tokens"]):
            t[b].narrow(1 + i % 2, 0, n).copy_(t[a].narrow(1 + i % 2, 0, n))
        got.append(t.double())
    return got


def exact(case, seed):
    if case["kind"] == "copy":
        return _exact_copy(case, seed)
    if case["kind"] == "rules":
        return _exact_rules(case, seed)
    s = _prepare_score(dict(case), seed)
    out, top = [], []
    for part in torch.split(torch.arange(case["rows"], device="cuda"), 256):
        x = s["logits"][part].double()
        lse = torch.logsumexp(x, dim=1)
        out.append(x[torch.arange(len(part), device="cuda"), s["tokens"][part].long()] - lse)
        if case["top"]:
            top.append(torch.topk(x, case["top"], dim=1).values - lse[:, None])
    got = {"log_prob": torch.cat(out)}
    if case["top"]:
        got.update(top_log_probs=torch.cat(top), top_tokens=None)
    return got
