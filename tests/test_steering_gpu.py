"""Copied rows, steered logits and log-probabilities on the GPU, against copies and loops in 64 bits."""
import numpy as np
import pytest
import torch

from steering_cases import adjusted, history_tensors, log_probs_in_64, random_rules

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from transformers_neuronx_amd.kernels import make_ops
    return make_ops("hip", torch.float32, "cuda:0")


# ---------------------------------------------------------------- rows

def _pages(shapes, dtype, pad, seed, rows=13):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for shape in shapes:
        count = int(np.prod(shape))
        whole = torch.empty(rows, count + pad, device="cuda", dtype=dtype)
        whole.copy_(torch.randn(whole.shape, generator=g, device="cuda") * 8)
        out.append(whole[:, :count].view(rows, *shape))
    return out


def _copied(tensors, axes, sources, targets, tokens):
    out = [t.clone() for t in tensors]
    for i, (s, d) in enumerate(zip(sources, targets)):
        for t, axis in zip(out, axes):
            n = t.shape[axis] if axis is not None and tokens is None else None if axis is None else tokens[i]
            if axis is None:
                t[d].copy_(t[s])
            else:
                t[d].narrow(axis - 1, 0, n).copy_(t[s].narrow(axis - 1, 0, n))
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
@pytest.mark.parametrize("heads, page, size, pad", [(1, 16, 2, 0), (2, 16, 8, 16), (3, 64, 80, 192), (5, 48, 33, 8), (1, 16, 1, 1), (4, 32, 128, 3)])
def test_copied_rows(ops, dtype, heads, page, size, pad):
    tensors = _pages([(heads, page, size), (heads, size, page), (7,), (heads, page)], dtype, pad, seed=page + size)
    axes = [2, 3, None, 2]
    rows = ops.row_set(tensors, axes)
    for sources, targets, tokens in (([3], [0], [page]), ([5, 5, 5, 1], [12, 0, 2, 4], [1, 1, 1, page - 1]),
                                     ([0, 1, 1, 2], [8, 9, 10, 11], [0, 3, 5, 7]), ([9, 8, 7], [6, 1, 0], None)):
        want = _copied(tensors, axes, sources, targets, tokens)
        ops.copy_rows(rows, sources, targets, tokens)
        assert all(torch.equal(a, b) for a, b in zip(tensors, want)), (sources, targets, tokens)


def test_rows_leave_what_lies_between_them(ops):
    whole = torch.arange(8 * 40, device="cuda", dtype=torch.float32).view(8, 40)
    before = whole.clone()
    ops.copy_rows(ops.row_set([whole[:, 4:37].view(8, 3, 11)], [1]), [0, 6], [3, 7], [2, 3])
    before[3, 4:26], before[7, 4:37] = before[0, 4:26], before[6, 4:37]
    assert torch.equal(whole, before)


def test_rows_of_many_sources_and_targets(ops):
    t = torch.randn(2000, 24, device="cuda")
    order = np.random.default_rng(1).permutation(2000)
    sources, targets = np.repeat(order[:150], 10), order[150:1650]
    want = t.clone()
    want[torch.from_numpy(targets).cuda()] = t[torch.from_numpy(sources).cuda()]
    ops.copy_rows(ops.row_set([t]), sources, targets)
    assert torch.equal(t, want)


def test_rows_beyond_four_gigabytes(ops):
    """Row 5 of a tensor of rows 1 GB apart begins beyond 32 bits of bytes."""
    whole = torch.zeros(6, 1 << 28, device="cuda", dtype=torch.float32)
    t = whole[:, :1000]
    t[5] = torch.arange(1000, device="cuda")
    ops.copy_rows(ops.row_set([t]), [5], [4])
    assert torch.equal(t[4], t[5]) and not t[:4].any()


def test_rows_to_tensors_of_another_size(ops):
    a, b = _pages([(2, 16, 24)], torch.bfloat16, 16, 3, rows=5)[0], _pages([(2, 16, 24)], torch.bfloat16, 48, 4, rows=11)[0]
    want = b.clone()
    want[10], want[0, :, :7] = a[4], a[1, :, :7]
    ops.copy_rows(ops.row_set([a], [2], targets=[b]), [4, 1], [10, 0], [16, 7])
    assert torch.equal(b, want)


# ---------------------------------------------------------------- adjusted logits

def _adjust(ops, case, logits=None):
    from transformers_neuronx_amd.kernels.steering import TokenHistory
    e, u = history_tensors(case, "cuda")
    logits = torch.from_numpy(case["logits"]).cuda() if logits is None else logits
    rules = ops.logit_rules(case["vocab"], **case["rules"])
    last, masks = torch.from_numpy(case["last"]).cuda(), torch.from_numpy(case["masks"]).cuda()
    return logits, rules, TokenHistory(e, u), last, masks


def _check_adjusted(case, logits, history):
    want, entries, used = adjusted(case)
    assert np.array_equal(history.entries.cpu().numpy(), entries) and np.array_equal(history.used.cpu().numpy(), used)
    got = logits.cpu().numpy()
    assert np.array_equal(np.isneginf(got), np.isneginf(want)) and np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isposinf(got), np.isposinf(want))
    fine = np.isfinite(want)
    # a quotient or product, a product and a sum, a difference, a sum: five roundings of half a step of what is added
    assert (np.abs(got[fine] - want[fine]) <= 5 * 2.0 ** -24 * case["scale"][fine]).all()


@pytest.mark.parametrize("rows, vocab, seen, biases, allowed", [
    (1, 1, 1, 1, -1.0), (1, 1, 1, 1, 0.0), (2, 7, 7, 7, 0.5), (3, 31, 31, 10, 0.0), (4, 32, 5, 0, 1.0), (4, 33, 33, 33, 0.9),
    (5, 1000, 0, 0, -1.0), (5, 1003, 400, 30, 0.001), (9, 4097, 3000, 700, 0.5), (3, 32001, 2500, 300, 0.98), (2, 50272, 1500, 300, 0.002),
    (64, 513, 100, 10, 0.5)])
def test_adjusted_logits(ops, rows, vocab, seen, biases, allowed):
    case = random_rules(rows, vocab, seen, biases, allowed, seed=rows * 7 + vocab)
    logits, rules, history, last, masks = _adjust(ops, case)
    out = ops.adjust_logits(logits, rules, history, last, masks)
    assert out is logits
    _check_adjusted(case, logits, history)


def test_rows_that_begin_anywhere(ops):
    """Logits that are a part of a larger tensor, beginning 4 bytes behind a boundary of 16; what lies around them stays."""
    case = random_rules(6, 1001, 300, 40, 0.5, seed=3)
    whole = torch.full((6 * 1001 + 9,), 7.0, device="cuda")
    part = whole[1:1 + 6 * 1001].view(6, 1001)
    part.copy_(torch.from_numpy(case["logits"]))
    logits, rules, history, last, masks = _adjust(ops, case, part)
    ops.adjust_logits(logits, rules, history, last, masks)
    _check_adjusted(case, logits, history)
    assert whole[0] == 7 and (whole[1 + 6 * 1001:] == 7).all()


def test_odd_values_under_rules(ops):
    """Masked places become -inf whatever they were; a bias of -inf bars a token at +inf too; NaN elsewhere stays one."""
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    logits = torch.tensor([[nan, inf, -inf, low, 1.0, inf, nan, -2.0]], device="cuda")
    masks = torch.tensor([[0b11111000]], dtype=torch.int32, device="cuda")
    ops.adjust_logits(logits, ops.logit_rules(8, biases=[{5: -inf, 4: 2.0, 7: -1.0}], mask_rows=[0]), masks=masks)
    assert logits[0, :3].tolist() == [-inf] * 3 and logits[0, 3] == low and logits[0, 4] == 3 and logits[0, 5] == -inf
    assert torch.isnan(logits[0, 6]) and logits[0, 7] == -3


def test_a_full_history_and_tokens_of_no_vocabulary(ops):
    """A history without room takes no further token; entries and tokens outside the vocabulary touch nothing."""
    from transformers_neuronx_amd.kernels.steering import TokenHistory
    entries = torch.tensor([[[0, 2], [1, 2]], [[50, 2], [-3, 2]]], dtype=torch.int32, device="cuda")
    used = torch.tensor([2, 2], dtype=torch.int32, device="cuda")
    logits = torch.ones(2, 4, device="cuda")
    rules = ops.logit_rules(4, slots=[0, 1], presence=[0.5, 0.5])
    ops.adjust_logits(logits, rules, TokenHistory(entries.clone(), used), torch.tensor([3, 99], dtype=torch.int32, device="cuda"))
    assert logits.tolist() == [[0.5, 0.5, 1, 1], [1, 1, 1, 1]] and used.tolist() == [2, 2]


def test_histories_over_steps_and_replays(ops):
    """A step recorded and replayed enters each step's token and gives what the eager steps give."""
    vocab, rows = 1500, 5
    g = torch.Generator(device="cuda").manual_seed(2)
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (1, 40, 300, 0, 7)]
    steps = [(torch.randn(rows, vocab, generator=g, device="cuda"), torch.randint(0, 60, (rows,), generator=g, device="cuda").to(torch.int32))
             for _ in range(6)]
    slots = [4, 0, 3, 1, 2]
    rules = ops.logit_rules(vocab, slots=slots, repetition=[1.3] * rows, presence=[0.4] * rows, frequency=[0.2] * rows)

    def start():
        h, last = ops.token_history(rows, vocab), torch.full((rows,), 9, dtype=torch.int32, device="cuda")
        ops.start_history(h, slots, prompts, last=last)
        assert last.tolist() == [-1] * rows
        return h, last
    eager, (h, last) = [], start()
    for x, chosen in steps:
        eager.append(ops.adjust_logits(x.clone(), rules, h, last))
        last.copy_(chosen)
    want = h.entries.clone(), h.used.clone()
    h, last = start()
    static = steps[0][0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adjust_logits(static, rules, h, last)
    for (x, chosen), y in zip(steps, eager):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(static, y)
        last.copy_(chosen)
    assert torch.equal(h.entries, want[0]) and torch.equal(h.used, want[1])
    # and what the histories hold is what a list of the same tokens gives
    from transformers_neuronx_amd.kernels.steering import TokenHistory
    for i, s in enumerate(slots):
        chosen = [int(c[s]) for _, c in steps[:-1]]
        entries = TokenHistory.distinct(prompts[i], chosen)
        assert h.used[s] == len(entries) and np.array_equal(h.entries[s, :len(entries)].cpu().numpy(), entries)


# ---------------------------------------------------------------- log-probabilities

def _check_log_probs(logits, tokens, top, got):
    want, want_ids, want_best = log_probs_in_64(logits.cpu().numpy(), tokens.cpu().numpy(), top)
    # A logit less the largest is rounded once (2^-24 of it), the logarithm of a sum to a few 2^-24 of itself and of the sum's own
    # error: the sum of n terms in 32 bits is off by at most log2(n) + n / 256 roundings where threads add up their own terms first.
    vocab = logits.shape[1]
    steps = 8 + np.log2(vocab) + vocab / 256
    for a, b in ((got[0], want), (got[2], want_best)) if top else ((got[0], want),):
        a = a.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isfinite(a), np.isfinite(b)) and np.array_equal(np.isneginf(a), np.isneginf(b))
        fine = np.isfinite(b)
        assert (np.abs(a[fine] - b[fine]) <= steps * 2.0 ** -24 * (1 + np.abs(b[fine]))).all()
    if top:
        assert np.array_equal(got[1].cpu().numpy(), want_ids)
    else:
        assert got[1] is None and got[2] is None


@pytest.mark.parametrize("rows, vocab, top", [
    (1, 1, 1), (1, 2, 2), (3, 31, 31), (2, 32, 32), (5, 63, 1), (4, 257, 20), (7, 1000, 0), (3, 1023, 5), (2, 1025, 32), (9, 4096, 3),
    (1, 16384, 20), (2, 32001, 20), (1, 50272, 32), (33, 50272, 5), (300, 513, 2), (2, 70001, 9), (1, 200003, 32)])
def test_log_probs(ops, rows, vocab, top):
    g = torch.Generator(device="cuda").manual_seed(vocab + top)
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * 3
    logits[:, vocab // 2] += 9
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    _check_log_probs(logits, tokens, top, ops.log_probs(logits, tokens, top))


@pytest.mark.parametrize("vocab", [5, 300, 5000, 50272])
@pytest.mark.parametrize("how", ["equal", "few values", "rising", "falling", "barred", "blocks", "crowd"])
def test_log_probs_of_ties_and_orders(ops, how, vocab):
    """Rows whose largest logits are many, alike, or all in one place."""
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    row = {"equal": torch.zeros_like(i), "few values": (i * 7) % 3, "rising": i / vocab * 9, "falling": -i / vocab * 9,
           "barred": torch.where(i % 97 == 3, i / vocab, torch.tensor(float("-inf"), device="cuda")),
           "blocks": torch.where((i % 1024) < 4, 5 + i / vocab, -i / vocab),
           "crowd": torch.where(i // 16 % 256 < 8, 5 + i * 7919 % 1000 / 1000, -i / vocab)}[how]
    logits = torch.stack([row, row.roll(1), -row])
    tokens = torch.tensor([0, vocab // 2, vocab - 1], dtype=torch.int32, device="cuda")
    top = min(20, vocab)
    few = ops.log_probs(logits, tokens, top)
    _check_log_probs(logits, tokens, top, few)
    # many rows are worked on by smaller blocks
    many = ops.log_probs(logits.repeat(200, 1), tokens.repeat(200), top)
    for k in (0, 199):
        _check_log_probs(logits, tokens, top, [t[3 * k:3 * k + 3] for t in many])


@pytest.mark.parametrize("vocab", [3, 40, 3000])
def test_log_probs_of_rows_with_infinities(ops, vocab):
    inf, nan = float("inf"), float("nan")
    logits = torch.randn(7, vocab, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    logits[0] = -inf
    logits[1, [0, vocab - 1]] = inf
    logits[2, 0], logits[2, vocab - 1] = nan, -inf
    logits[3] = nan
    logits[4] = inf
    logits[5, 1:] = -inf
    logits[6, :2] = torch.finfo(torch.float32).min
    tokens = torch.tensor([0, vocab - 1, 0, 1, 2, vocab, -1], dtype=torch.int32, device="cuda")
    top = min(5, vocab)
    _check_log_probs(logits, tokens, top, ops.log_probs(logits, tokens, top))


@pytest.mark.parametrize("vocab", [60, 20001])
def test_log_probs_of_values_far_out(ops, vocab):
    """Rows whose values, or some of them, lie where powers overflow, and sums of very many alike."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(10, vocab, generator=g, device="cuda")
    low = torch.finfo(torch.float32).min
    x[0] = low
    x[1, ::2] = low
    x[2, 1:] = low
    x[3] = x[3].abs() * 1e37
    x[4] = -x[4].abs() * 3e38
    x[5] = -1e31 + x[5] * 1e25
    x[6] = 1000 + x[6]
    x[7] = -3e4 + x[7] * 300
    x[8, 5] = 3e38
    x[9] = x[9] * 1e-30
    tokens = torch.randint(0, vocab, (10,), generator=g, device="cuda").to(torch.int32)
    got = ops.log_probs(x, tokens, 3)
    want, ids, best = log_probs_in_64(x.cpu().numpy(), tokens.cpu().numpy(), 3)
    steps = 8 + np.log2(vocab) + vocab / 256
    for a, b in ((got[0], want), (got[2], best)):
        a = a.cpu().numpy().astype(np.float64)
        with np.errstate(over="ignore"):
            b = b.astype(np.float32).astype(np.float64)         # a difference of two lowest values overflows
        fine = np.isfinite(b)
        assert np.array_equal(fine, np.isfinite(a))
        # beside the sum's own error the difference of a logit and the largest is rounded once, and both count by their size
        assert (np.abs(a[fine] - b[fine]) <= steps * 2.0 ** -24 * (1 + np.abs(b[fine]))).all()
    assert np.array_equal(got[1].cpu().numpy(), ids)


def test_log_probs_beyond_two_to_the_31_elements(ops):
    rows, vocab = 43000, 50001
    logits = torch.empty(rows, vocab, device="cuda")
    logits[-3:].normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    logits[:-3].fill_(1.0)
    tokens = torch.arange(rows, device="cuda", dtype=torch.int32) % vocab
    got = ops.log_probs(logits, tokens, 2)
    _check_log_probs(logits[-3:], tokens[-3:], 2, [t[-3:] for t in got])
    assert torch.allclose(got[0][:-3], torch.full((1,), -np.log(vocab), device="cuda").float(), atol=1e-4)
    rules = ops.logit_rules(vocab, rows=rows, biases=[None] * (rows - 1) + [{vocab - 1: 5.0, 0: float("-inf")}])
    before = logits[-1].clone()
    ops.adjust_logits(logits, rules)
    before[vocab - 1] += 5.0
    before[0] = float("-inf")
    assert torch.equal(logits[-1], before) and (logits[-4] == 1).all()


def test_log_probs_of_a_part_and_in_a_graph(ops):
    g = torch.Generator(device="cuda").manual_seed(4)
    whole = torch.randn(4 * 999 + 3, generator=g, device="cuda")
    logits = whole[3:].view(4, 999)
    tokens = torch.randint(0, 999, (4,), generator=g, device="cuda").to(torch.int32)
    want = ops.log_probs(logits, tokens, 7)
    _check_log_probs(logits, tokens, 7, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.log_probs(logits, tokens, 7)
    for k in range(3):
        logits.copy_(torch.randn(4, 999, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.log_probs(logits, tokens, 7)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_on_another_stream(ops):
    """Everything is launched on the current stream."""
    case = random_rules(4, 3001, 500, 30, 0.5, seed=11)
    side = torch.cuda.Stream()
    t = torch.randn(6, 5, 64, device="cuda")
    want = t.clone()
    want[3] = want[1]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        logits, rules, history, last, masks = _adjust(ops, case)
        ops.adjust_logits(logits, rules, history, last, masks)
        got = ops.log_probs(logits, last[:4].clamp(min=0), 3)
        ops.copy_rows(ops.row_set([t]), [1], [3])
    side.synchronize()
    _check_adjusted(case, logits, history)
    _check_log_probs(logits, last[:4].clamp(min=0), 3, got)
    assert torch.equal(t, want)


def test_rules_and_rows_made_on_one_stream_and_used_on_another(ops):
    """What was sent from the host may still be on its way where another stream works by it."""
    case = random_rules(4, 3001, 500, 30, 0.5, seed=12)
    logits, _, history, last, masks = _adjust(ops, case)
    t = torch.randn(6, 5, 64, device="cuda")
    want = t.clone()
    want[3] = want[1]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    rules, rows = ops.logit_rules(3001, **case["rules"]), ops.row_set([t])
    with torch.cuda.stream(side):
        ops.adjust_logits(logits, rules, history, last, masks)
        ops.copy_rows(rows, [1], [3])
        ops.copy_rows(rows, [], [])
    del rules, rows
    torch.cuda.synchronize()
    _check_adjusted(case, logits, history)
    assert torch.equal(t, want)


def test_refusals(ops):
    from transformers_neuronx_amd.kernels.steering import TokenHistory
    x = torch.zeros(2, 40, device="cuda")
    tokens = torch.zeros(2, dtype=torch.int32, device="cuda")
    history = ops.token_history(2, 8)
    last = torch.zeros(2, dtype=torch.int32, device="cuda")
    plain, kept, masked = ops.logit_rules(40, rows=2), ops.logit_rules(40, slots=[0, 2]), ops.logit_rules(40, mask_rows=[1, 0])
    good = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.adjust_logits(x[:, :39], plain), lambda: ops.adjust_logits(x[:1], plain), lambda: ops.adjust_logits(x.cpu(), plain),
                 lambda: ops.adjust_logits(x.t().contiguous().t(), plain), lambda: ops.adjust_logits(x, kept),
                 lambda: ops.adjust_logits(x, kept, history, last), lambda: ops.adjust_logits(x, ops.logit_rules(40, slots=[0, 1]), history, last[:1]),
                 lambda: ops.adjust_logits(x, masked), lambda: ops.adjust_logits(x, masked, masks=good[:1]),
                 lambda: ops.adjust_logits(x, masked, masks=torch.zeros(2, 1, dtype=torch.int32, device="cuda")),
                 lambda: ops.start_history(history, [0], [list(range(9))]), lambda: ops.start_history(history, [0, 0], [[1], [2]]),
                 lambda: ops.start_history(history, [2], [[1]]), lambda: ops.start_history(history, [0], [[-1]]),
                 lambda: ops.start_history(history, [0], [[1]], last=last[:1]), lambda: ops.start_history(history, [0], []),
                 lambda: ops.log_probs(x, tokens[:1]), lambda: ops.log_probs(x, tokens, 33), lambda: ops.log_probs(x, tokens, -1),
                 lambda: ops.log_probs(x[:, :3].contiguous(), tokens, 4), lambda: ops.log_probs(x.cpu(), tokens), lambda: ops.log_probs(x[0], tokens),
                 lambda: ops.row_set([torch.zeros(3, 4)]), lambda: TokenHistory(torch.zeros(2, 8, 2), torch.zeros(2))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.adjust_logits(x.double(), plain), lambda: ops.log_probs(x.bfloat16(), tokens), lambda: ops.log_probs(x, tokens.long())):
        with pytest.raises(TypeError):
            call()
    rows = ops.row_set([torch.zeros(3, 4, device="cuda")])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="recorded"):
            ops.copy_rows(rows, [0], [1])
        with pytest.raises(RuntimeError, match="recorded"):
            ops.logit_rules(40, rows=2)
        x.add_(1)
    assert ops.adjust_logits(x[:0], ops.logit_rules(40, rows=0)).shape == (0, 40)
    assert ops.log_probs(x[:0], tokens[:0], 2)[1].shape == (0, 2)


def test_log_probs_sent_to_the_host(ops):
    """Two on their way at a time, with and without alternatives."""
    g = torch.Generator(device="cuda").manual_seed(6)
    logits = torch.randn(5, 700, generator=g, device="cuda")
    tokens = torch.randint(0, 700, (5,), generator=g, device="cuda").to(torch.int32)
    for tops in ((0, 4), (4, 1), (9, 0)):
        got = [ops.log_probs(logits, tokens, t) for t in tops]
        sent = [ops.send_log_probs(*x) for x in got]
        for x, s in zip(got, sent):
            assert ops.receive_log_probs(s) == tuple(None if t is None else t.tolist() for t in x)
    a = ops.log_probs(logits, tokens, 3)
    with pytest.raises(ValueError):
        ops.send_log_probs(a[0][:4], a[1], a[2])


@pytest.mark.parametrize("vocab, copies", [(60, 1), (20001, 1), (700, 6)])
def test_log_probs_of_maxima_between_ten_millions_and_ten_billions(ops, vocab, copies):
    """Where one unit of the last place of a logit is more than one, and more than what a power of two can put back."""
    g = np.random.default_rng(vocab)
    maxima = np.concatenate([[2000003840, 2007735680, 2.06e9, 2175962880, 3000016896, 3000050432, 5000029696, 5.58e9, 5661881856, 10000146432, 10618571776],
                             10.0 ** g.uniform(7, 13, 50)])
    maxima = np.tile(np.concatenate([maxima, -maxima]).astype(np.float32), copies)          # (and as many rows as smaller blocks take)
    x = g.normal(0, 3, (len(maxima), vocab)).astype(np.float32)
    below = np.nextafter(maxima, np.float32(-np.inf))
    low = maxima < 0
    x[low] = maxima[low, None] * (1 + np.abs(x[low]))
    at, near, tie = g.permuted(np.tile(np.arange(vocab), (len(maxima), 1)), axis=1)[:, :3].T
    rows = np.arange(len(maxima))
    x[rows, near], x[rows, at] = below, maxima
    x[rows[::3], tie[::3]] = maxima[::3]
    tokens = np.where(rows % 2, at, near).astype(np.int32)
    got = ops.log_probs(torch.from_numpy(x).cuda(), torch.from_numpy(tokens).cuda(), 3)
    want, ids, best = log_probs_in_64(x, tokens, 3)
    # a thread adds a 512th of the row term by term, the threads' sums meet in ten additions; the rest are the roundings of the power and
    # its argument (at most 8 and a half where it is not one by one), of the logarithm and of the two differences
    steps = 20 + vocab / 512
    for a, b in ((got[0], want), (got[2], best)):
        a = a.cpu().numpy().astype(np.float64)
        off = ~np.isfinite(a).reshape(len(maxima), -1).all(1)
        assert not off.any(), maxima[off][:20]
        assert (np.abs(a - b) <= steps * 2.0 ** -24 * (1 + np.abs(b))).all()
    assert np.array_equal(got[1].cpu().numpy(), ids)


def test_log_probs_of_a_long_row_are_off_by_a_few_roundings(ops):
    """16 logits of a round are added up by two chains of eight, rounds one by one, threads' sums in at most ten additions."""
    for rows, vocab in ((3, 50272), (600, 50272), (2, 200003), (1, 5000)):
        x = torch.randn(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda") * 2
        tokens = torch.arange(rows, device="cuda", dtype=torch.int32)
        want = x.double()[torch.arange(rows), :rows].diagonal() - torch.logsumexp(x.double(), 1)
        got = ops.log_probs(x, tokens)[0].double()
        # and eight more for the powers, their arguments, the logarithm and the differences
        steps = 8 + -(-vocab // (16 * 512)) + 10 + 8
        assert ((got - want).abs() <= steps * 2.0 ** -24 * (1 + want.abs())).all()


def test_what_a_copy_of_rows_says_that_it_moves(ops):
    """As many places as the rows hold, a source once for all that it becomes."""
    from transformers_neuronx_amd import debug
    k, v, s = _pages([(2, 16, 8), (2, 8, 16), (7,)], torch.bfloat16, 0, 1)
    rows = ops.row_set([k, v, s], [2, 3, None])
    for (sources, targets, tokens), places, whole in (((([3, 3, 5], [0, 1, 2], [5, 5, 9])), 3 * 5 + 2 * 9, 5), (([3, 4], [0, 1], None), 4 * 16, 4)):
        with debug.kernel_timer() as t:
            ops.copy_rows(rows, sources, targets, tokens)
        (calls, _, moved, _), = t.work_table().values()
        assert calls == 1 and moved == places * 2 * (2 * 8) * 2 + whole * 7 * 2


@pytest.mark.parametrize("vocab", [7, 500, 20004])
def test_the_largest_alternative_is_the_token_of_a_greedy_choice(ops, vocab):
    """One order for both: by logit, ties to the lower id, zeros of both signs alike, NaN as -inf."""
    inf, nan = float("inf"), float("nan")
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.full((8, vocab), -1.0, device="cuda")
    x[0, [2, 4]] = torch.tensor([-0.0, 0.0], device="cuda")
    x[1, [2, 4]] = torch.tensor([0.0, -0.0], device="cuda")
    x[2, [0, 5]] = torch.tensor([nan, 3.0], device="cuda")
    x[3, [1, 6]] = inf
    x[4] = nan
    x[5] = -inf
    x[6, 1:] = nan
    x[7] = torch.randint(0, 3, (vocab,), generator=g, device="cuda").float()
    ids = ops.log_probs(x, torch.zeros(8, dtype=torch.int32, device="cuda"), min(5, vocab))[1]
    want = torch.sort(torch.where(torch.isnan(x), -inf, x), dim=1, descending=True, stable=True).indices
    assert torch.equal(ops.argmax(x.clone()).long(), ids[:, 0].long()) and torch.equal(ids.long(), want[:, :ids.shape[1]])


def test_room_on_the_host_is_kept_until_all_has_arrived(ops):
    """What was sent before and is waited for by nobody, when a larger one takes its place; and no recording writes there."""
    small, large = torch.randn(2, 40, device="cuda"), torch.randn(1000, 40, device="cuda")
    few, many = (ops.log_probs(x, torch.zeros(len(x), dtype=torch.int32, device="cuda"), 3) for x in (small, large))
    ops._scores = [None, None]
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    first = ops.send_log_probs(*few)
    ops.send_log_probs(*few)
    third = ops.send_log_probs(*many)
    assert first[-1].query() and third[0] is not first[0]
    assert ops.receive_log_probs(third) == tuple(t.tolist() for t in many)
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="recorded"):
            ops.send_log_probs(*few)
        x.add_(1)
