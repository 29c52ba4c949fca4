"""Copied rows, steered logits and log-probabilities on the host: the plain renditions against loops in 64 bits, and what is refused."""
import math

import numpy as np
import pytest
import torch

from steering_cases import adjusted, history_tensors, log_probs_in_64, random_rules
from transformers_neuronx_amd.kernels import make_ops
from transformers_neuronx_amd.kernels.row_set import RowSet
from transformers_neuronx_amd.kernels.steering import LogitRules, TokenHistory, mask_words, pack_mask

OPS = make_ops("reference", torch.float32, "cpu")


# ---------------------------------------------------------------- rows

def test_rows_are_copied_as_far_as_they_hold_tokens():
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(6, 2, 16, 8, generator=g), torch.randn(6, 2, 8, 16, generator=g)
    state = torch.randn(6, 3, generator=g)
    before = [t.clone() for t in (k, v, state)]
    rows = OPS.row_set([k, v, state], [2, 3, None])
    OPS.copy_rows(rows, [4, 4, 1], [0, 5, 3], [5, 16, 0])
    for s, d, n in ((4, 0, 5), (4, 5, 16), (1, 3, 0)):
        before[0][d, :, :n] = before[0][s, :, :n]
        before[1][d, :, :, :n] = before[1][s, :, :, :n]
        before[2][d] = before[2][s]
    assert all(torch.equal(a, b) for a, b in zip((k, v, state), before))


def test_rows_go_to_tensors_of_another_size():
    a, b = torch.arange(12.0).view(4, 3), torch.zeros(9, 3)
    OPS.copy_rows(OPS.row_set([a], targets=[b]), [3, 0], [0, 8])
    assert torch.equal(b[0], a[3]) and torch.equal(b[8], a[0]) and not b[1:8].any()


def test_how_rows_lie_is_what_the_kernel_is_told():
    whole = torch.zeros(5, 2 * 16 * 8 + 16)
    k = whole[:, :256].view(5, 2, 16, 8)
    rows = RowSet([k, torch.zeros(5, 3, dtype=torch.bfloat16), torch.zeros(5, 7, dtype=torch.uint8)], [2, None, None])
    assert rows.words[0, 2:].tolist() == [272 * 4, 272 * 4, 16 * 8 * 4, 8 * 4, 2, 16]
    assert rows.words[1, 2:].tolist() == [6, 6, 6, 0, 1, 2] and rows.words[2, 7] == 1
    assert rows.row_bytes == 1024 + 6 + 7 and rows.places == 16
    assert rows.units(-1) == 64 and rows.units(3) == 12 and rows.units(0) == 7


@pytest.mark.parametrize("what, sources, targets, tokens", [
    ("outside", [6], [0], None), ("outside", [-1], [0], None), ("outside", [0], [6], None), ("named twice", [0, 1], [2, 2], None),
    ("both source and target", [0, 1], [1, 2], None), ("both source and target", [3], [3], None), ("targets", [0, 1], [2], None),
    ("holds 0 to 16", [0], [1], [17]), ("holds 0 to 16", [0], [1], [-1]), ("numbers of tokens", [0, 1, 2], [3, 4, 5], [1, 2])])
def test_rows_that_are_refused(what, sources, targets, tokens):
    rows = OPS.row_set([torch.zeros(6, 2, 16, 8)], [2])
    with pytest.raises(ValueError, match=what):
        OPS.copy_rows(rows, sources, targets, tokens)


def test_sets_of_rows_that_are_refused():
    t = torch.zeros(6, 4, 8)
    for bad in (dict(tensors=[]), dict(tensors=[t], token_axes=[0]), dict(tensors=[t], token_axes=[3]),
                dict(tensors=[t.transpose(1, 2)]), dict(tensors=[t, torch.zeros(6, 4, 16)], token_axes=[2, 2]),
                dict(tensors=[t], targets=[t.double()]), dict(tensors=[t], targets=[torch.zeros(6, 8, 4)]),
                dict(tensors=[t, t]), dict(tensors=[t[:3]], targets=[t[2:]]), dict(tensors=[t[:, :2], t[:, 2:]]),
                dict(tensors=[t, torch.zeros(6, 3)], token_axes=[1]), dict(tensors=[torch.zeros(0, 3)]), dict(tensors=[torch.zeros(1, 4).expand(3, 4)])):
        with pytest.raises(ValueError):
            RowSet(**bad)
    with pytest.raises(ValueError, match="counts tokens"):
        OPS.copy_rows(OPS.row_set([t]), [0], [1], [2])
    OPS.copy_rows(OPS.row_set([t]), [], [])


# ---------------------------------------------------------------- histories, rules, masks

def test_a_history_is_its_distinct_tokens_in_order():
    e = TokenHistory.distinct([7, 3, 7, 5], [3, 9, 9, 9])
    assert e.tolist() == [[7, 1], [3, 3], [5, 1], [9, 6]]
    assert TokenHistory.distinct([], [4, 4]).tolist() == [[4, 4]] and TokenHistory.distinct([]).shape == (0, 2)
    h = OPS.token_history(3, 8)
    last = torch.tensor([5, 6, 7], dtype=torch.int32)
    OPS.start_history(h, [2, 0], [[1, 2, 1], []], [[2], []], last)
    assert h.used.tolist() == [0, 0, 2] and h.entries[2, :2].tolist() == [[1, 1], [2, 3]] and last.tolist() == [-1, 6, -1]


@pytest.mark.parametrize("rows, vocab, seen, biases, allowed", [
    (1, 40, 0, 0, -1.0), (3, 33, 7, 5, 0.5), (4, 64, 64, 64, 0.0), (5, 1000, 100, 30, 1.0), (2, 1, 1, 1, 0.5), (6, 101, 20, 0, 0.9)])
def test_adjusted_logits(rows, vocab, seen, biases, allowed):
    case = random_rules(rows, vocab, seen, biases, allowed, seed=rows + vocab)
    want, entries, used = adjusted(case)
    logits = torch.from_numpy(case["logits"].astype(np.float32))
    e, u = history_tensors(case, "cpu")
    last, masks = torch.from_numpy(case["last"]), torch.from_numpy(case["masks"])
    OPS.adjust_logits(logits, OPS.logit_rules(vocab, **case["rules"]), TokenHistory(e, u), last, masks)
    assert np.array_equal(e.numpy(), entries) and np.array_equal(u.numpy(), used)
    assert np.array_equal(np.isneginf(logits.numpy()), np.isneginf(want))
    fine = np.isfinite(want)
    # a division or product, a product and a sum in float32, a difference, a sum: five roundings of half a step of what is added
    assert (np.abs(logits.numpy()[fine] - want[fine]) <= 5 * 2.0 ** -24 * case["scale"][fine]).all()


@pytest.mark.parametrize("bad", [
    dict(slots=[0, 0]), dict(repetition=[0.0, 1.0]), dict(repetition=[-1.0, 1.0]), dict(repetition=[float("nan"), 1.0]),
    dict(repetition=[1e-60, 1.0]), dict(presence=[float("inf"), 0.0]), dict(frequency=[0.0, 1e300]), dict(biases=[{0: float("nan")}, None]),
    dict(biases=[{0: float("inf")}, None]), dict(biases=[{10: 1.0}, None]), dict(biases=[{-1: 1.0}, None]), dict(biases=[None]),
    dict(slots=[0]), dict(mask_rows=[0, 1, 2]), dict(mask_rows=[2 ** 31, 0]), dict(slots=[2 ** 31, 0]), dict(biases=[{3: -1e300}, None])])
def test_rules_that_are_refused(bad):
    with pytest.raises(ValueError):
        LogitRules(10, 2, **bad)


def test_masks():
    assert mask_words(33) == 2
    assert pack_mask(33, [0, 31, 32]).tolist() == [1 | -2 ** 31, 1]
    assert pack_mask(33, np.arange(33) == 32).tolist() == [0, 1]
    assert pack_mask(33, {32, 0}).tolist() == [1, 1] and pack_mask(33, range(3)).tolist() == [7, 0] and not pack_mask(33, []).any()
    for bad in ([33], [-1], np.ones(32, dtype=bool), [1.5], ["a"]):
        with pytest.raises(ValueError):
            pack_mask(33, bad)


# ---------------------------------------------------------------- log-probabilities

@pytest.mark.parametrize("rows, vocab, top", [(1, 1, 1), (3, 5, 5), (4, 100, 0), (2, 1000, 20)])
def test_log_probs(rows, vocab, top):
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(rows, vocab, generator=g) * 4
    tokens = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32)
    got, ids, best = OPS.log_probs(logits, tokens, top)
    want, want_ids, want_best = log_probs_in_64(logits.numpy(), tokens.numpy(), top)
    assert np.allclose(got.numpy(), want, rtol=1e-6, atol=1e-6)
    if top:
        assert np.array_equal(ids.numpy(), want_ids) and np.allclose(best.numpy(), want_best, rtol=1e-6, atol=1e-6)
    else:
        assert ids is None and best is None


def test_log_probs_of_rows_with_infinities():
    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[-inf, -inf, -inf], [inf, 1.0, inf], [nan, 2.0, -inf], [1.0, 1.0, nan], [nan, nan, nan]])
    got, ids, best = OPS.log_probs(logits, torch.tensor([0, 2, 1, 7, 1], dtype=torch.int32), 3)
    assert got.tolist() == [-inf, pytest.approx(-math.log(2)), 0.0, -inf, -inf]
    assert ids.tolist() == [[0, 1, 2], [0, 2, 1], [1, 0, 2], [0, 1, 2], [0, 1, 2]]
    assert best[0].tolist() == [-inf] * 3 and best[1].tolist()[2] == -inf and best[3].tolist() == [pytest.approx(-math.log(2))] * 2 + [-inf]


def test_a_full_history_and_tokens_of_no_vocabulary_on_the_host():
    """A history without room takes no further token; entries and tokens outside the vocabulary touch nothing."""
    entries = torch.tensor([[[0, 2], [1, 2]], [[50, 2], [-3, 2]]], dtype=torch.int32)
    history = TokenHistory(entries.clone(), torch.tensor([2, 2], dtype=torch.int32))
    logits = torch.ones(2, 4)
    rules = OPS.logit_rules(4, slots=[0, 1], presence=[0.5, 0.5])
    OPS.adjust_logits(logits, rules, history, torch.tensor([3, 99], dtype=torch.int32))
    assert logits.tolist() == [[0.5, 0.5, 1, 1], [1, 1, 1, 1]] and torch.equal(history.entries, entries) and history.used.tolist() == [2, 2]


@pytest.mark.parametrize("bad", [2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1, -1])
def test_tokens_that_are_no_32_bits_begin_no_history(bad):
    """They would be entered as other tokens."""
    for prompt, output in (([1, bad], []), ([1], [bad])):
        with pytest.raises(ValueError, match="token"):
            TokenHistory.distinct(prompt, output)
    assert TokenHistory.distinct([2 ** 31 - 1], [0]).tolist() == [[2 ** 31 - 1, 1], [0, 2]]
