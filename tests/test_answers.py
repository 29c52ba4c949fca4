"""Several answers to one prompt, steered and scored, through the engine: on the host with the plain renditions of the kernels, and on the
GPU with the kernels. Forked and resized caches are compared with requests that were computed by themselves."""
import dataclasses
import random

import numpy as np
import pytest
import torch

import gubulorn_cases
import sunatar_cases
import tadolix_cases
import zudusun_cases
from transformers_neuronx_amd.cache import CacheManager, OutOfPages, OutOfSlots, PagePool
from transformers_neuronx_amd.config import EngineConfig
from transformers_neuronx_amd.engine import StepEntry
from transformers_neuronx_amd.engine.engine import LLMEngine
from transformers_neuronx_amd.engine.factory import build_runner, runner_from_folder
from transformers_neuronx_amd.kernels import make_ops
from transformers_neuronx_amd.parts.base import CacheNeed
from transformers_neuronx_amd.sampling import Sampler, SamplingParams, Steering
from transformers_neuronx_amd.weights.loader import TensorDict

BOTH = pytest.mark.parametrize("kernels", ["reference", pytest.param("hip", marks=pytest.mark.gpu)])


def device_of(kernels):
    return "cuda:0" if kernels == "hip" else "cpu"


def engine_of(folder, kernels, max_tokens=640, max_num_seqs=8, **kw):
    cfg = EngineConfig(dtype="float32", kernels=kernels, device=device_of(kernels), page_size=16, max_tokens=max_tokens,
                       max_num_seqs=max_num_seqs, **kw)
    return LLMEngine(runner_from_folder(folder, cfg), cfg)


def prompts_of(vocab, lengths, seed):
    rng = random.Random(seed)
    return [[rng.randrange(3, vocab) for _ in range(n)] for n in lengths]


# ---------------------------------------------------------------- pools and tables

def test_shared_pages_are_free_when_the_last_holder_gives_them_back():
    pool = PagePool(4)
    a = pool.allocate(2, "a")
    pool.share(a, "b")
    assert pool.holders_of(a[0]) == ("a", "b") and pool.num_free == 2
    with pytest.raises(ValueError, match="already"):
        pool.share(a[:1], "b")
    with pytest.raises(ValueError, match="nobody"):
        pool.share([p for p in range(4) if p not in a][:1], "c")
    pool.free(a, "a")
    assert pool.num_free == 2 and pool.holder_of(a[0]) == "b"
    with pytest.raises(ValueError, match="held by"):
        pool.free(a, "a")
    with pytest.raises(ValueError, match="twice"):
        pool.free([a[0], a[0]], "b")
    pool.rename(a, "b", "c")
    pool.free(a, "c")
    assert pool.num_free == 4
    pool.check()


def test_where_pages_go_when_a_pool_is_packed():
    pool = PagePool(6)
    held = pool.allocate(6, "a")
    pool.free([p for p in held if p in (0, 3, 4)], "a")
    where = pool.packed(6)
    assert where == {1: 1, 2: 2, 5: 0}
    with pytest.raises(OutOfPages):
        pool.packed(2)
    pool.repack(where, 3)
    assert pool.num_free == 0 and pool.num_pages == 3 and pool.holder_of(0) == "a"
    pool.check()


def manager(kernels="reference", window=40, state=False, num_pages=40, max_seqs=8, dtype=torch.float32):
    needs = {0: CacheNeed("paged", kv_heads=2, head_size=16), 1: CacheNeed("paged", kv_heads=1, head_size=8)}
    if window:
        needs[2] = CacheNeed("paged", kv_heads=1, head_size=16, window=window)
    if state:
        needs[3] = CacheNeed("state", state_shapes=(("m", (3, 5)), ("n", (7,))))
    dev = device_of(kernels)
    return CacheManager(needs, 16, num_pages, max_seqs, dtype, dev, page_pad_bytes=32, ops=make_ops(kernels, dtype, dev))


def fill(m, req, start, values):
    """The keys and values of tokens from `start` on, as numbers that name them."""
    r = m.requests[req]
    for cid, lc in m.caches.items():
        if lc.group is None:
            continue
        for i, v in enumerate(values):
            page = r.tables[lc.group][(start + i) // 16]
            lc.pages["k"][page, :, (start + i) % 16] = v + cid
            lc.pages["v"][page, :, :, (start + i) % 16] = -v - cid


def holds(m, req, values):
    r = m.requests[req]
    assert r.num_tokens == len(values)
    for cid, lc in m.caches.items():
        if lc.group is None:
            continue
        g = m.groups[lc.group]
        first = 0 if g.window is None else max(0, len(values) - g.window + 1)
        for i in range(first, len(values)):
            page = r.tables[lc.group][i // 16]
            assert page >= 0 and (lc.pages["k"][page, :, i % 16] == values[i] + cid).all(), (req, cid, i)
            assert (lc.pages["v"][page, :, :, i % 16] == -values[i] - cid).all(), (req, cid, i)


@BOTH
@pytest.mark.parametrize("state", [False, True])
def test_requests_forked_grown_ended_compacted_and_resized_in_any_order(kernels, state):
    m = manager(kernels, state=state, num_pages=60)
    rng = random.Random(5)
    live, states, named = {}, {}, 0
    for turn in range(120):
        what = rng.choice(["new", "grow", "grow", "fork", "fork", "end", "compact", "resize", "rename"])
        m.check()
        if what == "new" and len(live) < 8:
            name, named = f"r{named}", named + 1
            m.add_request(name)
            live[name], states[name] = [], 0.0
        elif what == "grow" and live:
            name = rng.choice(sorted(live))
            n = rng.choice([1, 1, 5, 16, 23])
            if m.can_grow(name, len(live[name]) + n):
                m.grow(name, len(live[name]) + n)
                values = [rng.randrange(1, 1 << 12) for _ in range(n)]
                fill(m, name, len(live[name]), values)
                m.advance(name, n)
                live[name] = live[name] + values
                states[name] += 1.5
                if state:
                    for t in m.caches[3].state.values():
                        t[m.slot_of(name)] = states[name]
        elif what == "fork" and live:
            name = rng.choice(sorted(live))
            n = len(live[name]) if state else rng.randint(0, len(live[name]))
            child, named = f"r{named}", named + 1
            if not m.can_fork(name, n):
                with pytest.raises(ValueError):
                    m.fork(name, child, n)
            else:
                try:
                    m.fork(name, child, n)
                    live[child], states[child] = live[name][:n], states[name]
                except (OutOfPages, OutOfSlots):
                    assert not m.has(child)
        elif what == "end" and len(live) > 2:
            name = rng.choice(sorted(live))
            m.free_request(name)
            del live[name], states[name]
        elif what == "compact":
            m.compact()
            for g in m.groups.values():
                held = g.pool.num_pages - g.pool.num_free
                assert all(g.pool.holders_of(p) for p in range(held))
            assert m.compact() == 0
        elif what == "resize":
            size = rng.randint(30, 70)
            if all(g.pool.num_pages - g.pool.num_free <= size for g in m.groups.values()):
                m.resize(size)
                assert all(g.pool.num_pages == size and len(m.caches[g.cache_ids[0]].pages["k"]) == size for g in m.groups.values())
            else:
                with pytest.raises(OutOfPages):
                    m.resize(size)
        elif what == "rename" and live:
            name = rng.choice(sorted(live))
            m.rename(name, name + "x")
            live[name + "x"], states[name + "x"] = live.pop(name), states.pop(name)
        for name in live:
            holds(m, name, live[name])
            if state and live[name]:
                assert all((t[m.slot_of(name)] == states[name]).all() for t in m.caches[3].state.values())
    assert named > 20
    m.reset()
    m.check()


def test_forks_that_are_refused():
    m = manager(num_pages=3, window=20, max_seqs=2)
    m.add_request("a")
    m.grow("a", 40)
    m.advance("a", 40)                      # the window's first page is gone: blocks 0 of positions up to 20
    assert m.can_fork("a", 40) and not m.can_fork("a", 30) and not m.can_fork("a", 41) and not m.can_fork("a", -1)
    assert not m.can_fork("b", 0)
    with pytest.raises(ValueError, match="already live"):
        m.fork("a", "a")
    with pytest.raises(OutOfPages):
        m.fork("a", "b")                    # no page for the one that is not full
    assert not m.has("b") and m.slots.num_free == 1
    m.check()
    m.add_request("c")
    m.free_request("a")
    m.grow("c", 16)
    m.advance("c", 16)
    m.add_request("d")
    with pytest.raises(OutOfSlots):
        m.fork("c", "e")
    m.check()
    no_kernels = CacheManager({0: CacheNeed("paged", kv_heads=1, head_size=8)}, 16, 4, 2, torch.float32, "cpu")
    no_kernels.add_request("a")
    no_kernels.grow("a", 3)
    no_kernels.advance("a", 3)
    with pytest.raises(RuntimeError, match="backend"):
        no_kernels.fork("a", "b")
    no_kernels.check()
    with pytest.raises(ValueError):
        m.resize(0)


def test_a_cache_that_finds_no_memory_halfway_stays_whole(monkeypatch):
    for size in (60, 12):
        m = manager(num_pages=20, window=None)
        for name, n in (("a", 20), ("b", 35), ("c", 7)):
            m.add_request(name)
            m.grow(name, n)
            fill(m, name, 0, list(range(1, n + 1)))
            m.advance(name, n)
        m.free_request("a")
        new, made = m._new_pages, []

        def fails_the_second_time(need, num_pages):
            made.append(num_pages)
            if len(made) == 2:
                raise MemoryError
            return new(need, num_pages)
        monkeypatch.setattr(m, "_new_pages", fails_the_second_time)
        with pytest.raises(MemoryError):
            m.resize(size)
        m.check()
        assert m.groups["full"].pool.num_pages == min(size, 20)
        holds(m, "b", list(range(1, 36)))
        holds(m, "c", list(range(1, 8)))
        m.fork("b", "d")
        m.resize(size)
        assert {len(m.caches[c].pages["k"]) for c in (0, 1)} == {size}
        for name in ("b", "d"):
            holds(m, name, list(range(1, 36)))


# ---------------------------------------------------------------- answers that share a prompt

@BOTH
@pytest.mark.parametrize("run_ahead", [True, False])
@pytest.mark.parametrize("seqs, tokens, chunk", [(8, 640, None), (8, 640, 11), (3, 640, None), (8, 256, 9)])
def test_samples_are_what_requests_of_their_own_give(tiny_folders, kernels, run_ahead, seqs, tokens, chunk):
    """Also where slots or pages run out, so that some of them are computed by themselves, put back and admitted again."""
    folder, cfg, _ = tiny_folders["A"]
    prompts = prompts_of(cfg["vocab_size"], [37, 16, 1, 2, 33], 3)
    params = SamplingParams(max_new_tokens=14, temperature=1.3, top_k=40, seed=11, ignore_eos=True)
    alone = engine_of(folder, kernels, run_ahead=run_ahead)
    want = [alone.generate([p], dataclasses.replace(params, seed=11 + i))[0] for p in prompts for i in range(4)]
    engine = engine_of(folder, kernels, tokens, seqs, chunk_size=chunk, run_ahead=run_ahead)
    assert engine.generate(prompts, params, samples=4) == want
    engine.runner.cache.check()
    assert not engine.runner.cache.requests and all(g.pool.num_free == g.pool.num_pages for g in engine.runner.cache.groups.values())


@BOTH
def test_a_prompt_is_computed_once(tiny_folders, kernels):
    folder, cfg, _ = tiny_folders["A"]
    engine = engine_of(folder, kernels)
    names = engine.add_samples(prompts_of(cfg["vocab_size"], [50], 1)[0], SamplingParams(max_new_tokens=4, seed=1), 5, "p")
    assert names == ["p", ("p", 1), ("p", 2), ("p", 3), ("p", 4)]
    seen = []
    step = engine.runner.step
    engine.runner.step = lambda entries, **kw: (seen.append([len(e.tokens) for e in entries]), step(entries, **kw))[1]
    engine.step()
    engine.step()
    cache = engine.runner.cache
    assert seen == [[49], [1] * 5]
    full = [cache.requests[n].tables["full"][:3] for n in names]
    assert all(t == full[0] for t in full) and len({cache.requests[n].tables["full"][3] for n in names}) == 5
    cache.check()
    engine.abort_request("p")
    cache.check()
    engine.run()
    assert [len(engine.requests[n].output) for n in names[1:]] == [4] * 4


CASES = {"sunatar": (sunatar_cases, "a"), "gubulorn": (gubulorn_cases, "a"), "tadolix": (tadolix_cases, "a"), "zudusun": (zudusun_cases, "a")}


@BOTH
@pytest.mark.parametrize("design", list(CASES))
def test_samples_of_designs_that_keep_state(design, kernels):
    module, name = CASES[design]
    cfg = module.config(name)
    w = module.weights(cfg, 4)
    prompt = module.requests(cfg, [41], 2)["r0"]
    params = SamplingParams(max_new_tokens=7, temperature=1.1, seed=5, ignore_eos=True)

    def fresh():
        runner = module.runner(cfg, w, kernels=kernels, device=device_of(kernels), max_tokens=512, max_seqs=5)
        ecfg = EngineConfig(dtype="float32", page_size=16, max_tokens=512, max_num_seqs=5, device=device_of(kernels), kernels=kernels)
        return LLMEngine(runner, ecfg)
    want = [fresh().generate([prompt], dataclasses.replace(params, seed=5 + i))[0] for i in range(4)]
    engine = fresh()
    forks = []
    fork = engine.runner.cache.fork
    engine.runner.cache.fork = lambda *a: (forks.append(a), fork(*a))[1]
    assert engine.generate([prompt], params, samples=4) == want
    assert len(forks) == 3
    engine.runner.cache.check()


@BOTH
def test_a_request_forked_midway(tiny_folders, kernels):
    folder, cfg, _ = tiny_folders["B"]
    prompt = prompts_of(cfg["vocab_size"], [21], 8)[0]
    params = SamplingParams(max_new_tokens=20, temperature=1.2, seed=3, ignore_eos=True, logprobs=1)
    engine = engine_of(folder, kernels)
    engine.add_request(prompt, params, "a")
    for _ in range(6):
        engine.step()
    have = [t for t in engine.requests["a"].output if t >= 0]
    assert 3 <= len(have) < 20
    greedy = dataclasses.replace(params, do_sample=False)
    assert engine.fork_request("a", greedy, "b") == "b"
    again = engine.fork_request("a")
    engine.run()
    a, b, c = (engine.requests[n] for n in ("a", "b", again))
    alone = engine_of(folder, kernels)
    assert a.output == alone.generate([prompt], params)[0]
    assert b.output[:len(have)] == have and b.output[len(have):] == alone.generate(
        [prompt + have], dataclasses.replace(greedy, max_new_tokens=20 - len(have)))[0]
    assert c.output[:len(have)] == have and len(c.output) == 20 and len(c.logprobs) == len(c.top_logprobs) == 20
    with pytest.raises(ValueError, match="tokens already"):
        engine.fork_request("a")
    engine.runner.cache.check()


@BOTH
def test_the_cache_resized_between_steps(tiny_folders, kernels):
    folder, cfg, _ = tiny_folders["A"]
    prompts = prompts_of(cfg["vocab_size"], [30, 45, 5], 6)
    params = SamplingParams(max_new_tokens=24, do_sample=False, ignore_eos=True)
    want = engine_of(folder, kernels).generate(prompts, params)
    engine = engine_of(folder, kernels)
    names = [engine.add_request(p, params) for p in prompts]
    for n, size in enumerate([40, 13, 13, 80, 15, 14]):
        engine.step()
        engine.step()
        engine.resize_cache(size)
        engine.runner.cache.check()
    with pytest.raises(OutOfPages):
        engine.resize_cache(3)
    engine.run()
    assert [engine.requests[n].output for n in names] == want


# ---------------------------------------------------------------- steered and scored

def adjusted_row(row, request, index, vocab):
    """The logits that token `index` of the request was chosen from, in 64 bits."""
    p, x = request.params, row.double().numpy().copy()
    before = request.output[:index]
    for t in set(request.prompt) | set(before):
        times = before.count(t)
        x[t] = x[t] / p.repetition_penalty if x[t] > 0 else x[t] * p.repetition_penalty
        x[t] -= p.frequency_penalty * times + (p.presence_penalty if times else 0.0)
    for t, b in (p.logit_bias or {}).items():
        x[t] = -np.inf if b == -np.inf else x[t] + b
    if p.allowed_tokens is not None:
        allowed = p.allowed_tokens(list(before)) if callable(p.allowed_tokens) else p.allowed_tokens
        keep = np.zeros(vocab, dtype=bool)
        keep[np.asarray(allowed)] = True
        x[~keep] = -np.inf
    return x


def check_steered(engine, vocab, run):
    """Every chosen token is the largest of the steered logits, and what is said of it is their log-probability."""
    rows = []

    def keep(requests, logits):
        rows.extend((q, len(q.output), x.clone()) for q, x in zip(requests, logits.cpu()))
    engine.logits_hook = keep
    run()
    seen = 0
    for q, index, row in rows:
        if index >= len(q.output):
            continue                                  # a step started when the request had ended
        x = adjusted_row(row, q, index, vocab)
        scale = np.abs(x[np.isfinite(x)]).max()
        # two roundings a penalty and bias, of values up to the scale: the largest is met to 1e-6 of it
        assert x[q.output[index]] >= x.max() - 1e-6 * scale, (q.req_id, index)
        if q.params.logprobs is not None:
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            assert abs(q.logprobs[index] - lp[q.output[index]]) <= 1e-6 * (1 + scale)
            top = q.top_logprobs[index]
            assert len(top) == q.params.logprobs and [v for _, v in top] == sorted((v for _, v in top), reverse=True)
            if top:
                assert top[0][0] == q.output[index]
                assert all(abs(v - lp[t]) <= 1e-6 * (1 + scale) or (np.isneginf(v) and np.isneginf(lp[t])) for t, v in top)
        seen += 1
    return seen


@BOTH
@pytest.mark.parametrize("run_ahead", [True, False])
@pytest.mark.parametrize("tokens", [640, 160])
def test_steered_requests_beside_plain_ones(tiny_folders, kernels, run_ahead, tokens):
    """With room for all, and with so little that requests are put back and their histories begun again."""
    folder, cfg, _ = tiny_folders["A"]
    vocab = cfg["vocab_size"]
    rng = random.Random(4)
    engine = engine_of(folder, kernels, tokens, run_ahead=run_ahead)
    base = dict(max_new_tokens=25, do_sample=False, ignore_eos=True)
    sets = [dict(), dict(repetition_penalty=1.6), dict(presence_penalty=0.8, frequency_penalty=0.5, logprobs=3), dict(logprobs=0),
            dict(logit_bias={t: rng.uniform(-2, 2) for t in range(100, 140)}), dict(allowed_tokens=list(range(0, vocab, 3)), logprobs=5),
            dict(repetition_penalty=0.7, frequency_penalty=-0.2, logit_bias={7: float("-inf"), 8: 1.0}, allowed_tokens=np.arange(vocab) % 2 == 0)]
    for i, (s, p) in enumerate(zip(sets, prompts_of(vocab, [20, 31, 3, 17, 40, 1, 26], 9))):
        engine.add_request(p, SamplingParams(**base, **s), i)
    assert check_steered(engine, vocab, engine.run) == 7 * 25
    if tokens == 160:
        assert engine.scheduler.num_preemptions > 0
    engine.runner.cache.check()


@BOTH
def test_a_grammar(tiny_folders, kernels):
    """Tokens that have to rise by at most five each time, and end where none is left."""
    folder, cfg, _ = tiny_folders["A"]
    vocab = cfg["vocab_size"]

    def rising(output):
        last = output[-1] if output else vocab - 41
        return [t for t in range(last + 1, last + 6) if t < vocab]
    engine = engine_of(folder, kernels)
    prompts = prompts_of(vocab, [9, 12], 2)
    engine.add_request(prompts[0], SamplingParams(max_new_tokens=60, do_sample=False, allowed_tokens=rising, logprobs=2), "a")
    engine.add_request(prompts[1], SamplingParams(max_new_tokens=5, do_sample=False, ignore_eos=True), "b")
    ends = {}

    def run():
        while engine.has_work:
            for o in engine.step():
                if o.finished:
                    ends[o.req_id] = o
    assert check_steered(engine, vocab, run) == len(engine.requests["a"].output) + 5
    out = engine.requests["a"].output
    assert all(0 < b - a <= 5 for a, b in zip(out, out[1:])) and out[-1] == vocab - 1
    assert ends["a"].finish_reason == "grammar" and ends["a"].token == vocab - 1 and ends["b"].finish_reason == "length"
    assert ends["a"].logprob == engine.requests["a"].logprobs[-1] and len(ends["a"].top_logprobs) == 2


@BOTH
def test_the_best_of_several(tiny_folders, kernels):
    folder, cfg, _ = tiny_folders["A"]
    prompts = prompts_of(cfg["vocab_size"], [12, 30], 7)
    params = SamplingParams(max_new_tokens=8, temperature=1.5, seed=2, ignore_eos=True)
    engine = engine_of(folder, kernels)
    every = engine.generate_requests(prompts, dataclasses.replace(params, logprobs=0), samples=5)
    best = engine.generate(prompts, params, samples=2, best_of=5)
    want = [q.output for family in every for q in sorted(family, key=lambda q: -q.cumulative_logprob)[:2]]
    assert best == want
    for bad in (dict(samples=0), dict(samples=3, best_of=2)):
        with pytest.raises(ValueError):
            engine.generate(prompts, params, **bad)


def test_params_that_are_refused(tiny_folders):
    nan, inf = float("nan"), float("inf")
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=nan), dict(repetition_penalty=inf),
                dict(repetition_penalty=1e-50), dict(frequency_penalty=nan), dict(presence_penalty=inf), dict(logit_bias={3: nan}),
                dict(logit_bias={3: inf}), dict(logit_bias={3: 1e300}), dict(logprobs=-1), dict(logprobs=33), dict(logprobs=1.5)):
        with pytest.raises(ValueError):
            SamplingParams(**bad)
    folder, cfg, _ = tiny_folders["A"]
    engine = engine_of(folder, "reference")
    vocab = cfg["vocab_size"]
    for bad in (dict(logit_bias={vocab: 1.0}), dict(logit_bias={-1: 1.0}), dict(allowed_tokens=[vocab]), dict(allowed_tokens=[]),
                dict(allowed_tokens=lambda out: []), dict(allowed_tokens=np.ones(vocab - 1, dtype=bool)),
                dict(allowed_tokens=[5], logit_bias={5: -inf}), dict(allowed_tokens=[2], ban_eos=True, eos_token_id=2)):
        with pytest.raises(ValueError):
            engine.add_request([3, 4, 5], SamplingParams(**bad))
    for count, params in ((0, SamplingParams()), (2, SamplingParams(max_new_tokens=0))):
        with pytest.raises(ValueError):
            engine.add_samples([3], params, count)
    assert not engine.has_work and not engine.requests
    calls = []

    def refuses_the_third(output):
        calls.append(output)
        return [5] if len(calls) < 3 else []
    with pytest.raises(ValueError, match="no token"):
        engine.add_samples([3, 4], SamplingParams(allowed_tokens=refuses_the_third), 4, "q")
    assert not engine.has_work and not engine.requests              # all of them or none
    engine.add_request([3], SamplingParams(), ("p", 1))
    with pytest.raises(ValueError, match="already live"):
        engine.add_samples([3], SamplingParams(), 2, "p")
    with pytest.raises(KeyError):
        engine.fork_request("nobody")
    # a sampler that keeps no histories has nothing to penalise by
    ops = make_ops("reference", torch.float32, "cpu")
    with pytest.raises(ValueError, match="slot"):
        Sampler(ops, "cpu").draw(torch.zeros(1, 4), [SamplingParams(repetition_penalty=2.0)], [0], steering=[Steering(0)])


@BOTH
def test_rules_follow_the_batch(kernels):
    """Rows that change places, leave and return, with one sampler: each batch goes by its own rules and masks."""
    dev = device_of(kernels)
    ops = make_ops(kernels, torch.float32, dev)
    last = torch.full((4,), -1, dtype=torch.int32, device=dev)
    sampler = Sampler(ops, dev, slots=4, capacity=50, last=last)
    masks = [np.array([0b1110, 0], dtype=np.int32), np.array([0b0110, 0], dtype=np.int32)]
    greedy = dict(do_sample=False)
    rows = [(SamplingParams(presence_penalty=5.0, **greedy), 0, None), (SamplingParams(**greedy), 1, masks[0]),
            (SamplingParams(logit_bias={3: 9.0}, **greedy), 2, masks[1]), (SamplingParams(logit_bias={4: 2.5}, **greedy), 3, None)]
    logits = torch.zeros(4, 50)
    logits[:, 9], logits[:, 3], logits[:, 2] = 2.0, 1.0, 0.5
    want = {0: [9, 3, 2], 1: [3] * 9, 2: [2] * 9, 3: [4] * 9}
    turns = {i: 0 for i in range(4)}
    for batch in ([0, 1, 2, 3], [3, 1], [0, 2], [2, 0], [1], [1], [2, 1]):
        steering = [Steering(rows[i][1], start=([], []) if turns[i] == 0 else None, mask=rows[i][2]) for i in batch]
        drawn = sampler.draw(logits[batch].to(dev), [rows[i][0] for i in batch], [0] * len(batch), steering=steering)
        for i, t in zip(batch, drawn.tolist()):
            assert t == want[i][turns[i]], (batch, i)
            last[rows[i][1]] = t
            turns[i] += 1


# ---------------------------------------------------------------- the user's model class

def model_of(folder, kernels, batch_size=4, **kw):
    from transformers_neuronx_amd import OPTForSampling
    return OPTForSampling.from_pretrained(folder, batch_size=batch_size, amp="f32", n_positions=64, page_size=16, kernels=kernels,
                                          device=device_of(kernels), **kw).load()


@BOTH
def test_sequences_from_the_entry_point(tiny_folders, kernels):
    folder, cfg, _ = tiny_folders["A"]
    ids = torch.tensor(prompts_of(cfg["vocab_size"], [10, 10], 1))
    model = model_of(folder, kernels, 6)
    one = [model.sample(ids[b:b + 1], 18, top_k=20, seed=7 + 3 * b + i) for b in range(2) for i in range(3)]
    out = model.sample(ids, 18, top_k=20, seed=7, num_return_sequences=3)
    assert torch.equal(out, torch.cat(one))
    best = model.sample(ids, 18, top_k=20, seed=7, best_of=3)
    score = model.log_probs(out)[:, 10:].sum(1)
    # the sums are of the same log-probabilities, but that the token no answer may have is barred in the one and not in the other
    assert best.shape == (2, 18) and all((best[b].unsqueeze(0) == out[3 * b:3 * b + 3]).all(1).any() for b in range(2))
    for b in range(2):
        chosen = (best[b].unsqueeze(0) == out[3 * b:3 * b + 3]).all(1).nonzero()[0, 0]
        assert score[3 * b + chosen] >= score[3 * b:3 * b + 3].max() - 0.05
    greedy = model.sample(ids, 18, top_k=1, repetition_penalty=1e6)
    assert all(len(set(row.tolist()[10:])) == 8 and not set(row.tolist()[10:]) & set(row.tolist()[:10]) for row in greedy)
    assert torch.equal(model.sample(ids, 7, num_return_sequences=2), ids[[0, 0, 1, 1], :7])        # nothing to generate
    assert (model.sample(ids, 14, top_k=5, allowed_tokens=[40, 41])[:, 10:] // 2 == 20).all()
    for bad in (dict(num_return_sequences=0), dict(num_return_sequences=3, best_of=2)):
        with pytest.raises(ValueError):
            model.sample(ids, 18, **bad)


@pytest.mark.gpu
def test_the_command_line(tiny_folders, capsys, tmp_path):
    from transformers_neuronx_amd.opt.demo import main
    folder, cfg, _ = tiny_folders["A"]
    main(["--amp", "f32", "run", folder, "--batch_size", "2", "--n_positions", "32", "--prompt_len", "9", "--max_new_tokens", "6", "--do_sample",
          "--top_k", "30", "--num_return_sequences", "2", "--best_of", "3", "--repetition_penalty", "1.2", "--frequency_penalty", "0.1",
          "--presence_penalty", "0.1", "--dump_logits", str(tmp_path / "d"), "--dump_logits_limit", "-1"])
    out = capsys.readouterr().out
    assert out.count("[") >= 5 and "Dumped the logits of" in out


@BOTH
def test_a_text_scored(tiny_folders, kernels):
    import plain_opt
    folder, cfg, weights = tiny_folders["A"]
    rows = prompts_of(cfg["vocab_size"], [30, 17], 5)
    ids = torch.zeros(2, 30, dtype=torch.long)
    ids[0], ids[1, 13:] = torch.tensor(rows[0]), torch.tensor(rows[1])
    with pytest.raises(ValueError, match="vocabulary"):
        model_of(folder, kernels).log_probs(torch.tensor([[3, cfg["vocab_size"]]]))
    for portion in (2048, 7):
        got = model_of(folder, kernels, max_num_batched_tokens=portion).log_probs(ids, start_ids=[0, 13])
        for b, toks in enumerate(rows):
            lp = torch.log_softmax(plain_opt.forward_logits(weights, cfg, toks).double(), -1)
            want = lp[torch.arange(len(toks) - 1), torch.tensor(toks[1:])]
            first = 30 - len(toks) + 1
            assert (got[b, :first] == 0).all() and torch.allclose(got[b, first:].double(), want, atol=3e-5)


@BOTH
def test_rows_reordered_and_sequences_forked(tiny_folders, kernels):
    folder, cfg, _ = tiny_folders["A"]
    vocab = cfg["vocab_size"]
    ids = torch.tensor(prompts_of(vocab, [19] * 4, 3))
    model = model_of(folder, kernels)
    model.forward(ids)
    texts = ids.tolist()
    nxt = 19
    for beams in ([1, 1, 0, 1], [3, 2, 1, 0], [2, 2, 2, 2], [0, 1, 2, 3]):
        model.reorder_cache(beams)
        texts = [list(texts[b]) for b in beams]
        new = torch.tensor(prompts_of(vocab, [4], nxt)[0]).unsqueeze(1)
        texts = [t + [int(n)] for t, n in zip(texts, new)]
        logits = model.forward(new, cache_ids=[nxt])
        nxt += 1
        model.engine.runner.cache.check()
    want = model_of(folder, kernels).forward(torch.tensor(texts))
    assert torch.allclose(logits, want, atol=2e-5 * float(want.abs().max()))
    for bad in ([0, 1, 2], [0, 1, 2, 4], [0, 1, 2, 3, 4]):
        with pytest.raises(ValueError):
            model.reorder_cache(bad) if len(bad) != 3 else model.engine.runner.reorder([("row", b) for b in range(4)], bad)
    from transformers_neuronx_amd import ContinuousBatchingConfig, NeuronConfig
    model = model_of(folder, kernels, neuron_config=NeuronConfig(continuous_batching=ContinuousBatchingConfig(max_num_seqs=4)))
    model.forward(ids[:1], cache_ids=torch.arange(19).unsqueeze(0), start_ids=[2])
    model.fork_sequence(2, 0)
    a = model.forward(torch.tensor([[5], [6]]), cache_ids=torch.tensor([[19], [19]]), start_ids=[0, 2])
    fresh = model_of(folder, kernels)
    want = fresh.forward(torch.cat([ids[:1].repeat(2, 1), torch.tensor([[5], [6]])], 1))
    assert torch.allclose(a, want, atol=2e-5 * float(want.abs().max()))
    with pytest.raises(ValueError):
        model.fork_sequence(3, 1)
    with pytest.raises(ValueError):
        model.fork_sequence(0, 0)


@BOTH
@pytest.mark.parametrize("run_ahead, prompts_first", [(True, False), (False, False), (True, True)])
@pytest.mark.parametrize("design, seed", [("opt", 0), ("opt", 1), ("opt", 2), ("opt", 3)] + [(d, i) for d in CASES for i in range(2)])
def test_everything_together_in_any_order(tiny_folders, kernels, run_ahead, prompts_first, design, seed):
    """Families of samples, forks midway, requests taken out, a pool that is too small and changes its size, steered and scored requests
    among plain ones: each generates what it would alone."""
    if design == "opt":
        folder, cfg, _ = tiny_folders["A"]
        vocab = cfg["vocab_size"]

        def made(**kw):
            return engine_of(folder, kernels, **kw)
    else:
        module, name = CASES[design]
        cfg = module.config(name)
        vocab, w = cfg.vocab, module.weights(cfg, 4)

        def made(max_tokens=640, max_num_seqs=8, **kw):
            ecfg = EngineConfig(dtype="float32", kernels=kernels, device=device_of(kernels), page_size=16, max_tokens=max_tokens,
                                max_num_seqs=max_num_seqs, **kw)
            return LLMEngine(build_runner(cfg, TensorDict({k: v.clone() for k, v in w.items()}), ecfg), ecfg)
    rng = random.Random(seed)
    engine = made(max_tokens=rng.choice([176, 256, 400]), max_num_seqs=rng.choice([3, 5, 8]), chunk_size=rng.choice([None, 7]),
                  max_num_batched_tokens=rng.choice([24, 2048]), run_ahead=run_ahead, prompts_first=prompts_first)
    cache = engine.runner.cache
    told = {}                     # name -> (prompt, params, tokens it began with)
    reported = {}

    def rules():
        return rng.choice([{}, {}, dict(repetition_penalty=1.4), dict(frequency_penalty=0.3, logprobs=2), dict(logprobs=0),
                           dict(logit_bias={5: 3.0, 9: float("-inf")}), dict(allowed_tokens=sorted(rng.sample(range(vocab), vocab // 3))),
                           dict(presence_penalty=0.5, allowed_tokens=lambda out: range(len(out) % 7, vocab, 7))])
    for turn in range(60):
        what = rng.choice(["add", "step", "step", "step", "fork", "abort", "resize", "compact"])
        if what == "add" and len(told) < 14:
            prompt = [rng.randrange(3, vocab) for _ in range(rng.choice([1, 2, 9, 17, 33, 48]))]
            params = SamplingParams(max_new_tokens=rng.choice([1, 3, 12, 20]), temperature=1.2, top_k=rng.choice([0, 1, 30]), seed=rng.randrange(999),
                                    ignore_eos=True, **rules())
            for i, name in enumerate(engine.add_samples(prompt, params, rng.choice([1, 1, 2, 4]), f"n{turn}")):
                told[name] = prompt, dataclasses.replace(params, seed=params.seed + i), []
        elif what == "fork" and told:
            name = rng.choice([n for n in told])
            if name in engine.requests and len([t for t in engine.requests[name].output if t >= 0]) < told[name][1].max_new_tokens:
                have = [t for t in engine.requests[name].output if t >= 0]
                params = dataclasses.replace(told[name][1], seed=rng.randrange(999))
                told[engine.fork_request(name, params, f"f{turn}")] = told[name][0], params, have
        elif what == "abort" and len(told) > 3 and rng.random() < 0.4:
            name = rng.choice([n for n in told])
            if name in engine.requests:
                engine.abort_request(name)
            del told[name]
            reported.pop(name, None)
        elif what == "resize" and rng.random() < 0.5:
            held = max(g.pool.num_pages - g.pool.num_free for g in cache.groups.values())
            engine.resize_cache(max(held, rng.choice([11, 16, 25])))
        elif what == "compact":
            cache.compact()
        else:
            for o in engine.step():
                reported.setdefault(o.req_id, []).append(o.token)
        cache.check()
    while engine.has_work:
        for o in engine.step():
            reported.setdefault(o.req_id, []).append(o.token)
    cache.check()
    assert not cache.requests and all(g.pool.num_free == g.pool.num_pages for g in cache.groups.values())
    alone = made()
    for name, (prompt, params, begun) in told.items():
        q = engine.requests[name]
        assert q.output == begun + reported[name] and len(q.output) == params.max_new_tokens
        if params.logprobs is not None:
            assert len(q.logprobs) == len(q.top_logprobs) == len(q.output)
        alone.reset()
        alone.add_request(prompt, params, "x")
        if begun:
            # a request that begins with tokens it did not draw itself
            alone.abort_request("x")
            alone._add(prompt, params, "x", output=begun)
        alone.run()
        assert alone.requests["x"].output == q.output, (name, params)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "C"])
@pytest.mark.parametrize("graphs", [True, False])
def test_forked_requests_of_a_bfloat16_engine(tiny_folders_bf16, name, graphs):
    """Forks of one request, fed the same tokens in one batch, give the same bits, wherever pages move in between."""
    folder, cfg, _ = tiny_folders_bf16[name]
    ecfg = EngineConfig(dtype="bfloat16", device="cuda:0", page_size=16, num_pages=60, max_num_seqs=6, use_graphs=graphs)
    runner = runner_from_folder(folder, ecfg)
    assert runner.cache.page_pad_bytes == 384
    prompt = prompts_of(cfg["vocab_size"], [45], 1)[0]
    runner.step([StepEntry("a", prompt, [])])
    for i, child in enumerate("bcd"):
        runner.fork("a", child)
    names, rng = list("abcd"), random.Random(0)
    for turn in range(30):
        token = rng.randrange(3, cfg["vocab_size"])
        logits = runner.step([StepEntry(n, [token], [0]) for n in names])
        assert all(torch.equal(logits[0], row) for row in logits[1:]), turn
        assert torch.isfinite(logits).all()
        if turn % 5 == 1:
            runner.finish(names[1])
            runner.fork(names[3], names[1])
        elif turn % 5 == 2:
            runner.reorder(names, [2, 2, 0, 1])
        elif turn % 5 == 3:
            runner.cache.compact()
        elif turn % 10 == 4:
            runner.resize_cache(30 if turn == 4 else 70)
        runner.cache.check()
    assert len(runner.cache.requests["a"].tables["full"]) == 5


@BOTH
def test_a_search_over_beams(tiny_folders, kernels):
    """As a program does it with the model's own calls: the likeliest continuations of every beam, the best of them all kept, the cache
    reordered. Against the same search over whole sequences without a cache, in 64 bits."""
    import plain_opt
    folder, cfg, weights = tiny_folders["A"]
    prompt, beams, new = prompts_of(cfg["vocab_size"], [18], 12)[0], 3, 12
    want = [(0.0, [])]
    for _ in range(new):
        every = []
        for score, tail in want:
            lp = torch.log_softmax(plain_opt.forward_logits(weights, cfg, prompt + tail)[-1].double(), -1)
            every += [(score + float(lp[t]), tail + [int(t)]) for t in torch.topk(lp, beams).indices]
        want = sorted(every, key=lambda x: -x[0])[:beams]
    model = model_of(folder, kernels, beams)
    ops = model.engine.runner.ops
    logits = model.forward(torch.tensor([prompt]))
    kept = [(0.0, [])]
    for step in range(new):
        rows = len(kept)
        _, ids, best = ops.log_probs(logits, torch.zeros(rows, dtype=torch.int32, device=logits.device), beams)
        every = [(kept[b][0] + float(best[b, k]), kept[b][1] + [int(ids[b, k])], b) for b in range(rows) for k in range(beams)]
        every = sorted(every, key=lambda x: -x[0])[:beams]
        if rows == 1:
            for b in range(1, beams):
                model.engine.runner.fork(("row", 0), ("row", b))
        else:
            model.reorder_cache([b for _, _, b in every])
        kept = [(score, tail) for score, tail, _ in every]
        if step + 1 < new:
            logits = model.forward(torch.tensor([[tail[-1]] for _, tail in kept]), cache_ids=[len(prompt) + step])
        model.engine.runner.cache.check()
    assert [tail for _, tail in kept] == [tail for _, tail in want]
    # twelve log-probabilities a beam, each off by what float32 logits of this size are
    assert all(abs(a - b) < 12 * 3e-5 for (a, _), (b, _) in zip(kept, want))


@BOTH
@pytest.mark.parametrize("how", ["raises", "no token"])
def test_a_grammar_that_fails_ends_its_request_alone(tiny_folders, kernels, how):
    folder, cfg, _ = tiny_folders["A"]
    vocab = cfg["vocab_size"]
    prompts = prompts_of(vocab, [9, 12, 7], 2)

    def fails(output):
        if len(output) == 4 and how == "raises":
            raise KeyError("no rule")
        return [7, 8, vocab if len(output) == 4 else 9]
    plain = SamplingParams(max_new_tokens=9, do_sample=False, ignore_eos=True)
    steered = dataclasses.replace(plain, allowed_tokens=fails, logprobs=0)
    want = engine_of(folder, kernels).generate(prompts[1:], plain)
    engine = engine_of(folder, kernels)
    for name, prompt, params in (("a", prompts[1], plain), ("b", prompts[0], steered), ("c", prompts[2], plain)):
        engine.add_request(prompt, params, name)
    reported, ends = {}, {}
    while engine.has_work:
        for o in engine.step():
            reported.setdefault(o.req_id, []).append(o.token)
            if o.finished:
                ends[o.req_id] = o.finish_reason
    assert [reported["a"], reported["c"]] == want and ends == {"a": "length", "b": "error", "c": "length"}
    b = engine.requests["b"]
    assert reported["b"] == b.output and len(b.output) == len(b.logprobs) == 4 and set(b.output) <= {7, 8, 9}
    assert isinstance(b.error, KeyError if how == "raises" else ValueError) and engine.requests["a"].error is None
    engine.runner.cache.check()
    assert not engine.runner.cache.requests
    # calls that give whole answers raise it, and nothing is left behind
    engine = engine_of(folder, kernels)
    for kw in (dict(), dict(samples=2), dict(samples=1, best_of=3)):
        with pytest.raises(type(b.error)):
            engine.generate(prompts[:2], [steered, plain], **kw)
        assert not engine.has_work and not engine.requests and not engine.runner.cache.requests
    with pytest.raises(type(b.error)):
        model_of(folder, kernels).sample(torch.tensor(prompts[:1]), 20, allowed_tokens=fails)
    assert engine.generate(prompts[1:], plain) == want


@BOTH
def test_forks_without_params_draw_from_streams_of_their_own(tiny_folders, kernels):
    folder, cfg, _ = tiny_folders["A"]
    prompt = prompts_of(cfg["vocab_size"], [11], 4)[0]
    params = SamplingParams(max_new_tokens=20, temperature=1.5, seed=3, ignore_eos=True)
    engine = engine_of(folder, kernels, max_num_seqs=16, max_tokens=2048)
    names = engine.add_samples(prompt, params, 3, "a")
    for _ in range(5):
        engine.step()
    have = [t for t in engine.requests["a"].output if t >= 0]
    forked = [engine.fork_request("a"), engine.fork_request("a"), engine.fork_request(names[1])]
    forked += [engine.fork_request(forked[0]), engine.fork_request("a", dataclasses.replace(params, temperature=1.4, seed=50))]
    forked += [engine.fork_request(forked[-1]), engine.fork_request(forked[-1])]
    engine.run()
    forked.append(engine.fork_request(names[0], dataclasses.replace(params, max_new_tokens=24)))        # of one that has ended
    forked.append(engine.fork_request(forked[-1]))
    engine.run()
    every = [engine.requests[n] for n in names + forked]
    assert engine.requests[forked[-2]].params.seed == 3               # (as it was told)
    seeds = [q.params.seed for q in every if q.req_id != forked[-2]]
    assert len(set(seeds)) == len(seeds) == 11 and seeds[:3] == [3, 4, 5]
    assert all(engine.requests[n].output[:len(have)] == have for n in forked[:2])
    outs = [tuple(q.output) for q in every[:-2]]
    assert len(set(outs)) == len(outs)
    # a stream is the same whenever the same is asked for, and a seed of 64 bits has forks too
    again = engine_of(folder, kernels, max_num_seqs=16, max_tokens=2048)
    again.add_samples(prompt, params, 3, "a")
    for _ in range(5):
        again.step()
    first = again.fork_request("a")
    again.add_request(prompt, dataclasses.replace(params, seed=2 ** 63 - 1), "far")
    far = [again.fork_request("far") for _ in range(2)]
    again.run()
    assert again.requests[first].output == engine.requests[forked[0]].output
    assert len({tuple(again.requests[n].output) for n in ["far"] + far}) == 3


@BOTH
@pytest.mark.parametrize("run_ahead", [True, False])
def test_prompts_that_waited_for_pages_go_first_once_there_are_some(tiny_folders, kernels, run_ahead):
    """`prompts_first` holds again when a pool that was too small has been made larger."""
    folder, cfg, _ = tiny_folders["A"]
    engine = engine_of(folder, kernels, max_tokens=64, prompts_first=True, run_ahead=run_ahead)
    for i, p in enumerate(prompts_of(cfg["vocab_size"], [20, 30, 18], 6)):
        engine.add_request(p, SamplingParams(max_new_tokens=8, do_sample=False, ignore_eos=True), i)
    seen = []
    step = engine.runner.step
    engine.runner.step = lambda entries, **kw: (seen.append([(e.req, len(e.tokens)) for e in entries]), step(entries, **kw))[1]
    for _ in range(3):
        engine.step()
    assert seen == [[(0, 20), (1, 30)], [(0, 1), (1, 1)], [(0, 1), (1, 1)]] and engine.scheduler.waiting[0].req_id == 2
    engine.resize_cache(40)
    engine.step()
    assert seen[3] == [(2, 18)]
    engine.run()
    want = engine_of(folder, kernels).generate(prompts_of(cfg["vocab_size"], [20, 30, 18], 6),
                                               SamplingParams(max_new_tokens=8, do_sample=False, ignore_eos=True))
    assert [engine.requests[i].output for i in range(3)] == want
    # a pool that is too small still lets the requests that can end go on
    engine = engine_of(folder, kernels, max_tokens=64, prompts_first=True, run_ahead=run_ahead)
    for i, p in enumerate(prompts_of(cfg["vocab_size"], [20, 30, 18], 6)):
        engine.add_request(p, SamplingParams(max_new_tokens=8, do_sample=False, ignore_eos=True), i)
    for size in (4, 5, 4, 4, 5):
        engine.step()
        engine.resize_cache(size)
    engine.run()
    assert [engine.requests[i].output for i in range(3)] == want


def everything_of(m):
    """What the tables say and what the tensors hold of every request, as values to compare."""
    def raw(t):                  # (what was never written may be no number)
        return t.contiguous().cpu().numpy().tobytes()
    out = {}
    for req, r in m.requests.items():
        out[req] = (r.slot, r.num_tokens, {g: list(t) for g, t in r.tables.items()},
                    [raw(t[[p for p in r.tables[lc.group] if p >= 0]]) for lc in m.caches.values() if lc.group for t in lc.pages.values()],
                    [raw(t[r.slot]) for lc in m.caches.values() for t in lc.state.values()])
    return out, sorted(m.slots._free), {n: sorted(g.pool._free) for n, g in m.groups.items()}


@BOTH
@pytest.mark.parametrize("state", [False, True])
def test_a_reorder_that_fails_changes_nothing(kernels, state, monkeypatch):
    from types import SimpleNamespace
    from transformers_neuronx_amd.engine.runner import ModelRunner
    m = manager(kernels, state=state, num_pages=30, max_seqs=5)
    runner = SimpleNamespace(cache=m, raise_if_lost=lambda: None)
    names, held = list("abcd"), {}
    for i, name in enumerate(names):
        m.add_request(name)
        held[name] = [100 * i + k for k in range(1, 46)]
        m.grow(name, 45)
        fill(m, name, 0, held[name])
        m.advance(name, 45)
        if state:
            for t in m.caches[3].state.values():
                t[m.slot_of(name)] = i + 1.0
    m.fork("a", "e")
    m.free_request("e")
    before = everything_of(m)
    copy, calls = m.ops.copy_rows, []
    for fails_at in range(1, 3 + state):                     # of the pages of two groups, and the slots
        calls.clear()

        def fails(*a):
            calls.append(a)
            if len(calls) == fails_at:
                raise MemoryError
            return copy(*a)
        monkeypatch.setattr(m.ops, "copy_rows", fails)
        with pytest.raises(MemoryError):
            ModelRunner.reorder(runner, names, [2, 2, 0, 2])
        monkeypatch.setattr(m.ops, "copy_rows", copy)
        m.check()
        assert everything_of(m) == before, fails_at
    ModelRunner.reorder(runner, names, [2, 2, 0, 2])
    m.check()
    for name, p in zip(names, [2, 2, 0, 2]):
        holds(m, name, held[names[p]])
        assert not state or all((t[m.slot_of(name)] == p + 1).all() for t in m.caches[3].state.values())
    assert sorted(m.requests) == names


@BOTH
def test_a_search_over_beams_by_the_calls_of_the_model_alone(tiny_folders, kernels):
    """From one row of a prompt: `forward`, `reorder_cache`, `forward` and so on. Against whole sequences without a cache."""
    import plain_opt
    folder, cfg, weights = tiny_folders["A"]
    prompt, beams, new = prompts_of(cfg["vocab_size"], [21], 14)[0], 4, 9
    want = [(0.0, [])]
    for _ in range(new):
        every = []
        for score, tail in want:
            lp = torch.log_softmax(plain_opt.forward_logits(weights, cfg, prompt + tail)[-1].double(), -1)
            every += [(score + float(lp[t]), tail + [int(t)]) for t in torch.topk(lp, beams).indices]
        want = sorted(every, key=lambda x: -x[0])[:beams]
    model = model_of(folder, kernels, beams)
    logits, kept = model.forward(torch.tensor([prompt])), [(0.0, [])]
    for step in range(new):
        lp = torch.log_softmax(logits.double(), -1).cpu()
        every = sorted(((kept[b][0] + float(lp[b, t]), kept[b][1] + [int(t)], b) for b in range(len(kept))
                        for t in torch.topk(lp[b], beams).indices), key=lambda x: -x[0])[:beams]
        model.reorder_cache(torch.tensor([b for _, _, b in every]))
        kept = [(score, tail) for score, tail, _ in every]
        if step + 1 < new:
            logits = model.forward(torch.tensor([[tail[-1]] for _, tail in kept]), cache_ids=[len(prompt) + step])
    assert [tail for _, tail in kept] == [tail for _, tail in want]
    model.engine.runner.cache.check()
    # no more rows than there are slots, none from a row that is not there, and nothing changes where it is refused
    before = everything_of(model.engine.runner.cache)
    for bad, error in (([0] * (beams + 1), OutOfSlots), ([0, 1, 2, 3, 4], ValueError), ([-1, 0, 0, 0], ValueError)):
        with pytest.raises(error):
            model.reorder_cache(bad)
        assert everything_of(model.engine.runner.cache) == before
    model.forward(torch.tensor([prompt, prompt]))
    with pytest.raises(ValueError, match="live"):
        model.reorder_cache([0, 1, 2])
    model.reorder_cache([1, 0, 0, 1])
    logits = model.forward(torch.tensor([[5]] * 4), cache_ids=[len(prompt)])
    assert torch.allclose(logits, logits[:1].expand(4, -1), atol=1e-5 * float(logits.abs().max()))
    model.engine.runner.cache.check()


@BOTH
def test_a_sequence_is_kept_where_another_cannot_take_its_name(tiny_folders, kernels):
    from transformers_neuronx_amd import ContinuousBatchingConfig, NeuronConfig
    folder, cfg, _ = tiny_folders["A"]
    prompts = prompts_of(cfg["vocab_size"], [19, 16, 13], 3)
    model = model_of(folder, kernels, 3, num_pages=4, neuron_config=NeuronConfig(continuous_batching=ContinuousBatchingConfig(max_num_seqs=3)))

    def begin(seq, prompt):
        model.forward(torch.tensor([prompt]), cache_ids=torch.arange(len(prompt)).unsqueeze(0), start_ids=[seq])
    begin(0, prompts[0])
    begin(1, prompts[1])
    cache = model.engine.runner.cache
    model.fork_sequence(1, 2)                              # a full page needs no copy
    assert cache.num_tokens(("seq", 2)) == 16
    model.forward(torch.tensor([[7]]), cache_ids=torch.tensor([[16]]), start_ids=[2])          # the last page
    before = everything_of(cache)
    with pytest.raises(OutOfPages):
        model.fork_sequence(0, 1)                          # a page for the part of a page, and sequence 2 shares the one that 1 holds
    assert everything_of(cache) == before
    with pytest.raises(ValueError):
        model.fork_sequence(5, 1)
    assert everything_of(cache) == before
    model.fork_sequence(0, 2)                              # its own page is the one that is needed
    cache.check()
    got = model.forward(torch.tensor([[9]]), cache_ids=torch.tensor([[19]]), start_ids=[2])
    want = model_of(folder, kernels, 3).forward(torch.tensor([prompts[0] + [9]]))
    assert torch.allclose(got, want, atol=2e-5 * float(want.abs().max()))
    assert everything_of(cache)[0]["seq", 1] == before[0]["seq", 1]


def test_a_score_of_a_lost_step_is_not_given(tiny_folders):
    """The last step of a text may be found void when its numbers have reached the host."""
    from transformers_neuronx_amd.kernels import LostStep
    folder, cfg, _ = tiny_folders["A"]
    model = model_of(folder, "reference")
    runner = model.engine.runner
    ids = torch.tensor(prompts_of(cfg["vocab_size"], [12, 12], 5))
    want = model.log_probs(ids)
    scored, lost = runner.ops.log_probs, []

    def after_the_launch(*a):
        lost.append(True)
        return scored(*a)

    def raise_if_lost():
        if lost:
            lost.clear()
            raise LostStep("void")
    runner.ops.log_probs, runner._raise_if_lost = after_the_launch, raise_if_lost
    model.engine.add_request(ids[0].tolist(), SamplingParams(max_new_tokens=4), "r")
    model.engine.step()
    with pytest.raises(LostStep):
        model.log_probs(ids[:1])
    # what was cached beside it is void too
    assert not runner.cache.requests and not model.engine.has_work
    runner.cache.check()
    runner.ops.log_probs = scored
    assert torch.equal(model.log_probs(ids), want)


@BOTH
def test_requests_that_allow_the_same_share_their_mask(tiny_folders, kernels):
    """Samples of one prompt, and requests with equal lists."""
    folder, cfg, _ = tiny_folders["A"]
    vocab = cfg["vocab_size"]
    engine = engine_of(folder, kernels, max_num_seqs=8)
    prompts = prompts_of(vocab, [9, 12], 2)
    seen, adjust = [], engine.runner.ops.adjust_logits

    def look(logits, rules, *a):
        seen.append(rules.flat[:8 * rules.rows].reshape(-1, 8)[:, 6].tolist())             # which of the masks each row goes by
        return adjust(logits, rules, *a)
    engine.runner.ops.adjust_logits = look
    fixed = SamplingParams(max_new_tokens=6, seed=1, ignore_eos=True, allowed_tokens=list(range(5, 90)))
    engine.add_samples(prompts[0], fixed, 4, "a")
    engine.add_request(prompts[1], dataclasses.replace(fixed, allowed_tokens=np.arange(5, 90)), "b")
    engine.add_request(prompts[1], dataclasses.replace(fixed, logit_bias={7: float("-inf")}), "c")
    masks = [engine.requests[n].mask for n in ("a", ("a", 3), "b", "c")]
    assert masks[0] is masks[1] is masks[2] and masks[3] is not masks[0]
    engine.run()
    assert [0, 0, 0, 0, 0, 1] in [sorted(rows) for rows in seen] and all(max(rows) <= 1 for rows in seen)
    assert all(5 <= t < 90 for q in engine.requests.values() for t in q.output) and 7 not in engine.requests["c"].output
    # one kept by nobody is not kept
    engine.reset()
    engine.sampler._masks_of = masks = []
    assert not engine._masks


@pytest.mark.parametrize("call", ["resize", "reorder", "fork", "score"])
def test_a_lost_step_found_between_two_steps_forgets_every_request(tiny_folders, call):
    """Also where it is found by a call that runs no step of the engine's: nothing goes on from a cache that is void."""
    from transformers_neuronx_amd import ContinuousBatchingConfig, NeuronConfig
    from transformers_neuronx_amd.kernels import LostStep
    folder, cfg, _ = tiny_folders["A"]
    model = model_of(folder, "reference", neuron_config=NeuronConfig(continuous_batching=ContinuousBatchingConfig(max_num_seqs=4)))
    engine, ids = model.engine, torch.tensor(prompts_of(cfg["vocab_size"], [12], 5))
    model.forward(ids)
    model.forward(ids, cache_ids=torch.arange(12).unsqueeze(0), start_ids=[1])
    params = SamplingParams(max_new_tokens=6, do_sample=False, ignore_eos=True)
    engine.add_request(ids[0].tolist(), params, "r")
    for _ in range(3):
        engine.step()
    asked = engine.runner._raise_if_lost

    def lost():
        engine.runner._raise_if_lost = asked
        raise LostStep("void")
    engine.runner._raise_if_lost = lost
    with pytest.raises(LostStep):
        {"resize": lambda: engine.resize_cache(30), "reorder": lambda: model.reorder_cache([0, 0]),
         "fork": lambda: model.fork_sequence(1, 2), "score": lambda: model.log_probs(ids)}[call]()
    assert not engine.has_work and not engine.requests and not engine.runner.cache.requests
    engine.runner.cache.check()
    assert engine.generate([ids[0].tolist()], params) == model_of(folder, "reference").engine.generate([ids[0].tolist()], params)


@BOTH
@pytest.mark.parametrize("state", [False, True])
def test_reorders_at_random_with_hardly_any_room(kernels, state):
    """Beams that grow, change places and become more or fewer, in pools where the pages and slots of those that are over are needed at once:
    done and right, or refused and unchanged."""
    rng = random.Random(7)
    done = refused = 0
    for trial in range(12):
        m = manager(kernels, state=state, num_pages=rng.choice([14, 18, 26]), max_seqs=rng.choice([4, 5, 6]))
        texts, states = {}, {}
        m.add_request("other")                                    # one that takes no part, and shares nothing
        m.grow("other", 9)
        fill(m, "other", 0, list(range(1, 10)))
        m.advance("other", 9)
        m.add_request(0)
        texts[0], states[0] = [], 0.0
        for turn in range(25):
            n = rng.choice([1, 1, 3, 15, 16])
            for name in sorted(texts):
                if m.can_grow(name, len(texts[name]) + n) and len(texts[name]) < 70:
                    values = [rng.randrange(1, 1 << 12) for _ in range(n)]
                    m.grow(name, len(texts[name]) + n)
                    fill(m, name, len(texts[name]), values)
                    m.advance(name, n)
                    texts[name] = texts[name] + values
                states[name] = rng.randrange(1 << 12)
                for t in m.caches[3].state.values() if state else ():
                    t[m.slot_of(name)] = states[name]
            width = rng.randint(1, 5)
            parents = [rng.choice(sorted(texts)) for _ in range(width)]
            before = everything_of(m) if kernels == "reference" else None
            try:
                m.reorder(list(range(width)), parents)
            except (OutOfPages, OutOfSlots, ValueError):
                refused += 1
                assert before is None or everything_of(m) == before
            else:
                done += 1
                kept = {b: texts[b] for b in texts if b >= width}
                kept_states = {b: states[b] for b in kept}
                texts = {**kept, **{b: texts[p] for b, p in enumerate(parents)}}
                states = {**kept_states, **{b: states[p] for b, p in enumerate(parents)}}
            m.check()
            assert set(m.requests) == set(texts) | {"other"} and m.slots.num_free == m.max_seqs - len(m.requests)
            holds(m, "other", list(range(1, 10)))
            for name in texts:
                holds(m, name, texts[name])
                assert not state or all((t[m.slot_of(name)] == states[name]).all() for t in m.caches[3].state.values())
            if rng.random() < 0.3 and len(texts) > 1:
                name = rng.choice(sorted(texts))
                m.free_request(name)
                del texts[name], states[name]
    assert done > 100 and refused > 10


def test_samples_of_the_last_seed_there_is(tiny_folders):
    """Seeds are 64 bits: the one behind the last is the first."""
    folder, cfg, _ = tiny_folders["A"]
    prompt = prompts_of(cfg["vocab_size"], [8], 3)[0]
    params = SamplingParams(max_new_tokens=12, temperature=1.5, seed=2 ** 63 - 2, ignore_eos=True)
    engine = engine_of(folder, "reference")
    names = engine.add_samples(prompt, params, 4)
    engine.run()
    assert [engine.requests[n].params.seed for n in names] == [2 ** 63 - 2, 2 ** 63 - 1, -2 ** 63, -2 ** 63 + 1]
    assert len({tuple(engine.requests[n].output) for n in names}) == 4
    model = model_of(folder, "reference")
    assert model.sample(torch.tensor([prompt, prompt]), 14, seed=2 ** 63 - 2, num_return_sequences=2).shape == (4, 14)


def test_biases_are_those_at_the_beginning(tiny_folders):
    """A dictionary that its owner goes on to change steers neither a request made before nor what is made of its params."""
    folder, cfg, _ = tiny_folders["A"]
    biases = {40: 1000.0}
    params = SamplingParams(max_new_tokens=4, seed=5, ignore_eos=True, logit_bias=biases)
    biases[41] = 2000.0
    engine = engine_of(folder, "reference")
    names = engine.add_samples([3, 4, 5], params, 3)
    names.append(engine.fork_request(names[0]))
    names.append(engine.add_request([3, 4, 5], dataclasses.replace(params, seed=None)))
    engine.run()
    assert all(engine.requests[n].output == [40] * 4 for n in names)
    assert params.logit_bias == {40: 1000.0} and SamplingParams().logit_bias is None
