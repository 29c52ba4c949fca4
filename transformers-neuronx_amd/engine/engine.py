"""The engine: requests in, tokens out. It joins the scheduler, the step
function and the sampler; everything between a request's tokens and its next
token passes through `step()`.
"""
import contextlib
import dataclasses
import itertools
import time
import weakref
from dataclasses import dataclass
from typing import Callable, Dict, Hashable, List, Optional, Sequence

import torch

from ..config.engine_config import EngineConfig
from ..kernels import LostStep
from ..sampling.params import SamplingParams
from ..kernels.steering import pack_mask
from ..sampling.sampler import Sampler, Steering, banned_ngram_tokens
from .batch import StepEntry
from .runner import ModelRunner
from .scheduler import PENDING, Family, Request, ScheduledRun, Scheduler, seed_behind


@dataclass
class StepOutput:
    req_id: Hashable
    token: int
    finished: bool
    finish_reason: Optional[str]
    # of a request that asks for them (`SamplingParams.logprobs`): the token's log-probability, and (token, its own) of the largest logits
    logprob: Optional[float] = None
    top_logprobs: Optional[list] = None


@dataclass
class _StartedStep:
    """A step whose tokens are chosen on the device and not read yet."""
    runs: List[ScheduledRun]
    sampling: List[ScheduledRun]
    sent: object                         # the tokens on their way to the host (`ops.send_tokens`)
    started: float
    scores: object = None                # the tokens' log-probabilities on their way (`ops.send_log_probs`), where asked for


class LLMEngine:
    """With `run_ahead` (the default) a call of `step()` starts one step and returns the tokens of the
    step before it: the device chooses a step's tokens and keeps them where the next step's embedding
    finds them, so the host can plan, lay out and start that next step while the device still works,
    and reads the tokens only afterwards. What a request generates is the same either way; a request
    that ends at its end-of-sequence token is found out one step late, and the run it has in the step
    started meanwhile is wasted and dropped."""

    def __init__(self, runner: ModelRunner, config: EngineConfig):
        self.runner, self.config = runner, config
        max_len = min(config.max_model_len or runner.max_positions, runner.max_positions)
        self.scheduler = Scheduler(runner.cache, config.max_num_seqs, config.max_num_batched_tokens, max_len,
                                   max_portion=config.chunk_size, prompts_first=config.prompts_first)
        self.sampler = Sampler(runner.ops, runner.model.device, slots=runner.cache.max_seqs, capacity=min(runner.vocab, max_len + 1),
                               last=runner.kept_tokens)
        self.requests: Dict[Hashable, Request] = {}
        self._masks = weakref.WeakValueDictionary()       # the masks of lists of allowed tokens that requests go by, by their bytes
        self._ids = itertools.count()
        self._taken = 0                        # requests taken since the start or the last reset
        self.timings: List[dict] = []          # one record per step when `record_timings`
        self.record_timings = False
        # called with (requests that sample in this step, their logits [n, vocab] float32) before the draw
        self.logits_hook: Optional[Callable] = None
        self.run_ahead = bool(getattr(config, "run_ahead", True))
        self._started: Optional[_StartedStep] = None
        self._planned = False                  # the last call of `step()` found something to run

    # ---------------------------------------------------------------- requests

    def add_request(self, prompt: Sequence[int], params: SamplingParams, req_id: Optional[Hashable] = None):
        if params.max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        return self._add(prompt, params, req_id)

    def _add(self, prompt: Sequence[int], params: SamplingParams, req_id: Optional[Hashable], leader: Optional[Request] = None,
             output: Sequence[int] = (), family: Optional[Family] = None):
        rid = req_id if req_id is not None else next(self._ids)
        if rid in self.requests and not self.requests[rid].finished:
            raise ValueError(f"request {rid!r} is already live")
        prompt = [int(t) for t in prompt]
        vocab = self.runner.vocab
        if prompt and not 0 <= min(prompt) <= max(prompt) < vocab:
            raise ValueError(f"request {rid!r}: a token id of the prompt is outside the vocabulary of {vocab}")
        if params.biases and not 0 <= params.biases[0][0] <= params.biases[-1][0] < vocab:
            raise ValueError(f"request {rid!r}: a logit bias names a token outside the vocabulary of {vocab}")
        if params.seed is None:
            # a stream of the request's own, the same whatever else runs beside it
            params = dataclasses.replace(params, seed=int(self.config.seed) + self._taken)
        req = Request(rid, prompt, params, output=list(output), leader=leader, family=family or Family(int(params.seed)))
        if params.logprobs is not None:            # (of tokens it begins with nothing is known: 0, and no others)
            req.logprobs, req.top_logprobs = [0.0] * len(output), [[] for _ in output]
        req.mask = self._mask(req)
        if req.mask is not None and not req.mask.any():
            raise ValueError(f"request {rid!r}: no token is allowed")
        if req.mask is not None and not params.follows_grammar:
            # requests that allow the same share the array, and its row on the device. (Not those that follow a grammar: looked up for
            # every token it costs 4 us a request, and 32 requests at one place of a grammar took 2.43 ms a step for 2.39.)
            req.mask = self._masks.setdefault(req.mask.tobytes(), req.mask)
        self.scheduler.add(req)
        self._taken += 1
        self.requests[rid] = req
        return rid

    def add_samples(self, prompt: Sequence[int], params: SamplingParams, count: int, req_id: Optional[Hashable] = None) -> List[Hashable]:
        """`count` requests for one prompt, each with a random stream of its own (the seeds that follow `params.seed`). The prompt is
        computed once, by the first of them, all but its newest token; the others take its pages over, where they are admitted while
        it still runs. Their names: `req_id`, (`req_id`, 1), (`req_id`, 2) and so on, or a number each where none is given."""
        if count < 1:
            raise ValueError(f"at least one sample is wanted, got {count}")
        if params.max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        names = [next(self._ids) if req_id is None else (req_id, i) if i else req_id for i in range(count)]
        for name in names:
            if name in self.requests and not self.requests[name].finished:
                raise ValueError(f"request {name!r} is already live")
        streams = [params] + [params if params.seed is None else dataclasses.replace(params, seed=seed_behind(params.seed, i))
                               for i in range(1, count)]
        for i, (name, stream) in enumerate(zip(names, streams)):
            try:
                self._add(prompt, stream, name, leader=self.requests[names[0]] if i else None)
            except Exception:
                for added in names[:i]:                # all of them or none
                    self.abort_request(added)
                raise
        return names

    def fork_request(self, req_id: Hashable, params: Optional[SamplingParams] = None, new_id: Optional[Hashable] = None) -> Hashable:
        """Another request that goes on from where `req_id` stands, with its prompt and the tokens that have been reported of it, by
        `params` (its own with a random stream that no other of them has, if not given; `max_new_tokens` counts the tokens taken over
        too). It shares the pages of the tokens it has in common while `req_id` runs; where it cannot, they are computed again. Its name
        is returned."""
        req = self.requests[req_id]
        output = req.output[:req.output.index(PENDING)] if PENDING in req.output else list(req.output)
        if params is None:
            params = dataclasses.replace(req.params, seed=req.family.next_seed())
        if params.max_new_tokens <= len(output):
            raise ValueError(f"request {req_id!r} has {len(output)} tokens already, max_new_tokens is {params.max_new_tokens}")
        child = self._add(req.prompt, params, new_id, leader=None if req.finished else req, output=output, family=req.family)
        if params.logprobs is not None and req.params.logprobs is not None:
            q = self.requests[child]
            q.logprobs, q.top_logprobs = req.logprobs[:len(output)], req.top_logprobs[:len(output)]
        return child

    def resize_cache(self, num_pages) -> None:
        """Another number of cache pages, between two steps; live requests keep theirs (`ModelRunner.resize_cache`)."""
        with self.forgets_if_lost():
            self.runner.resize_cache(num_pages)
        self.scheduler.pool_resized()

    def _mask(self, req: Request):
        """The tokens that may come next, where the request says which: those it allows but for those barred otherwise."""
        p = req.params
        if p.allowed_tokens is None:
            return None
        vocab = self.runner.vocab
        words = pack_mask(vocab, p.allowed_tokens(list(req.output)) if p.follows_grammar else p.allowed_tokens)
        barred = [t for t, b in p.biases if b == float("-inf")] + (list(p.eos_ids) if p.ban_eos else [])
        if p.no_repeat_ngram_size:
            barred += banned_ngram_tokens(req.prompt + req.output, p.no_repeat_ngram_size)
        if barred:
            words &= ~pack_mask(vocab, [t for t in set(barred) if 0 <= t < vocab])
        return words

    @property
    def has_work(self) -> bool:
        return self.scheduler.has_work or self._started is not None

    # ---------------------------------------------------------------- one step

    def _start(self) -> Optional[_StartedStep]:
        """Plan a step, run it, choose its tokens on the device and record it with the tokens pending."""
        runs = self.scheduler.schedule()
        self._planned = bool(runs)
        if not runs:
            return None
        t0 = time.perf_counter()
        entries = []
        for run in runs:
            toks = run.request.span(run.start, run.count)
            if toks[-1] == PENDING:
                # drawn by the step before this one and not read yet: the device has it under the slot
                toks = toks[:-1] + [-1 - self.runner.cache.slot_of(run.request.req_id)]
            entries.append(StepEntry(run.request.req_id, toks, [run.count - 1] if run.samples else []))
        logits = self.runner.step(entries, kept_allowed=True)
        sampling = [r for r in runs if r.samples]
        sent = scores = None
        if sampling:
            requests = [r.request for r in sampling]
            if self.logits_hook is not None:
                self.logits_hook(requests, logits)
            histories = None
            if any(q.params.no_repeat_ngram_size for q in requests):
                # (such requests never run ahead, see `step`: every token they hold is known here)
                histories = [list(q.prompt) + list(q.output) if q.params.no_repeat_ngram_size else None
                             for q in requests]
            drawn = self.sampler.draw(logits, [q.params for q in requests], [len(q.output) for q in requests],
                                      histories, self._steering(requests))
            tops = [q.params.logprobs for q in requests if q.params.logprobs is not None]
            if tops:
                scores = self.runner.ops.send_log_probs(*self.runner.ops.log_probs(logits, drawn, min(max(tops), logits.shape[1])))
            sent = self.runner.keep_tokens(drawn)
        self.scheduler.record(runs)
        return _StartedStep(runs, sampling, sent, t0, scores)

    def _steering(self, requests: List[Request]) -> Optional[List[Optional[Steering]]]:
        if not any(q.mask is not None or q.params.penalised for q in requests):
            return None
        out: List[Optional[Steering]] = []
        for q in requests:
            steering = None
            if q.mask is not None or q.params.penalised:
                slot = self.runner.cache.slot_of(q.req_id)
                steering = Steering(slot, mask=q.mask)
                # the device goes on with the history it has, but for a request that was just admitted, or admitted again
                if q.params.penalised and q.history_of != (slot, q.preemptions):
                    if PENDING in q.output:
                        raise AssertionError(f"request {q.req_id!r} was admitted with a token that is not known yet")
                    steering.start = (q.prompt, list(q.output))
                    q.history_of = (slot, q.preemptions)
            out.append(steering)
        return out

    def _finish(self, step: _StartedStep) -> List[StepOutput]:
        """Read the tokens of a started step and give them to their requests."""
        tokens: List[Optional[int]] = [None] * len(step.runs)
        if step.sampling:
            it = iter(self.runner.receive_tokens(step.sent))
            tokens = [next(it) if r.samples else None for r in step.runs]
        kept = self.scheduler.resolve(step.runs, tokens)
        if step.scores is not None:
            log_probs, ids, best = self.runner.ops.receive_log_probs(step.scores)
            at = 0
            for r, t in zip(step.runs, kept):
                if t is not None and r.request.params.logprobs is not None:
                    top = r.request.params.logprobs
                    r.request.logprobs.append(log_probs[at])
                    r.request.top_logprobs.append(list(zip(ids[at][:top], best[at][:top])) if top else [])
                at += r.samples
        for r, t in zip(step.runs, kept):
            q = r.request
            if t is not None and not q.finished and q.mask is not None and (q.params.follows_grammar or q.params.no_repeat_ngram_size):
                try:
                    q.mask = self._mask(q)
                except Exception as error:         # the caller's function is at fault: this request ends, the others' tokens are theirs
                    q.error = error
                    self.scheduler.end(q, "error")
                else:
                    if not q.mask.any():
                        self.scheduler.end(q, "grammar")
        self.scheduler.finished.clear()        # the engine reports ends through `StepOutput`; nothing piles up
        if self.record_timings:
            self.runner.ops.synchronize()
            self.timings.append({"seconds": time.perf_counter() - step.started,
                                 "tokens": sum(r.count for r in step.runs),
                                 "prefill_tokens": sum(r.count for r in step.runs if r.count > 1 or not r.samples),
                                 "sampled": len(step.sampling)})
        out = []
        for r, t in zip(step.runs, kept):
            if t is not None:
                q = r.request
                last = q.finished and r.out_index == len(q.output) - 1
                scored = q.params.logprobs is not None
                out.append(StepOutput(q.req_id, t, last, q.finish_reason if last else None,
                                      q.logprobs[r.out_index] if scored else None, q.top_logprobs[r.out_index] if scored else None))
        return out

    @torch.no_grad()
    def step(self) -> List[StepOutput]:
        """Schedule, run, sample, record: one batch of portions and decoded tokens. Returns the tokens of
        the step it ran, or with `run_ahead` those of the step started by the call before. `LostStep`, wherever it is found:
        the tokens under way, and the keys and values cached with them, are void, and every request is forgotten."""
        try:
            return self._step()
        except LostStep:
            self.reset()
            raise

    @contextlib.contextmanager
    def forgets_if_lost(self):
        """Where what has run is found void, every request is forgotten with what is cached of it: for calls between two steps."""
        try:
            yield
        except LostStep:
            self.reset()
            raise

    def _step(self) -> List[StepOutput]:
        # a request that may not repeat its n-grams, or follows a grammar, needs its last token on the host before the next is chosen
        in_step = any((q.params.no_repeat_ngram_size or q.params.follows_grammar) and not q.finished for q in self.requests.values())
        idle = self._started is None
        if not self.run_ahead or self.record_timings or in_step:
            out = self._finish(self._started) if self._started is not None else []
            self._started = None
            started = self._start()
            self._check_progress(idle)
            return out + (self._finish(started) if started is not None else [])
        started = self._start()
        out = self._finish(self._started) if self._started is not None else []
        self._started = started
        self._check_progress(idle)
        return out

    def _check_progress(self, idle: bool) -> None:
        """Requests wait, no step was under way when this call began and the scheduler has planned none: no
        later call would do better (a pool too small for a lone request raises `OutOfPages` where it is
        found; this is what is left, and every loop over `step()` meets it)."""
        if idle and not self._planned and self.scheduler.has_work:
            raise RuntimeError("no progress: requests wait, the scheduler plans no step and none is under way")

    def profile(self, steps: int = 1, work: bool = False):
        """Run `steps` steps with events around every kernel launch (no recording, no running ahead) and
        return ({kernel: (launches, milliseconds)}, the steps' outputs); with `work` the table's entries are
        (launches, milliseconds, bytes, flops), with what the launches said they move and compute, and its
        names carry their sizes. Reference: `profile`, base.py:754-759."""
        from .. import debug
        ahead, self.run_ahead = self.run_ahead, False
        outs: List[StepOutput] = []
        try:
            with debug.kernel_timer() as t:
                for _ in range(steps):
                    if not self.has_work:
                        break
                    outs += self.step()
                table = t.work_table() if work else t.table()
        finally:
            self.run_ahead = ahead
        return table, outs

    def run(self, on_token: Optional[Callable[[StepOutput], None]] = None) -> None:
        """Step until every request has ended."""
        while self.has_work:
            for out in self.step():
                if on_token:
                    on_token(out)

    def generate(self, prompts: Sequence[Sequence[int]], params, samples: int = 1, best_of: Optional[int] = None) -> List[List[int]]:
        """Generated tokens (without the prompts) of a set of prompts; `params` is one
        `SamplingParams` for all or a list with one each. `samples` answers to each prompt, one behind the other (`add_samples`); with
        `best_of`, so many are made and those kept whose tokens have the largest sum of log-probabilities, largest first."""
        return [list(q.output) for family in self.generate_requests(prompts, params, samples, best_of) for q in family]

    def generate_requests(self, prompts: Sequence[Sequence[int]], params, samples: int = 1,
                          best_of: Optional[int] = None) -> List[List[Request]]:
        """The same as requests that have ended, `samples` a prompt."""
        plist = params if isinstance(params, (list, tuple)) else [params] * len(prompts)
        made = samples if best_of is None else best_of
        if samples < 1 or made < samples:
            raise ValueError(f"{samples} samples, at least one and no more than best_of ({best_of}), are wanted")
        if made > samples:
            plist = [sp if sp.logprobs is not None else dataclasses.replace(sp, logprobs=0) for sp in plist]
        families = [self.add_samples(p, sp, made) if made > 1 else [self.add_request(p, sp)] for p, sp in zip(prompts, plist)]
        self.run()
        out = [[self.pop_request(name) for name in names] for names in families]
        for family in out:
            self.raise_errors(family)
        if made > samples:
            out = [sorted(family, key=lambda q: -q.cumulative_logprob)[:samples] for family in out]     # (of equal ones the earlier)
        return out

    @staticmethod
    def raise_errors(requests: Sequence[Request]) -> None:
        """What the function of one of these requests raised (`Request.error`), for callers that see no `StepOutput`."""
        for q in requests:
            if q.error is not None:
                raise q.error

    def abort_request(self, req_id: Hashable) -> Request:
        """Stop a request whose caller has gone, between two calls of `step()`: its pages and its slot are
        free for the next step, no further token of it is reported (one that a step already started would
        still deliver is dropped), and the request is handed over with what it has generated so far."""
        req = self.requests[req_id]
        self.scheduler.abort(req)
        self.scheduler.finished.clear()
        return self.requests.pop(req_id)

    def pop_request(self, req_id: Hashable) -> Request:
        """Hand over a request that has ended and forget it. A request stays in `requests`, with its prompt
        and output, until this is called (or `reset`): a caller that drives `step()` itself calls it when it
        has seen the request's last token."""
        req = self.requests[req_id]
        if not req.finished:
            raise ValueError(f"request {req_id!r} has not ended")
        if PENDING in req.output:
            raise ValueError(f"request {req_id!r} has ended, but its last token is in a step under way: "
                             "the next call of step() delivers it")
        return self.requests.pop(req_id)

    def reset(self) -> None:
        """Forget every request and give back all pages (reference: `reset()` zero-fills
        the caches, decoder.py:1957-1969; here nothing needs clearing)."""
        self._started = None
        self.scheduler.reset()
        self.runner.cache.reset()
        self._taken = 0
        self.requests.clear()
