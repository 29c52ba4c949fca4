"""The scheduler: admits requests, cuts prompts into portions under a token
budget, lets running requests decode, finishes them and frees what they hold.

The reference has none: `ContinuousBatchingConfig` (config.py:73-103) declares
capacities for a scheduler outside the repository, and its demo drives a fixed
batch in lock-step (generation_demo.py:474-500). The decisions below are ours.

Every decision is a function of arrival order, lengths and capacities only:
  * each step first gives one token to every running request that is decoding,
    then continues prompts in admission order, then admits waiting requests
    while a slot, pages and budget remain; a portion is what is left of the
    prompt, of the portion limit and of the budget, at least one token;
  * when the pool cannot cover a scheduled token, nothing new is admitted and
    the most recently admitted running request is put back: its pages and slot
    are freed, it rejoins the head of the waiting queue and is computed again
    from its first token later, generated tokens included (they are kept). A
    lone request that does not fit raises `OutOfPages`;
  * a request ends at its end-of-sequence token (unless told to ignore it), at
    `max_new_tokens`, or at the length limit, and frees its pages in that step
    (a `max_time`, the one decision that looks at a clock, ends it at the first
    token that comes too late).

A step's outcome may be recorded in two halves, so that the next step can be planned and started
while the device still works on this one: `record` notes what was computed and puts `PENDING` in
the place of every token that was drawn but not read yet (an end by length is known at once);
`resolve` fills in the tokens when the host has them and ends requests at their end-of-sequence
token. A request that is found to have ended this way may already be part of the step that was
started meanwhile: that run's work is wasted and its token is dropped when it is resolved.
`update` does both at once.
"""
import time
from collections import deque
from dataclasses import dataclass, field
from typing import Deque, Hashable, List, Optional

from ..cache.manager import CacheManager
from ..cache.pages import OutOfPages
from ..sampling.params import SamplingParams


PENDING = -1              # stands in `Request.output` for a token that is drawn but not read yet


def seed_behind(seed: int, count: int) -> int:
    """The seed that lies `count` behind another: 64 bits with a sign, the first behind the last."""
    return (int(seed) + count + 2 ** 63) % 2 ** 64 - 2 ** 63


@dataclass
class Family:
    """A request and all that were forked from it, and from those: no two of them draw from one random stream unless they are told to."""
    seed: int
    forks: int = 0

    def next_seed(self) -> int:
        """A seed that no other of the family has, nor the samples of a prompt beside it, whose seeds follow one another."""
        self.forks += 1
        return seed_behind(self.seed, self.forks << 40)


@dataclass(eq=False)      # a request is itself: lists of requests are searched by identity
class Request:
    req_id: Hashable
    prompt: List[int]
    params: SamplingParams
    output: List[int] = field(default_factory=list)
    num_computed: int = 0           # tokens whose keys and values are stored
    finished: bool = False
    finish_reason: Optional[str] = None
    preemptions: int = 0
    arrival: int = 0
    taken_in: float = 0.0           # when the scheduler took it in (time.monotonic), for `max_time`
    # The request whose pages this one takes its first `shared` tokens from, where it still can when it is admitted: all that both had
    # when this one was made but the newest, which it brings itself, to choose a token of its own from. The leader's portion ends there
    # too, for those waiting for it.
    leader: Optional["Request"] = field(default=None, repr=False)
    shared: int = 0
    followers: List["Request"] = field(default_factory=list, repr=False)      # that wait for this one
    family: Optional[Family] = field(default=None, repr=False)
    mask: Optional[object] = field(default=None, repr=False)   # the tokens that may be chosen next (`pack_mask`); None: all
    history_of: Optional[tuple] = None      # the (slot, preemptions) under which the device keeps its history
    # of every token of the output, where the request asks for them
    logprobs: List[float] = field(default_factory=list)
    top_logprobs: List[list] = field(default_factory=list)
    error: Optional[Exception] = field(default=None, repr=False)   # what `allowed_tokens` raised, of a request that ended for it

    @property
    def tokens(self) -> List[int]:
        return self.prompt + self.output

    @property
    def num_tokens(self) -> int:
        return len(self.prompt) + len(self.output)

    def span(self, start: int, count: int) -> List[int]:
        """Tokens start .. start + count - 1 of prompt and output taken as one sequence."""
        n = len(self.prompt)
        if start >= n:
            return self.output[start - n:start - n + count]
        if start + count <= n:
            return self.prompt[start:start + count]
        return self.prompt[start:] + self.output[:start + count - n]

    @property
    def cumulative_logprob(self) -> float:
        return float(sum(self.logprobs))

    @property
    def decoding(self) -> bool:
        """All tokens but the newest are stored: the next step brings that one token."""
        return len(self.output) > 0 and self.num_computed == self.num_tokens - 1


@dataclass(eq=False)
class ScheduledRun:
    request: Request
    start: int                      # first position of the portion
    count: int                      # tokens in the portion
    samples: bool = False           # the portion ends at the request's newest token: its last logits
                                    # pick the next one
    out_index: int = -1             # where in the request's output that token goes

    def __post_init__(self):
        self.samples = self.start + self.count == self.request.num_tokens


class Scheduler:
    def __init__(self, cache: CacheManager, max_num_seqs: int, max_num_batched_tokens: int, max_model_len: int,
                 max_portion: Optional[int] = None, prompts_first: bool = False):
        self.cache = cache
        self.max_num_seqs = min(max_num_seqs, cache.max_seqs)
        self.max_num_batched_tokens = max_num_batched_tokens
        self.max_model_len = max_model_len
        self.max_portion = max_portion or max_num_batched_tokens
        # prompts_first: while any prompt is waiting or under way, decoding requests wait (all prompts
        # are taken in before the first decode step); otherwise decoding requests go first every step
        self.prompts_first = prompts_first
        self.waiting: Deque[Request] = deque()
        self.running: List[Request] = []        # in admission order
        self.finished: List[Request] = []
        self._arrivals = 0
        self.num_preemptions = 0
        self._short = False      # pages have run out and none have come back since: no request has ended, the pool is what it was

    # ---------------------------------------------------------------- arrivals

    def add(self, request: Request) -> None:
        """Queue a request; one that can never fit the length limit is refused here
        (reference: opt/model.py:50-57 refuses a sequence longer than the position table)."""
        if not request.prompt:
            raise ValueError(f"request {request.req_id!r} has an empty prompt")
        # the last generated token is never fed back, so it needs no position
        need = len(request.prompt) + max(request.params.max_new_tokens, len(request.output)) - 1
        if need > self.max_model_len:
            raise ValueError(f"request {request.req_id!r} needs {need} positions "
                             f"({len(request.prompt)} prompt + {request.params.max_new_tokens} new); "
                             f"the limit is {self.max_model_len}")
        request.arrival = self._arrivals
        request.taken_in = time.monotonic()
        self._arrivals += 1
        if request.leader is not None:
            request.shared = request.num_tokens - 1
            request.leader.followers.append(request)
        self.waiting.append(request)

    @property
    def has_work(self) -> bool:
        return bool(self.waiting or self.running)

    def reset(self) -> None:
        """Forget every request and every count (the pages are the cache manager's to give back)."""
        self.waiting.clear()
        self.running.clear()
        self.finished.clear()
        self.num_preemptions = 0
        self._short = False

    def pool_resized(self) -> None:
        """The page pool is another: what waited for pages is tried again."""
        self._short = False

    # ---------------------------------------------------------------- requests that go on from others

    def _portion(self, req: Request, budget: int) -> int:
        """Tokens of `req` that the next step takes: what is left, of the portion limit and of the budget, and no further than where
        those that wait for it go on by themselves (at any later place a state of fixed size is no longer theirs)."""
        end = req.num_tokens
        for f in req.followers:
            if req.num_computed < f.shared < end:
                end = f.shared
        return min(end - req.num_computed, self.max_portion, budget)

    def _awaits_leader(self, req: Request) -> bool:
        return req.leader is not None and req.leader in self.running and req.leader.num_computed < req.shared

    def _take_over(self, req: Request) -> bool:
        """Fork `req` from its leader, if that still holds what it needs and there is a page for it."""
        if req.leader not in self.running or req.shared < 1 or not self.cache.can_fork(req.leader.req_id, req.shared):
            return False
        try:
            self.cache.fork(req.leader.req_id, req.req_id, req.shared)
        except OutOfPages:
            return False
        req.num_computed = req.shared
        return True

    def _leave_leader(self, req: Request) -> None:
        """It waits for its leader no longer (which may serve it again if it is put back)."""
        if req.leader is not None and req in req.leader.followers:
            req.leader.followers.remove(req)
        if req.leader is not None and req.leader.finished:
            req.leader = None

    # ---------------------------------------------------------------- one step's plan

    def _preempt_last(self, keep: Request) -> bool:
        """Put back the most recently admitted running request other than `keep`."""
        for victim in reversed(self.running):
            if victim is not keep:
                self.running.remove(victim)
                self.cache.free_request(victim.req_id)
                victim.num_computed = 0
                victim.preemptions += 1
                self.num_preemptions += 1
                self.waiting.appendleft(victim)
                return True
        return False

    def _reserve(self, req: Request, new_len: int, planned: List[ScheduledRun]) -> bool:
        """Pages for `req` up to `new_len`, putting later requests back if need be.
        False if `req` itself had to give way."""
        while True:
            try:
                self.cache.grow(req.req_id, new_len)
                return True
            except OutOfPages:
                victim_pool = [r for r in self.running if r is not req]
                if not victim_pool:
                    raise OutOfPages(f"request {req.req_id!r} alone does not fit the page pool "
                                     f"({new_len} tokens wanted)")
                victim = self.running[-1]
                if victim is req:
                    # the newest request gives way to the older ones that are already planned
                    self.running.remove(req)
                    self.cache.free_request(req.req_id)
                    req.num_computed = 0
                    req.preemptions += 1
                    self.num_preemptions += 1
                    self.waiting.appendleft(req)
                    return False
                self._preempt_last(req)
                planned[:] = [p for p in planned if p.request is not victim]

    def _plan_decoding(self, planned: List[ScheduledRun], budget: int, before_all: int) -> tuple:
        """One token for every decoding request, oldest first. Returns (budget left, pages ran out)."""
        blocked = False
        for req in list(self.running):
            if (self.num_preemptions != before_all and req not in self.running) or not req.decoding or budget <= 0:
                continue
            before = self.num_preemptions
            if self._reserve(req, req.num_computed + 1, planned):
                planned.append(ScheduledRun(req, req.num_computed, 1))
                budget -= 1
            blocked |= self.num_preemptions != before
        return budget, blocked

    def schedule(self) -> List[ScheduledRun]:
        budget = self.max_num_batched_tokens
        before_all = self.num_preemptions     # a request can have left `running` only if something was put back
        planned: List[ScheduledRun] = []
        blocked = False                       # pages ran out: admit nothing new this step
        # With `prompts_first` decoding requests wait while a prompt is waiting or under way, but only as
        # long as prompts can get on: once pages have run out (`_short`, until a request ends and frees
        # some or the pool is resized) the decoding requests go first again, since only they can end and free pages; and a step
        # in which no prompt could be planned (no slot, no page) is given to them too.
        hold = (self.prompts_first and not self._short
                and (bool(self.waiting) or any(not r.decoding for r in self.running)))
        # 1. one token for every decoding request, oldest first
        if not hold:
            budget, blocked = self._plan_decoding(planned, budget, before_all)
        # 2. the next portion of every prompt under way
        planned_ids = {id(p.request) for p in planned}
        for req in list(self.running):
            if (self.num_preemptions != before_all and req not in self.running) or req.decoding or budget <= 0:
                continue
            if id(req) in planned_ids:
                continue
            count = self._portion(req, budget)
            before = self.num_preemptions
            if self._reserve(req, req.num_computed + count, planned):
                planned.append(ScheduledRun(req, req.num_computed, count))
                budget -= count
            blocked |= self.num_preemptions != before
        # 3. admissions, in arrival order, while everything they need is there
        at = 0
        while at < len(self.waiting) and not blocked and budget > 0 and len(self.running) < self.max_num_seqs:
            req = self.waiting[at]
            if self._awaits_leader(req):
                at += 1                      # (others need not wait with it)
                continue
            if self.cache.slots.num_free == 0:
                break
            if not self._take_over(req):
                self.cache.add_request(req.req_id)
            count = self._portion(req, budget)
            if not self.cache.can_grow(req.req_id, req.num_computed + count):
                self.cache.free_request(req.req_id)
                wanted, req.num_computed = req.num_computed + count, 0
                if not self.running:
                    raise OutOfPages(f"request {req.req_id!r} alone does not fit the page pool "
                                     f"({wanted} tokens wanted)")
                self._short = True
                break
            self.cache.grow(req.req_id, req.num_computed + count)
            del self.waiting[at]
            self._leave_leader(req)
            self.running.append(req)
            planned.append(ScheduledRun(req, req.num_computed, count))
            budget -= count
        if self.num_preemptions != before_all:
            self._short = True
        if hold and not planned:
            budget, blocked = self._plan_decoding(planned, budget, before_all)
        # a request put back after it was planned is no longer in `running`
        live = {id(r) for r in self.running}
        return [p for p in planned if id(p.request) in live]

    # ---------------------------------------------------------------- after the step

    def _end(self, req: Request, reason: str, ended: List[Request]) -> None:
        req.finish_reason = reason
        if req.finished:
            return
        req.finished = True
        if req in self.running:
            self.running.remove(req)
        elif req in self.waiting:
            self.waiting.remove(req)
        if self.cache.has(req.req_id):
            self.cache.free_request(req.req_id)
        self._leave_leader(req)
        req.leader = None
        self._short = False
        self.finished.append(req)
        ended.append(req)

    def end(self, req: Request, reason: str) -> None:
        """The request is over behind the tokens it has."""
        self._end(req, reason, [])

    def abort(self, req: Request) -> None:
        """Take a request out, wherever it stands: it ends with the reason "aborted" and gives back what it
        holds. A token that a step under way is still to deliver for it is dropped when it comes (`resolve`
        finds the request shorter than the place the token was meant for)."""
        if PENDING in req.output:          # also of a request that has ended by its length with its last token under way
            del req.output[req.output.index(PENDING):]
        if not req.finished:
            self._end(req, "aborted", [])

    def record(self, runs: List[ScheduledRun]) -> List[Request]:
        """What the step computes, before its tokens are known: every run that samples gets `PENDING` as
        its request's newest token. Requests that reach `max_new_tokens` or the length limit with it end
        here and free what they hold (their last token is still to be resolved)."""
        ended = []
        for run in runs:
            req = run.request
            req.num_computed = run.start + run.count
            if not run.samples:
                continue
            run.out_index = len(req.output)
            req.output.append(PENDING)
            if len(req.output) >= req.params.max_new_tokens:
                self._end(req, "length", ended)
            elif req.num_tokens > self.max_model_len:
                self._end(req, "model_length", ended)
        return ended

    def resolve(self, runs: List[ScheduledRun], sampled: List[Optional[int]]) -> List[Optional[int]]:
        """The tokens of a recorded step (`sampled[i]` is None for runs that do not sample). Returns, run
        by run, the token that the request keeps, or None: for runs that do not sample and for runs of a
        request that had ended at an earlier token when the step was started."""
        kept: List[Optional[int]] = []
        for run, token in zip(runs, sampled):
            req = run.request
            if not run.samples:
                kept.append(None)
                continue
            if token is None:
                raise ValueError(f"request {req.req_id!r} needs a token this step")
            if run.out_index >= len(req.output):        # the request ended before this token
                kept.append(None)
                continue
            req.output[run.out_index] = int(token)
            kept.append(int(token))
            p = req.params
            if not p.ignore_eos and int(token) in p.eos_ids:
                del req.output[run.out_index + 1:]      # what was drawn after it is dropped
                self._end(req, "eos", [])
            elif p.max_time is not None and time.monotonic() - req.taken_in > p.max_time:
                del req.output[run.out_index + 1:]
                self._end(req, "time", [])
        return kept

    def update(self, runs: List[ScheduledRun], sampled: List[Optional[int]]) -> List[Request]:
        """Record what the step computed and the tokens drawn for the runs that
        sample (`sampled[i]` is None for the others). Returns the requests that ended."""
        before = len(self.finished)
        for run, token in zip(runs, sampled):
            if run.samples and token is None:
                raise ValueError(f"request {run.request.req_id!r} needs a token this step")
        self.record(runs)
        self.resolve(runs, sampled)
        return self.finished[before:]
