"""What a request asks of the sampler."""
import operator
from dataclasses import dataclass
from typing import Callable, Dict, List, Optional, Sequence, Tuple, Union

import numpy as np


@dataclass
class SamplingParams:
    """Per-request sampling options.

    The names and meanings follow the reference's host loops (sampling.py:131-180,
    :311-378) and its `GenerationConfig` (config.py:106-139):
    temperature  logits are divided by it before filtering (:337-338); 0 selects the
                 argmax, as does do_sample=False
    top_k        the k largest logits are kept (:151, :210-211); 0 keeps all
    top_p        of those, the shortest prefix in descending order whose softmax mass
                 reaches top_p (:213-249); 1.0 keeps all
    min_tokens_to_keep  neither filter leaves fewer tokens than this (:204-205, :232;
                 `top_p_min_tokens` of the `GenerationConfig`)
    seed         the request's own random stream: draw number n of the request uses the
                 counter n, whatever else is in the batch; None lets the engine give one
                 (its own seed plus the request's number of arrival)
    deterministic  every draw uses 0.5 in place of a random number (hlo.py:2455-2456)
    eos_token_id the token that ends the request, or a list of such tokens (sampling.py:319-322)
    ban_eos      the end-of-sequence token is never chosen (`scores[:, eos] = -inf`,
                 sampling.py:143-144, the OPT loop's behaviour)
    ignore_eos   generation does not stop at the end-of-sequence token
    no_repeat_ngram_size  n: no run of n tokens appears twice in the prompt and what follows it; a token
                 that would complete a run seen before gets the logit -inf before anything else is done
                 (sampling.py:267-309, :334-335); 0 switches it off
    repetition_penalty  the logit of every token of the prompt and of what follows it is divided by this if it is
                 above zero, multiplied by it otherwise; 1.0 switches it off
    frequency_penalty  subtracted from a token's logit for every time it was generated (the prompt does not count)
    presence_penalty   subtracted from the logit of every token that was generated
    logit_bias   {token: what is added to its logit}, after the penalties; -inf bars the token
    allowed_tokens  the tokens that may be chosen: their ids, or a truth value for every token of the vocabulary; all
                 others are barred, whatever their biases. A function of the list of tokens generated so far that gives
                 either steers the request through a grammar; the request ends, with the reason "grammar", where
                 nothing is allowed after a token (a request for which nothing is allowed to begin with is refused). Where
                 the function raises, or names what is no token, its request alone ends, with the reason "error"
                 and the exception as its `error`; calls that give whole answers raise it once all have ended
    logprobs     an integer: each token is reported with its log-probability and with those of this many tokens of the
                 largest logits (0: its own alone). They are those of the logits that the token was chosen from, with
                 penalties, biases and bars, before temperature, top-k and top-p; None: not reported
    max_time     seconds: the request ends after the first token that arrives later than this after it was
                 taken in (stopping_criteria.py:15-35, `MaxTimeCriteria`)
    max_new_tokens  the most tokens to generate
    """
    max_new_tokens: int = 16
    do_sample: bool = True
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    seed: Optional[int] = 0
    min_tokens_to_keep: int = 1
    deterministic: bool = False
    eos_token_id: Optional[Union[int, Sequence[int]]] = None      # one token or several (sampling.py:319-322)
    ban_eos: bool = False
    ignore_eos: bool = False
    no_repeat_ngram_size: int = 0
    max_time: Optional[float] = None
    repetition_penalty: float = 1.0
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    logit_bias: Optional[Dict[int, float]] = None
    allowed_tokens: Optional[Union[Sequence[int], Callable[[List[int]], Sequence[int]]]] = None
    logprobs: Optional[int] = None

    MOST_LOGPROBS = 32

    def __post_init__(self):
        least, most = float(np.finfo(np.float32).tiny), float(np.finfo(np.float32).max)
        if not least <= float(self.repetition_penalty) <= most:
            raise ValueError(f"repetition_penalty has to be a positive number, but is {self.repetition_penalty}")
        for name in ("frequency_penalty", "presence_penalty"):
            if not abs(float(getattr(self, name))) <= most:
                raise ValueError(f"{name} has to be a finite number, but is {getattr(self, name)}")
        biases = {operator.index(t): float(b) for t, b in dict(self.logit_bias or {}).items()}
        if any(not (abs(b) <= most or b == float("-inf")) for b in biases.values()):
            raise ValueError("a logit bias is a finite number, or -inf for a token that must not be chosen")
        if self.logit_bias is not None:
            self.logit_bias = biases                     # not the caller's, who may go on to change it
        self.biases: Tuple[Tuple[int, float], ...] = tuple(sorted(biases.items()))     # what is gone by from here on
        if self.logprobs is not None and not (isinstance(self.logprobs, int) and 0 <= self.logprobs <= self.MOST_LOGPROBS):
            raise ValueError(f"logprobs has to be an integer from 0 to {self.MOST_LOGPROBS}, but is {self.logprobs}")
        if self.max_new_tokens < 0:
            raise ValueError("max_new_tokens must not be negative")
        if not isinstance(self.top_k, int) or self.top_k < 0:
            raise ValueError("top_k has to be a non-negative int (0 keeps all tokens).")
        if not 0.0 < float(self.top_p) <= 1.0:
            raise ValueError("top_p has to be a strictly positive float that less than or equal to 1.0.")
        if not isinstance(self.min_tokens_to_keep, int) or self.min_tokens_to_keep < 1:
            raise ValueError("min_tokens_to_keep has to be a positive int.")
        if self.no_repeat_ngram_size and (not isinstance(self.no_repeat_ngram_size, int) or self.no_repeat_ngram_size <= 0):
            raise ValueError(f"`ngram_size` has to be a strictly positive integer, but is {self.no_repeat_ngram_size}")
        if float(self.temperature) < 0:
            raise ValueError("temperature has to be a non-negative float (0 is greedy).")
        # one token or several, of any integer type (a numpy or tensor scalar too): settled here, not when
        # the first token is compared with it
        if self.eos_token_id is not None:
            try:
                self.eos_token_id = operator.index(self.eos_token_id)
            except TypeError:
                try:
                    self.eos_token_id = tuple(operator.index(t) for t in self.eos_token_id)
                except TypeError:
                    raise ValueError(f"eos_token_id has to be an integer or a sequence of integers, got "
                                     f"{self.eos_token_id!r}") from None

    @property
    def eos_ids(self) -> Tuple[int, ...]:
        """The tokens that end the request, as a tuple (empty: none does)."""
        if self.eos_token_id is None:
            return ()
        if isinstance(self.eos_token_id, int):
            return (self.eos_token_id,)
        return tuple(int(t) for t in self.eos_token_id)

    @property
    def penalised(self) -> bool:
        """Whether the choice goes by what the request holds already."""
        return self.repetition_penalty != 1.0 or self.frequency_penalty != 0.0 or self.presence_penalty != 0.0

    @property
    def follows_grammar(self) -> bool:
        """Whether what is allowed is asked anew for every token."""
        return callable(self.allowed_tokens)

    @property
    def greedy(self) -> bool:
        return (not self.do_sample) or self.temperature == 0.0 or self.top_k == 1

    @staticmethod
    def greedy_params(max_new_tokens: int, eos_token_id=None, ignore_eos=True) -> "SamplingParams":
        return SamplingParams(max_new_tokens=max_new_tokens, do_sample=False, eos_token_id=eos_token_id,
                              ignore_eos=ignore_eos)
