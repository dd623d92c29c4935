"""Rules that a request puts on the choice of its tokens: penalties on tokens that were there before, biases, a set of
allowed tokens. ``TokenRules`` is what a request carries, ``RuleStore`` keeps the rules of the sequences in flight on the device
in the form that ``ops.llm.choose_tokens`` reads.

No reference counterpart (vLLM is a README bullet in the reference, README.md:73)."""
from __future__ import annotations

import math
import numbers
import operator
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..ops import llm

MAX_BIASES = 256


@dataclass(frozen=True)
class TokenRules:
    """Neutral values change nothing. `bias`: token id -> added to its logit. `allowed`: the only tokens that may be chosen."""
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: Dict[int, float] = field(default_factory=dict)
    allowed: Optional[Tuple[int, ...]] = None

    def check(self, vocab: int) -> "TokenRules":
        """These rules in plain ints and floats; ValueError unless every number is one, finite and in range for a vocabulary of
        `vocab` tokens, and every token a whole number below that."""
        def number(x) -> float:
            if isinstance(x, bool) or not isinstance(x, numbers.Real):
                raise ValueError(f"rules: {x!r} is no number")
            return float(x)

        def token(t) -> int:
            if isinstance(t, bool):
                raise ValueError(f"rules: {t!r} is no token")
            return operator.index(t)

        try:
            penalties = number(self.repetition), number(self.frequency), number(self.presence)
            bias = {token(t): number(x) for t, x in self.bias.items()}
            allowed = None if self.allowed is None else tuple(token(t) for t in self.allowed)
        except (TypeError, OverflowError, AttributeError) as e:
            raise ValueError(f"rules: {e}") from None
        if not all(math.isfinite(x) and abs(x) <= 1e30 for x in (*penalties, *bias.values())) or not 1e-30 <= penalties[0]:
            raise ValueError("rules: penalties and biases must be finite numbers, the repetition penalty above 0")
        if len(bias) > MAX_BIASES or not all(0 <= t < vocab for t in bias):
            raise ValueError(f"rules: at most {MAX_BIASES} biases, of tokens below {vocab}")
        if allowed is not None and (not allowed or not all(0 <= t < vocab for t in allowed)):
            raise ValueError(f"rules: allowed tokens must be a list of one token below {vocab} at least")
        return TokenRules(*penalties, bias, allowed)

    @staticmethod
    def from_request(req: dict, vocab: int) -> Optional["TokenRules"]:
        """From the fields of a completion request; None where it has none of them, ValueError where one is no good."""
        keys = ("repetition_penalty", "frequency_penalty", "presence_penalty", "logit_bias", "allowed_token_ids")
        if all(req.get(k) is None for k in keys):
            return None

        def number(key: str, neutral: float) -> float:
            x = req.get(key)
            if x is None:
                return neutral
            if isinstance(x, bool) or not isinstance(x, (int, float)):
                raise ValueError(f"{key} must be a number")
            return float(x)

        bias, allowed = req.get("logit_bias"), req.get("allowed_token_ids")
        bias = {} if bias is None else bias
        if not isinstance(bias, dict) or any(isinstance(x, bool) or not isinstance(x, (int, float)) for x in bias.values()):
            raise ValueError("logit_bias must map token ids to numbers")
        if allowed is not None and not (isinstance(allowed, list) and all(isinstance(t, int) and not isinstance(t, bool) for t in allowed)):
            raise ValueError("allowed_token_ids must be a list of token ids")
        try:
            return TokenRules(number("repetition_penalty", 1.0), number("frequency_penalty", 0.0), number("presence_penalty", 0.0),
                              {int(t): float(x) for t, x in bias.items()}, None if allowed is None else tuple(allowed)).check(vocab)
        except OverflowError as e:
            raise ValueError(f"rules: {e}") from None


class RuleStore:
    """`sets` sets of rules, each with room for a history of `max_len` tokens. A set belongs to one sequence from `take` to
    `give_back`; `follow` brings its history up to date before a launch."""

    def __init__(self, sets: int, max_len: int, vocab: int, device):
        self.vocab = vocab

        def zeros(*shape, dtype=torch.int32):
            return torch.zeros(shape, dtype=dtype, device=device)

        self.history, self.prompt_lens, self.lens = zeros(sets, max_len), zeros(sets), zeros(sets)
        self.penalties = zeros(3, sets, dtype=torch.float32)
        self.bias_ids, self.bias_values = zeros(sets, MAX_BIASES), zeros(sets, MAX_BIASES, dtype=torch.float32)
        self.mask, self.mask_rows = zeros(sets, -(-vocab // 32)), zeros(sets)
        self.device = self.lens.device
        self._free: List[int] = list(range(sets - 1, -1, -1))
        self._known = [0] * sets            # tokens of the sequence that the device has

    def take(self, rules: TokenRules, prompt_len: int) -> int:
        i = self._free.pop()
        try:
            self._fill(i, rules, prompt_len)
        except BaseException:
            self._free.append(i)
            raise
        return i

    def _fill(self, i: int, rules: TokenRules, prompt_len: int) -> None:
        ids = np.full(MAX_BIASES, -1, dtype=np.int32)
        values = np.zeros(MAX_BIASES, dtype=np.float32)
        ids[:len(rules.bias)] = list(rules.bias)
        values[:len(rules.bias)] = list(rules.bias.values())
        self.bias_ids[i].copy_(torch.from_numpy(ids))
        self.bias_values[i].copy_(torch.from_numpy(values))
        self.penalties[:, i] = torch.tensor([rules.repetition, rules.frequency, rules.presence], device=self.device)
        self.prompt_lens[i] = prompt_len
        if rules.allowed is not None:
            bits = np.zeros(self.mask.shape[1] * 32, dtype=np.uint8)
            bits[list(rules.allowed)] = 1
            self.mask[i].copy_(torch.from_numpy(np.packbits(bits, bitorder="little").view("<i4").astype(np.int32)))
        self.mask_rows[i] = i if rules.allowed is not None else -1
        self._known[i] = 0

    def give_back(self, i: int) -> None:
        self._free.append(i)

    def follow(self, sequences: Sequence[Tuple[int, Sequence[int], Sequence[int]]]) -> None:
        """(set, prompt, output) of sequences: their new tokens go to the device in one copy."""
        new: List[Tuple[int, int, int]] = []
        for i, prompt, out in sequences:
            n = len(prompt) + len(out)
            new.extend((i, k, prompt[k] if k < len(prompt) else out[k - len(prompt)]) for k in range(self._known[i], n))
            self._known[i] = n
        if new:
            sets, places, tokens = torch.tensor(new, dtype=torch.int64).t().contiguous().to(self.device)
            self.history[sets, places] = tokens.to(torch.int32)
            upto = torch.tensor([(i, len(p) + len(o)) for i, p, o in sequences], dtype=torch.int64).t().contiguous().to(self.device)
            self.lens[upto[0]] = upto[1].to(torch.int32)

    def rules(self, rows: torch.Tensor) -> llm.LogitRules:
        """For a launch whose row b follows set rows[b] (-1: none)."""
        return llm.LogitRules(self.history, self.prompt_lens, self.lens, self.penalties[0], self.penalties[1], self.penalties[2],
                              self.bias_ids, self.bias_values, self.mask, self.mask_rows, rows)
