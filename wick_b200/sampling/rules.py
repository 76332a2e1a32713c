"""What a caller asks of a sequence's logits beside the sampler's options, and its arrays on the device.

:class:`LogitRules` is one sequence's rules; :class:`Steering` holds those of a batch's rows with what each row has said so far, and applies
them to a step's logits in one launch (``ops.steer_logits``), before the sampler's cuts:

1. a token that occurred in the prompt or the output: its logit divided by the repetition penalty if positive, multiplied
   otherwise (wick ``src/sampler.rs:76-85``);
2. less ``frequency_penalty`` times the number of times it was generated, and less ``presence_penalty`` if it was;
3. plus its bias;
4. -inf for every token outside ``allowed``.
"""
from __future__ import annotations

import dataclasses
import math
from typing import Dict, Mapping, Optional, Sequence, Tuple

import numpy as np
import torch


@dataclasses.dataclass
class LogitRules:
    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    bias: Mapping[int, float] = dataclasses.field(default_factory=dict)      # token id -> what is added to its logit
    allowed: Optional[Sequence[int]] = None                                  # the only token ids that may be sampled

    def check(self, vocab: int) -> None:
        for name in ("frequency_penalty", "presence_penalty"):
            if not math.isfinite(getattr(self, name)):
                raise ValueError(f"{name} must be a finite number")
        for what, ids in (("bias", self.bias), ("allowed", () if self.allowed is None else self.allowed)):
            for t in ids:
                if not 0 <= int(t) < vocab:
                    raise ValueError(f"token id {t} of {what} is outside the vocabulary of {vocab}")
        if any(math.isnan(float(b)) for b in self.bias.values()):
            raise ValueError("a bias is not a number")
        ruled_out = {int(t) for t, b in self.bias.items() if float(b) == -math.inf}
        if len(ruled_out) >= vocab or (self.allowed is not None and ruled_out.issuperset(int(t) for t in self.allowed)):
            raise ValueError("no token is allowed")


class Steering:
    """The rules and histories of a batch's rows, on the device.  rules: one per row; repetition: the sampler's penalty."""

    def __init__(self, rules: Sequence[LogitRules], repetition: float, vocab: int, device):
        from .. import ops
        for r in {id(r): r for r in rules}.values():
            r.check(vocab)
        self.vocab = vocab
        n = len(rules)
        up = lambda v, dtype: torch.from_numpy(np.ascontiguousarray(v, dtype=dtype)).to(device)      # noqa: E731
        self.seen = self.counts = self.penalties = self.masks = self.mask_of = None
        self.bias: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None
        if repetition != 1.0 or any(r.frequency_penalty or r.presence_penalty for r in rules):
            self.seen = torch.zeros((n, ops.bit_words(vocab)), dtype=torch.int32, device=device)
            self.counts = torch.zeros((n, vocab), dtype=torch.int32, device=device)
            self.penalties = up([[repetition, r.frequency_penalty, r.presence_penalty] for r in rules], np.float32)
        if any(r.bias for r in rules):
            cu = np.cumsum([0] + [len(r.bias) for r in rules])
            self.bias = (up(cu, np.int32), up([int(t) for r in rules for t in r.bias], np.int32),
                         up([float(b) for r in rules for b in r.bias.values()], np.float32))
        if any(r.allowed is not None for r in rules):
            which: Dict[tuple, int] = {}
            mask_of = [-1 if r.allowed is None else which.setdefault(tuple(sorted(set(int(t) for t in r.allowed))), len(which)) for r in rules]
            words = np.zeros((len(which), ops.bit_words(vocab)), dtype=np.uint32)
            for ids, k in which.items():
                at = np.array(ids, dtype=np.int64)
                np.bitwise_or.at(words[k], at // 32, np.uint32(1) << (at % 32).astype(np.uint32))
            self.masks, self.mask_of = up(words.view(np.int32), np.int32), up(mask_of, np.int32)

    @staticmethod
    def wanted(rules: Sequence[Optional[LogitRules]]) -> bool:
        return any(r is not None for r in rules)

    def said(self, tokens: torch.Tensor, rows: torch.Tensor, generated: bool) -> None:
        """``tokens`` (int32 on the device) occurred in ``rows`` (int32, a row per token; a negative row: left out)."""
        if self.seen is not None:
            from .. import ops
            ops.history_add(self.seen, self.counts, tokens, rows, generated)

    def apply(self, logits: torch.Tensor, rows: torch.Tensor) -> None:
        """In place."""
        from .. import ops
        if self.seen is not None or self.bias is not None or self.masks is not None:
            ops.steer_logits(logits, rows, seen=self.seen, counts=self.counts, penalties=self.penalties, bias=self.bias, masks=self.masks,
                             mask_of=self.mask_of)
