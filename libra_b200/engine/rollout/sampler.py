"""Token sampling: temperature, top-k and top-p (nucleus), with the sampled
token's logprob under the temperature-scaled distribution (what the rollout
returns as ``token_logprobs``; reference ``engine/rollout_engine.py:255``).

Penalties, biases, allowed tokens and a grammar change the logits before all
of that (``ops.control_logits``), so a controlled request's logprobs, top
logprobs included, are those of the distribution it was sampled from."""

from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Any, Dict, List, Optional

import torch

# The controls are applied in fp32.  Lowering a logit may take it to -inf, which excludes the token, but no control may
# raise one out of fp32 (its softmax would be NaN): not with 2^31 occurrences, nor divided by a small temperature.
_MOST_LOWER = 3.4e38
_MOST_RAISE = 1e20
_REPETITION_RANGE = (1e-20, 1e20)
_TEMPERATURE_RANGE = (1e-8, 1e8)


@dataclass
class SamplingParams:
    max_tokens: int = 1024
    temperature: float = 1.0
    top_p: float = 1.0
    top_k: int = -1
    stop_token_ids: List[int] = field(default_factory=list)
    seed: Optional[int] = None
    logprobs: bool = True
    repetition_penalty: float = 1.0     # divides positive logits of tokens already present, multiplies others
    presence_penalty: float = 0.0       # subtracted once from tokens of the output so far
    frequency_penalty: float = 0.0      # and once per occurrence there
    logit_bias: Optional[Dict[int, float]] = None
    allowed_token_ids: Optional[List[int]] = None
    grammar: Optional[Any] = None       # engine.rollout.controls.Grammar
    top_logprobs: int = 0               # most likely tokens to report beside each sampled one

    def __post_init__(self):
        if math.isnan(self.temperature) or math.isnan(self.top_p):
            raise ValueError(f"temperature and top_p must be numbers, got {self.temperature} and {self.top_p}")
        if self.temperature > 0:  # the limits themselves, one-hot and uniform, would be inf or NaN in fp32
            self.temperature = min(max(self.temperature, _TEMPERATURE_RANGE[0]), _TEMPERATURE_RANGE[1])
        self.top_p = max(self.top_p, 0.0)
        self.top_k = max(-1, min(int(self.top_k), 2 ** 31 - 1))  # (no vocabulary is larger: no filter)
        lo, hi = _REPETITION_RANGE
        if not lo <= self.repetition_penalty <= hi:
            raise ValueError(f"repetition_penalty must lie in [{lo}, {hi}], got {self.repetition_penalty}")
        for name in ("presence_penalty", "frequency_penalty"):
            if not -_MOST_RAISE <= getattr(self, name) <= _MOST_LOWER:
                raise ValueError(f"{name} must lie in [{-_MOST_RAISE}, {_MOST_LOWER}], got {getattr(self, name)}")
        if self.logit_bias:
            self.logit_bias = {int(k): float(v) for k, v in self.logit_bias.items()}
            if not all(-_MOST_LOWER <= v <= _MOST_RAISE and 0 <= k < 2 ** 31 for k, v in self.logit_bias.items()):
                raise ValueError(f"logit_bias maps token ids to numbers in [{-_MOST_LOWER}, {_MOST_RAISE}]")
        if self.allowed_token_ids is not None:
            try:
                self.allowed_token_ids = [int(t) for t in self.allowed_token_ids]
            except (TypeError, ValueError, OverflowError) as exc:
                raise ValueError(f"allowed_token_ids must be token ids: {exc}") from exc
            if not self.allowed_token_ids:
                raise ValueError("allowed_token_ids must not be empty")
        if self.top_logprobs not in range(257):
            raise ValueError(f"top_logprobs must be a whole number in [0, 256], got {self.top_logprobs}")
        self.top_logprobs = int(self.top_logprobs)

    @property
    def penalized(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    @property
    def controlled(self) -> bool:
        return (self.penalized or bool(self.logit_bias) or self.allowed_token_ids is not None
                or self.grammar is not None)


# what a caller may pass through the rollout engines and the HTTP route besides the named arguments
EXTRA_SAMPLING_KEYS = ("repetition_penalty", "presence_penalty", "frequency_penalty", "logit_bias",
                       "allowed_token_ids", "top_logprobs")


def extra_sampling(kw: Dict[str, Any]) -> Dict[str, Any]:
    """The given ones of ``EXTRA_SAMPLING_KEYS``, as ``SamplingParams`` takes them."""
    cast = {"logit_bias": lambda v: {int(k): float(x) for k, x in v.items()},
            "allowed_token_ids": lambda v: [int(t) for t in v], "top_logprobs": int}
    try:
        return {k: cast.get(k, float)(kw[k]) for k in EXTRA_SAMPLING_KEYS if kw.get(k) is not None}
    except (TypeError, AttributeError, OverflowError) as exc:
        raise ValueError(f"bad sampling argument: {exc}") from exc


def sample(logits: torch.Tensor, temperature: torch.Tensor, top_p: torch.Tensor, top_k: torch.Tensor,
           generators: Optional[List[Optional[torch.Generator]]] = None):
    """logits [B, V] (any float dtype) -> (tokens [B] int64, logprobs [B] fp32).

    temperature 0 means greedy.  Filtering is applied per row.
    """
    x = logits.float()
    greedy = temperature <= 0
    t = torch.where(greedy, torch.ones_like(temperature), temperature).unsqueeze(1)
    x = x / t
    logp_full = torch.log_softmax(x, dim=-1)
    B, V = x.shape
    need_filter = bool(((top_k > 0) & (top_k < V)).any()) or bool((top_p < 1.0).any())
    probs_logits = x
    if need_filter:
        sorted_x, idx = torch.sort(x, dim=-1, descending=True)
        ranks = torch.arange(V, device=x.device).unsqueeze(0)
        k = torch.where(top_k > 0, top_k, torch.full_like(top_k, V)).unsqueeze(1)
        drop = ranks >= k
        cum = torch.softmax(sorted_x, dim=-1).cumsum(-1)
        drop |= (cum - torch.softmax(sorted_x, dim=-1)) > top_p.unsqueeze(1)
        sorted_x = sorted_x.masked_fill(drop, float("-inf"))
        probs_logits = torch.full_like(x, float("-inf")).scatter(1, idx, sorted_x)
    probs = torch.softmax(probs_logits, dim=-1)
    if generators is not None and any(g is not None for g in generators):
        toks = torch.stack([torch.multinomial(probs[i], 1, generator=g).squeeze(0) if g is not None
                            else torch.multinomial(probs[i], 1).squeeze(0) for i, g in enumerate(generators)])
    else:
        toks = torch.multinomial(probs, 1).squeeze(1)
    toks = torch.where(greedy, x.argmax(-1), toks)
    return toks, logp_full.gather(1, toks.unsqueeze(1)).squeeze(1)
