"""Penalties for repeated tokens, biases and masks on the logits of a generate() loop, before the choice.

No counterpart in the reference, whose ``sample_token`` (src/kivi_sycl/generation/sampling.py:10-25) takes logits as
they are.  With x the logit of a token that the row has had in its prompt or since::

    x = x / repetition if x > 0 else x * repetition

a token that the row has said (the prompt's are not said) loses ``frequency`` for each time and ``presence`` once;
then its bias is added; then what is not allowed becomes -inf.  Logits on a CUDA device go through one kernel of the
library (``kivi_adjust_logits``); logits on the CPU through the same formula in torch.
"""
from typing import Callable, Mapping, Optional

import torch

__all__ = ["LogitRules"]


class LogitRules:
    """The rules of one run over ``prompt`` [batch, tokens] with room for ``max_new`` tokens a row.

    ``said(ids)`` tells it what was chosen, ``rules(logits)`` gives adjusted logits [batch, vocab].  ``bias``: numbers by
    token id, the same for every row.  ``allowed(ids)``: called before each choice with the ids so far [batch, tokens]; returns
    int32 words [1 or batch, (vocab + 31) // 32], bit i % 32 of word i / 32 for token i, or None where everything is
    allowed."""

    def __init__(self, prompt: torch.Tensor, max_new: int, device=None, repetition: float = 1.0, frequency: float = 0.0, presence: float = 0.0,
                 bias: Optional[Mapping[int, float]] = None, allowed: Optional[Callable[[torch.Tensor], Optional[torch.Tensor]]] = None):
        if not repetition > 0:
            raise ValueError(f"repetition ({repetition}) must be positive")
        B, n = prompt.shape
        self.device = torch.device(device) if device is not None else prompt.device
        self.batch, self.given, self.held = B, n, n
        # ids that are not there yet are -1, which counts for nothing: the arrays stay the same from step to step
        self.tokens = torch.full((B, n + max_new), -1, dtype=torch.int64, device=self.device)
        self.tokens[:, :n] = prompt
        self.allowed, self.bias = allowed, dict(bias or {})
        self.penalties = (float(repetition), float(frequency), float(presence))
        full = lambda x, dtype=torch.float32: torch.full((B,), x, dtype=dtype, device=self.device)  # noqa: E731
        self._args = {}
        if self.penalties != (1.0, 0.0, 0.0):
            self._args.update(cu_tokens=(torch.arange(B + 1, dtype=torch.int32) * (n + max_new)).to(self.device), prompt_lens=full(n, torch.int32),
                              repetition=full(repetition), frequency=full(frequency), presence=full(presence))
        if self.bias:
            ids = torch.tensor(list(self.bias), dtype=torch.int64).repeat(B)
            numbers = torch.tensor(list(self.bias.values()), dtype=torch.float32).repeat(B)
            self._args.update(bias_ids=ids.to(self.device), bias=numbers.to(self.device),
                              cu_bias=(torch.arange(B + 1, dtype=torch.int32) * len(self.bias)).to(self.device))

    def said(self, ids: torch.Tensor) -> None:
        """The step's ids [batch] or [batch, 1]."""
        if self.held == self.tokens.shape[1]:
            raise RuntimeError(f"more than the {self.held - self.given} tokens that the rules were made for")
        self.tokens[:, self.held] = ids.reshape(self.batch)
        self.held += 1

    def __call__(self, logits: torch.Tensor) -> torch.Tensor:
        if logits.dim() != 2 or logits.shape[0] != self.batch:
            raise ValueError(f"logits must be [{self.batch}, vocab]")
        mask = self.allowed(self.tokens[:, :self.held]) if self.allowed is not None else None
        if mask is not None:
            words = (logits.shape[1] + 31) // 32
            if mask.dtype != torch.int32 or mask.dim() != 2 or mask.shape[0] not in (1, self.batch) or mask.shape[1] < words:
                raise ValueError(f"allowed must give int32 [1 or {self.batch}, {words}]")
        if not self._args and mask is None:
            return logits
        if not logits.is_cuda:
            return self._on_host(logits, mask)
        from ..extension.loader import kivi_native
        if logits.dtype not in (torch.float32, torch.bfloat16):
            logits = logits.float()
        if logits.stride(-1) != 1:
            logits = logits.contiguous()
        args = dict(self._args)
        if "cu_tokens" in args:
            args["tokens"] = self.tokens
        if mask is not None:
            args["allowed"] = mask.to(logits.device).expand(self.batch, -1).contiguous()
        return kivi_native.adjust_logits(logits, **args)

    def _on_host(self, logits: torch.Tensor, mask: Optional[torch.Tensor]) -> torch.Tensor:
        x, V = logits.float().clone(), logits.shape[1]
        repetition, frequency, presence = self.penalties
        for b in range(self.batch):
            if "cu_tokens" in self._args:
                had = self.tokens[b, :self.held]
                had = torch.where((had < 0) | (had > V), V, had)             # (ids outside count for nothing)
                said = torch.bincount(had[self.given:], minlength=V + 1)[:V].float()
                seen = torch.bincount(had, minlength=V + 1)[:V] > 0
                x[b] = torch.where(seen, torch.where(x[b] > 0, x[b] / repetition, x[b] * repetition), x[b]) - frequency * said - presence * (said > 0)
            for i, number in self.bias.items():
                if 0 <= i < V:
                    x[b, i] += number
            if mask is not None:
                at = torch.arange(V)
                x[b].masked_fill_((mask[min(b, mask.shape[0] - 1)].cpu()[at // 32] >> (at % 32)) & 1 == 0, float("-inf"))
        return x.to(logits.dtype)
