"""Per-request control of what is sampled: penalties for repeated tokens, biases and grammar masks (ops.process_logits).

``LogitControls`` is what a request asks for; ``LogitProcessor`` holds a batch's history, penalties, biases and mask on the
device and applies all of them in one kernel per step.  Both generation loops take them:

    gen.generate(prompts, 64, controls=LogitControls(repetition_penalty=1.2))
    batcher.submit(prompt, 64, controls=LogitControls(allowed=grammar.allowed_tokens))
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, Mapping, Optional, Sequence, Union

import torch

from .. import ops

# What is sampled from has to stay finite where a token is allowed (softmax makes NaN of a row without a finite entry, and
# sampling from that ends a process on the GPU).  Logits below 2^36 times a repetition penalty of 2^64, less 2^31 copies
# of a token times 2^64, plus a bias of 2^100 stay below 2^102 in 32 and in 16 bits, and below 2^127 when divided by a
# temperature of 2^-25.
MAX_PENALTY = 2.0 ** 64
MAX_BIAS = 2.0 ** 100


@dataclass
class LogitControls:
    """repetition_penalty r > 0: the logit of every token of the prompt or output is divided by r if positive, else
    multiplied; frequency / presence: subtracted for each generated copy / once (penalties of up to 2^64, repetition also
    of at least 2^-64); bias: {token: value} or fp32 [V], added (below -2^100, as a type's lowest value is, it stands for
    -inf: never this token); allowed: called with the generated ids before each token, returns a bool [V] tensor (True: may be sampled) or None for
    no limit."""
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    bias: Union[Mapping[int, float], torch.Tensor, None] = None
    allowed: Optional[Callable[[Sequence[int]], Optional[torch.Tensor]]] = None

    def __post_init__(self):
        if not 1 / MAX_PENALTY <= self.repetition_penalty <= MAX_PENALTY:
            raise ValueError(f"LogitControls: repetition_penalty must be in [2^-64, 2^64], got {self.repetition_penalty}")
        if not (abs(self.presence_penalty) <= MAX_PENALTY and abs(self.frequency_penalty) <= MAX_PENALTY):
            raise ValueError("LogitControls: penalties must be finite, 2^64 at most")

    @property
    def penalizes(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    def bias_row(self, vocab: int) -> Optional[torch.Tensor]:
        if self.bias is None:
            return None
        if isinstance(self.bias, torch.Tensor):
            row = self.bias.detach().cpu()
            if tuple(row.shape) != (vocab,):
                raise ValueError(f"LogitControls: bias must have {vocab} entries, got {tuple(row.shape)}")
        else:
            row = torch.zeros(vocab, dtype=torch.float64)
            for t, v in self.bias.items():
                if not 0 <= t < vocab:
                    raise ValueError(f"LogitControls: bias for token {t} outside the vocabulary of {vocab}")
                row[t] = v
        if bool((row.isnan() | (row > MAX_BIAS)).any()):
            raise ValueError("LogitControls: biases must be 2^100 at most, or -inf")
        row = row.masked_fill(row < -MAX_BIAS, -math.inf).float()
        if bool((row == -math.inf).all()):
            raise ValueError("LogitControls: biases of -inf leave no token")
        return row


class LogitProcessor:
    """Controls of ``batch`` rows (sequences or cache slots) of up to ``max_len`` tokens.

    ``start(i, prompt, controls)`` begins a row, ``restrict(i, generated)`` asks its ``allowed`` for the next token's mask,
    ``processor(logits)`` returns the controlled logits, ``push(tokens)`` appends one sampled token to every begun row and
    ``stop(i)`` ends one (its logits pass unchanged).  History and lengths stay on the device.  What can be refused is
    refused in ``start`` and ``restrict``, before a step has run."""

    def __init__(self, batch: int, max_len: int, vocab: int, device):
        self.vocab = vocab
        self.controls: list = [None] * batch
        self.banned: list = [None] * batch                      # host bool [V]: biases of -inf
        self.tokens = torch.zeros(batch, max_len, dtype=torch.long, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.prompt = torch.zeros(batch, dtype=torch.int32, device=device)
        self.live = torch.zeros(batch, dtype=torch.int32, device=device)
        self._held = [0] * batch                                # lengths, known on the host
        self.penalties = torch.zeros(3, batch, device=device)   # repetition, presence, frequency
        self.penalties[0] = 1.0
        self.bias: Optional[torch.Tensor] = None                # [batch, V], with the first row that has one
        self.mask = torch.full((batch, (vocab + 31) // 32), -1, dtype=torch.int32, device=device)

    def start(self, i: int, prompt: Sequence[int], controls: LogitControls) -> None:
        if len(prompt) > self.tokens.shape[1]:
            raise ValueError(f"LogitProcessor: prompt of {len(prompt)} tokens, room for {self.tokens.shape[1]}")
        row = controls.bias_row(self.vocab)
        self.stop(i)
        self.banned[i] = None if row is None else row == -math.inf
        self.controls[i] = controls
        self.tokens[i, :len(prompt)] = torch.as_tensor(list(prompt), dtype=torch.long)
        self.lengths[i] = self.prompt[i] = self._held[i] = len(prompt)
        self.live[i] = 1
        self.penalties[:, i] = torch.tensor([controls.repetition_penalty, controls.presence_penalty,
                                             controls.frequency_penalty])
        if row is not None:
            if self.bias is None:
                self.bias = torch.zeros(len(self.controls), self.vocab, device=self.tokens.device)
            self.bias[i] = row.to(self.bias.device)

    def stop(self, i: int) -> None:
        c, self.controls[i] = self.controls[i], None
        if c is None:
            return
        self.lengths[i] = self.live[i] = self._held[i] = 0
        if c.allowed is not None:
            self.mask[i] = -1
        if c.bias is not None:
            self.bias[i] = 0.0

    def push(self, tokens: torch.Tensor) -> None:
        """Append one token per begun row (LongTensor [batch] on the processor's device); the last place of a full history
        is overwritten."""
        at = self.lengths.clamp(max=self.tokens.shape[1] - 1).long()[:, None]
        self.tokens.scatter_(1, at, torch.where(self.live > 0, tokens, 0)[:, None])
        self.lengths.add_(self.live).clamp_(max=self.tokens.shape[1])
        self._held = [n if c is None else min(n + 1, self.tokens.shape[1]) for n, c in zip(self._held, self.controls)]

    def push_one(self, i: int, token: int) -> None:
        """Append one token to row i alone (the first token of a request that joins a running batch)."""
        n = min(int(self.lengths[i]), self.tokens.shape[1] - 1)
        self.tokens[i, n] = token
        self.lengths[i] = self._held[i] = n + 1

    def restrict(self, i: int, generated: Sequence[int]) -> None:
        """Mask of row i's next token, given the ids generated so far; nothing to do for a row without ``allowed``."""
        c = self.controls[i]
        if c is None or c.allowed is None:
            return
        a = c.allowed(list(generated))
        if a is None:
            self.mask[i] = -1
            return
        if a.dtype != torch.bool or tuple(a.shape) != (self.vocab,):
            raise ValueError(f"LogitControls: allowed must return a bool tensor of {self.vocab} entries")
        a = a.cpu()
        if not bool((a if self.banned[i] is None else a & ~self.banned[i]).any()):
            raise ValueError(f"LogitControls: allowed (and biases of -inf) leave no token for row {i}")
        self.mask[i] = ops.pack_token_mask(a).to(self.mask.device)

    def __call__(self, logits: torch.Tensor, row: Optional[int] = None) -> torch.Tensor:
        """logits [batch, V] of every row, or [1, V] of ``row``."""
        s = slice(None) if row is None else slice(row, row + 1)
        mine = [c for c in self.controls[s] if c is not None]
        history = {}
        if any(c.penalizes for c in mine):
            # the columns in use, not the room: the kernel is chosen by the width of the history that it is given
            history = dict(tokens=self.tokens[s, :max(self._held[s])], lengths=self.lengths[s],
                           prompt_lengths=self.prompt[s], repetition=self.penalties[0, s],
                           presence=self.penalties[1, s], frequency=self.penalties[2, s])
        bias = self.bias[s] if any(c.bias is not None for c in mine) else None
        mask = self.mask[s] if any(c.allowed is not None for c in mine) else None
        if not history and bias is None and mask is None:
            return logits
        return ops.process_logits(logits, **history, bias=bias, mask=mask)
