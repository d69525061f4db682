"""Control of the logits before sampling (csrc/logits.hip): penalties for repeated tokens, biases and grammar masks.

Per row of logits x [N, V], with the history tokens[n, :lengths[n]] whose first prompt_lengths[n] ids are the prompt's,
in this order and in 32 bits:

  token in the history   x = x / repetition if x > 0 else x * repetition   (the kernel: x * (1 / repetition))
  c > 0 generated copies x = x - (frequency * c + presence)
  bias                   x = x + bias
  mask bit 0             x = -inf

GPU tensors run the HIP kernel, CPU tensors the reference below, which is also the oracle of
tests/test_logits_gpu.py.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

Opt = Optional[torch.Tensor]


def pack_token_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool [..., V] (True: the token may be sampled) -> the bit mask of ``process_logits``, int32 [..., ceil(V / 32)]
    with bit v % 32 of word v // 32."""
    v = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.to(torch.int64), (0, -v % 32)).unflatten(-1, (-1, 32))
    words = (bits << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def _check(logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, mask) -> None:
    """The refusals of the native operator for the CPU path."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("process_logits: logits must be fp32 or bf16 [N, V]")
    n, v = logits.shape
    if tokens is None and any(t is not None for t in (lengths, prompt_lengths, repetition, presence, frequency)):
        raise ValueError("process_logits: lengths and penalties need tokens")
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.dim() != 2 or tokens.shape[0] != n):
        raise ValueError("process_logits: tokens must be int64 [N, L]")
    if tokens is not None and lengths is None:
        raise ValueError("process_logits: tokens need their lengths")
    for t, dt in ((lengths, torch.int32), (prompt_lengths, torch.int32), (repetition, torch.float32),
                  (presence, torch.float32), (frequency, torch.float32)):
        if t is not None and (t.dtype != dt or tuple(t.shape) != (n,)):
            raise ValueError("process_logits: lengths int32 [N] and penalties fp32 [N]")
    for t, dt, cols in ((bias, torch.float32, v), (mask, torch.int32, (v + 31) // 32)):
        if t is not None and (t.dtype != dt or tuple(t.shape) not in ((cols,), (n, cols))):
            raise ValueError("process_logits: bias fp32 [V] or [N, V], mask int32 [ceil(V / 32)] or [N, ceil(V / 32)]")


def process_logits_reference(logits, tokens=None, lengths=None, prompt_lengths=None, repetition=None, presence=None,
                             frequency=None, bias=None, mask=None):
    x = logits.float()
    n, v = x.shape
    if tokens is not None and tokens.shape[1]:
        at = torch.arange(tokens.shape[1], device=x.device)
        valid = (at < lengths[:, None]) & (tokens >= 0) & (tokens < v)
        made = valid & (at >= prompt_lengths[:, None]) if prompt_lengths is not None else valid
        ids = tokens.clamp(0, v - 1)
        seen = torch.zeros(n, v, dtype=torch.int32, device=x.device).scatter_add_(1, ids, valid.int()) > 0
        count = torch.zeros(n, v, dtype=torch.int32, device=x.device).scatter_add_(1, ids, made.int())
        if repetition is not None:
            r = repetition[:, None]
            x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        zero = x.new_zeros(n)
        f, a = (zero if t is None else t for t in (frequency, presence))
        x = torch.where(count > 0, x - (f[:, None] * count + a[:, None]), x)
    if bias is not None:
        x = x + bias
    if mask is not None:
        ids = torch.arange(v, device=x.device)
        x = torch.where((mask[..., ids // 32] >> (ids % 32)) & 1 == 1, x, -math.inf)
    return x.to(logits.dtype)


def process_logits(logits: torch.Tensor, tokens: Opt = None, lengths: Opt = None, prompt_lengths: Opt = None,
                   repetition: Opt = None, presence: Opt = None, frequency: Opt = None, bias: Opt = None,
                   mask: Opt = None) -> torch.Tensor:
    """The controlled copy of ``logits`` [N, V] (fp32 or bf16, any row stride).

    tokens int64 [N, L], lengths / prompt_lengths int32 [N] (ids outside 0 .. V - 1 are ignored; without prompt_lengths
    every id counts as generated), repetition / presence / frequency fp32 [N], bias fp32 [V] or [N, V], mask int32
    [ceil(V / 32)] or [N, ceil(V / 32)] (``pack_token_mask``).  Anything may be None.  A row whose mask allows nothing
    comes back as -inf throughout.  No backward: operands that require grad are refused."""
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("process_logits has no backward: call it under torch.no_grad() or on detached logits")
    if _lib.use_native(logits):
        return _lib.ops().process_logits(logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias,
                                         mask)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (repetition, presence, frequency, bias)):
        raise RuntimeError("process_logits has no backward: call it under torch.no_grad() or on detached tensors")
    _check(logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, mask)
    return process_logits_reference(logits, tokens, lengths, prompt_lengths, repetition, presence, frequency, bias, mask)
