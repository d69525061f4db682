"""Block-scaled 8-bit KV cache (csrc/kv8.hip): append, single-token decode attention and read-back.

The cache of ops.decode holds e4m3 entries under ONE scale that the caller has to know; here every block of T tokens of a
KV head has its own, taken from the block itself, so int8 (or e4m3) entries need no calibration.  With pos[b] tokens of
sequence b stored, ``KV8Cache`` holds

  k, v              [B, Smax, Hkv, D]     int8 / float8_e4m3fn codes of the blocks j < pos[b] // T
  k_scale, v_scale  [B, Smax // T, Hkv]   fp32, value = code * scale
  k_tail, v_tail    [B, T, Hkv, D]        bf16 rows of the open block (row t % T)

with scale = max(amax / QMAX, 2^-126) and code = round(x * (1 / scale)) over the bf16 entries x of a block that has just
been filled, QMAX = 127 (int8) or 448 (e4m3).  The open block stays bf16, so what n tokens leave in the cache does not
depend on how they were grouped into appends.  A block with an entry that is not finite has the scale NaN and reads back
as NaN; until it is full, its infinities are values like others.  Positions only grow (or restart at 0): an earlier token
cannot be taken back out of a block that was quantised.

GPU tensors run the HIP kernels (the extension must be present); CPU tensors run the PyTorch references below, which are
also the oracles of tests/test_kv8_gpu.py.  There is no backward: operands that require grad are refused.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib
from .decode import FP8_KV, FP8_MAX, _split

TINY_SCALE = 2.0 ** -126
HEAD_DIMS = (32, 64, 128)   # of the HIP kernels; the references take any even one
QMAX = {torch.int8: 127.0, FP8_KV: FP8_MAX}


class KV8Cache(NamedTuple):
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    k_tail: torch.Tensor
    v_tail: torch.Tensor

    @property
    def block(self) -> int:
        return self.k_tail.shape[1]

    def slot(self, i: int) -> "KV8Cache":
        """The cache of sequence i (a view)."""
        return KV8Cache(*(t[i:i + 1] for t in self))


def kv8_cache(batch: int, max_len: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.int8,
              block: int = 64, device=None) -> KV8Cache:
    """An empty cache.  A head's rows (and scales) lie next to each other in memory, [B, Hkv, Smax, D] under the
    [B, Smax, Hkv, D] view: decode attention streams one head's rows per workgroup."""
    if dtype not in QMAX:
        raise ValueError(f"kv8_cache: dtype must be torch.int8 or torch.float8_e4m3fn, got {dtype}")
    if block not in (16, 32, 64, 128):
        raise ValueError(f"kv8_cache: block must be 16, 32, 64 or 128 tokens, got {block}")

    def part(rows, dt, *d):
        return torch.zeros(batch, n_kv_heads, rows, *d, dtype=dt, device=device).transpose(1, 2)

    return KV8Cache(part(max_len, dtype, head_dim), part(max_len, dtype, head_dim),
                    part(max_len // block, torch.float32), part(max_len // block, torch.float32),
                    part(block, torch.bfloat16, head_dim), part(block, torch.bfloat16, head_dim))


def _no_grad(name: str, *ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad() or on detached tensors")


def _check(cache: KV8Cache, pos, qkv=None, n_heads: int = 0, n_kv_heads: int = 0, tables=()) -> None:
    """The refusals of the native operators for the CPU path, but for what only kernels need: HEAD_DIMS, strides, alignment
    and operands that lie apart."""
    k, v, ks, vs, kt, vt = cache
    b, smax, h, d = k.shape
    t = kt.shape[1]
    if k.dtype not in QMAX or v.dtype != k.dtype or any(x.dtype != torch.float32 for x in (ks, vs)) or \
            any(x.dtype != torch.bfloat16 for x in (kt, vt)):
        raise ValueError("kv8: int8 or float8_e4m3fn codes, fp32 scales, bf16 tails")
    if t not in (16, 32, 64, 128):
        raise ValueError("kv8: the block must be 16, 32, 64 or 128 tokens")
    if v.shape != k.shape or any(tuple(x.shape) != (b, smax // t, h) for x in (ks, vs)) or \
            any(tuple(x.shape) != (b, t, h, d) for x in (kt, vt)):
        raise ValueError("kv8: scales [B, Smax / T, Hkv] and tails [B, T, Hkv, D] must match k / v [B, Smax, Hkv, D]")
    if pos.dtype != torch.int32 or tuple(pos.shape) != (b,):
        raise ValueError("kv8: pos must be an int32 [B] tensor")
    if qkv is not None and (qkv.dim() != 3 or n_kv_heads != h or n_heads < 1 or n_heads % h or qkv.shape[0] != b
                            or qkv.shape[2] != (n_heads + 2 * h) * d):
        raise ValueError("kv8: qkv must be [B, S, (Hq + 2 Hkv) * D], Hq a multiple of Hkv")
    for c in tables:
        if c.dtype != torch.float32 or c.dim() != 2 or c.shape[0] < smax or c.shape[1] != d // 2:
            raise ValueError("kv8_append: rope tables must be fp32 [>= Smax, D / 2]")


# ------------------------------------------------------------------------------------------------- references
def quantize_block(x: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 blocks [..., T, Hkv, D] -> (codes, fp32 scales [..., Hkv])."""
    w = x.to(torch.bfloat16).float()
    amax = w.abs().amax((-3, -1))   # NaN propagates
    scale = torch.where(torch.isfinite(amax), (amax / QMAX[dtype]).clamp_min(TINY_SCALE), math.nan)
    q = w * scale.reciprocal()[..., None, :, None]
    q = torch.where(scale.isnan()[..., None, :, None], 0.0, q)
    q = q.round().clamp(-127, 127) if dtype == torch.int8 else q.clamp(-FP8_MAX, FP8_MAX)
    return q.to(dtype), scale


def _rotate64(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Interleaved pairs of [S, H, D] by the angles [S, D / 2]: products in 64 bits, one rounding to x's type."""
    a, b = x.double().unflatten(-1, (-1, 2)).unbind(-1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2).float().to(x.dtype)


def kv8_append_reference(qkv, cache: KV8Cache, pos, cos, sin, n_heads: int, n_kv_heads: int) -> None:
    t, smax = cache.block, cache.k.shape[1]
    q, k, v = _split(qkv, n_heads, n_kv_heads, cache.k.shape[-1])
    s = qkv.shape[1]
    for b, p in enumerate(pos.tolist()):   # before anything is stored
        if p < 0 or p + s > smax:
            raise ValueError(f"kv8 cache overflow: sequence {b} at {p} + {s} > capacity {smax}")
    for b, p in enumerate(pos.tolist()):
        for x in (q, k):
            x[b].copy_(_rotate64(x[b], cos[p:p + s], sin[p:p + s]))
        first, end = p // t, (p + s) // t
        for x, code, scale, tail in ((k[b], cache.k[b], cache.k_scale[b], cache.k_tail[b]),
                                     (v[b], cache.v[b], cache.v_scale[b], cache.v_tail[b])):
            rows = torch.cat([tail[:p % t], x.to(torch.bfloat16)])   # from row first * t on
            for j in range(first, end):
                c, sc = quantize_block(rows[(j - first) * t:(j - first + 1) * t], code.dtype)
                code[j * t:(j + 1) * t] = c
                scale[j] = sc
            left = rows[(end - first) * t:]
            tail[:left.shape[0]] = left


def _rows(cache: KV8Cache, b: int, n: int) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 keys and values [n, Hkv, D] of the n tokens of sequence b."""
    t = cache.block
    out = []
    for code, scale, tail in ((cache.k, cache.k_scale, cache.k_tail), (cache.v, cache.v_scale, cache.v_tail)):
        full = n // t
        x = code[b, :full * t].float() * scale[b, :full].repeat_interleave(t, 0)[..., None]
        out.append(torch.cat([x, tail[b, :n % t].float()]))
    return out[0], out[1]


def kv8_read_reference(cache: KV8Cache, pos, count: int) -> tuple[torch.Tensor, torch.Tensor]:
    bsz, smax, h, d = cache.k.shape
    ko = torch.zeros(bsz, count, h, d, dtype=torch.bfloat16, device=cache.k.device)
    vo = torch.zeros_like(ko)
    for b, n in enumerate(pos.tolist()):
        n = max(0, min(n, smax))
        m = min(n, count)
        for o, x in zip((ko, vo), _rows(cache, b, n)):
            o[b, count - m:] = x[n - m:].to(torch.bfloat16)
    return ko, vo


def kv8_decode_attention_reference(qkv, cache: KV8Cache, pos, n_heads: int, n_kv_heads: int, scale: float):
    d, smax = cache.k.shape[-1], cache.k.shape[1]
    q = _split(qkv, n_heads, n_kv_heads, d)[0]
    out = torch.zeros(qkv.shape[0], n_heads * d, dtype=qkv.dtype, device=qkv.device)
    for b, p in enumerate(pos.tolist()):
        n = max(0, min(p, smax - 1) + 1)
        if n:
            k, v = (x.transpose(0, 1) for x in _rows(cache, b, n))
            qb = q[b, 0].float().view(n_kv_heads, n_heads // n_kv_heads, d)
            w = torch.softmax(qb @ k.transpose(1, 2) * scale, -1)
            out[b] = (w @ v).reshape(-1).to(qkv.dtype)
    return out


# ------------------------------------------------------------------------------------------------- operators
def kv8_append_(qkv: torch.Tensor, cache: KV8Cache, pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                n_heads: int, n_kv_heads: int) -> None:
    """Store S new tokens per sequence at positions pos[b] .. pos[b] + S - 1: rotate q and k in place in ``qkv``
    [B, S, (Hq + 2 Hkv) * D], quantise every block that fills, keep the rest in the tail.  ``pos`` (int32 [B], on the
    cache's device: a captured graph advances it there) is not advanced; the caller checks the capacity -- on the GPU,
    tokens past Smax are dropped."""
    _no_grad("kv8_append_", qkv)
    if _lib.use_native(qkv):
        _lib.ops().kv8_append_(qkv, *cache, pos, cos, sin, n_heads, n_kv_heads)
        return
    _no_grad("kv8_append_", *cache, cos, sin)
    _check(cache, pos, qkv, n_heads, n_kv_heads, (cos, sin))
    kv8_append_reference(qkv, cache, pos, cos, sin, n_heads, n_kv_heads)


def kv8_decode_attention(qkv: torch.Tensor, cache: KV8Cache, pos: torch.Tensor, n_heads: int, n_kv_heads: int,
                         scale: float | None = None, max_len: int | None = None) -> torch.Tensor:
    """Attention of the single new token per sequence (qkv [B, 1, ...], already appended) over keys 0 .. pos[b];
    returns [B, Hq * D].  ``max_len`` bounds pos + 1 over the batch (default: the capacity, as in a captured graph); it
    only sets how the work is split.  A sequence with pos[b] < 0 has no key: its output is zero."""
    _no_grad("kv8_decode_attention", qkv)
    scale = 1.0 / math.sqrt(cache.k.shape[-1]) if scale is None else scale
    if _lib.use_native(qkv):
        return _lib.ops().kv8_decode_attention(qkv, *cache, pos, n_heads, n_kv_heads, scale,
                                               cache.k.shape[1] if max_len is None else max_len)
    _no_grad("kv8_decode_attention", *cache)
    _check(cache, pos, qkv, n_heads, n_kv_heads)
    if qkv.shape[1] != 1:
        raise ValueError("kv8_decode_attention: one token per sequence (qkv [B, 1, ...])")
    if max_len is not None and not 1 <= max_len <= cache.k.shape[1]:
        raise ValueError("kv8_decode_attention: max_len must be in [1, Smax]")
    return kv8_decode_attention_reference(qkv, cache, pos, n_heads, n_kv_heads, scale)


def kv8_read(cache: KV8Cache, pos: torch.Tensor, count: int,
             out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The last ``count`` of every sequence's pos[b] stored rows as bf16 (k, v) [B, count, Hkv, D]; rows before the first
    token are zero.  ``out``: two tensors (views) of that shape to write into."""
    if _lib.use_native(cache.k):
        if out is None:
            return _lib.ops().kv8_read(*cache, pos, count)
        if any(o.dim() != 4 or o.shape[1] != count for o in out):
            raise ValueError(f"kv8_read: out must be two [B, {count}, Hkv, D] tensors")
        _lib.ops().kv8_read_(*cache, pos, *out)
        return out
    _no_grad("kv8_read", *cache, *(out or ()))
    _check(cache, pos)
    if not 0 <= count <= cache.k.shape[1]:
        raise ValueError(f"kv8_read: count {count} is not in 0 .. {cache.k.shape[1]}")
    kv = kv8_read_reference(cache, pos, count)
    if out is None:
        return kv
    if any(o.shape != x.shape for o, x in zip(out, kv)):
        raise ValueError(f"kv8_read: out must be two tensors of shape {tuple(kv[0].shape)}")
    for o, x in zip(out, kv):
        o.copy_(x)
    return out
