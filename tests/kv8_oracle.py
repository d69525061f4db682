"""Inputs and 64-bit oracles of the 8-bit KV cache and logit tests, written apart from the operators' references."""
import math

import torch

LIM = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def make_qkv(b, s, hq, hkv, d, seed, device):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(b, s, (hq + 2 * hkv) * d, generator=g).to(torch.bfloat16).to(device)


def tables(d, n, device):
    f = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.arange(n, dtype=torch.float64)[:, None] * f
    return a.cos().float().to(device), a.sin().float().to(device)


def filled(cache, seed):
    """Fill every code, scale and tail row of a cache with values of ordinary size; returns the cache."""
    g = torch.Generator().manual_seed(seed)
    for code, scale, tail in ((cache.k, cache.k_scale, cache.k_tail), (cache.v, cache.v_scale, cache.v_tail)):
        x = torch.randn(code.shape, generator=g)
        lim = LIM[code.dtype]
        c = (x * lim / 4).clamp(-lim, lim)
        code.copy_((c.round() if code.dtype == torch.int8 else c).to(code.dtype))
        scale.copy_((0.5 + torch.rand(scale.shape, generator=g)) * 4 / lim)
        tail.copy_(torch.randn(tail.shape, generator=g).to(torch.bfloat16))
    return cache


def rows64(cache, b, n):
    """The n stored rows of sequence b as 64-bit keys and values [n, Hkv, D]."""
    out = []
    for code, scale, tail in ((cache.k, cache.k_scale, cache.k_tail), (cache.v, cache.v_scale, cache.v_tail)):
        t = tail.shape[1]
        x = [code[b, i].double() * scale[b, i // t].double()[:, None] if i < n // t * t else tail[b, i % t].double()
             for i in range(n)]
        out.append(torch.stack(x) if n else code[b, :0].double())
    return out


def attention64(qkv, cache, pos, hq, hkv, scale):
    """Output [B, Hq * D] in 64 bits and how far a kernel with 32-bit sums may be from it before its last rounding.

    Scores: a 32-bit dot product of D terms and two scalings are off by (D + 4) 2^-24 of the sum of magnitudes; a
    weight exp(s) by twice the largest such error (its own and the sum's), plus the exponential (2^-22).  The weighted
    sum over values adds n 2^-24 at most in any order of sums (counted as 32 levels of a tree and 64 serial steps) and,
    where weights enter a matrix instruction as two bf16 parts, 2^-16.  All relative to sum p |v|."""
    d = cache.k.shape[-1]
    outs, offs = [], []
    for b, p in enumerate(pos.tolist()):
        n = max(0, min(p, cache.k.shape[1] - 1) + 1)
        q = qkv[b, 0, :hq * d].double().view(hkv, hq // hkv, d)
        if n == 0:
            outs.append(torch.zeros(hq * d, dtype=torch.float64, device=qkv.device))
            offs.append(outs[-1])
            continue
        k, v = (x.transpose(0, 1) for x in rows64(cache, b, n))
        s = (q[:, :, None] * k[:, None]).sum(-1) * scale
        mag = (q[:, :, None] * k[:, None]).abs().sum(-1) * abs(scale)
        w = torch.exp(s - s.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        # an error of a score only moves the output by that key's own weight
        ds = (d + 4) * 2.0 ** -24 * mag
        dw = w * ds + w * (w * ds).sum(-1, keepdim=True) + w * (2.0 ** -22 + 2.0 ** -16 + 96 * 2.0 ** -24)
        outs.append((w[..., None] * v[:, None]).sum(2).reshape(-1))
        offs.append((dw[..., None] * v[:, None].abs()).sum(2).reshape(-1))
    return torch.stack(outs), torch.stack(offs)


def assert_close64(got, want, off):
    """Within the 32-bit error and the rounding to bf16: half a step, 2^-8 of the value, and the least subnormal."""
    tol = off + 2.0 ** -8 * (want.abs() + off) + 2.0 ** -133
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(err / tol)[bad].max():.3f} of the tolerance"


def logits64(logits, tokens, lengths, prompt, rep, pres, freq, bias, mask):
    x = logits.double().clone()
    n, v = x.shape
    for i in range(n):
        if tokens is not None:
            ids = tokens[i, :max(0, int(lengths[i]))].tolist()
            np = 0 if prompt is None else int(prompt[i])
            made = {}
            for j, t in enumerate(ids):
                if 0 <= t < v:
                    made[t] = made.get(t, 0) + (j >= np)
            for t, c in made.items():
                if rep is not None:
                    r = float(rep[i])
                    x[i, t] = x[i, t] / r if x[i, t] > 0 else x[i, t] * r
                if c:
                    x[i, t] -= (0.0 if freq is None else float(freq[i])) * c + (0.0 if pres is None else float(pres[i]))
        if bias is not None:
            x[i] += (bias if bias.dim() == 1 else bias[i]).double()
        if mask is not None:
            words = (mask if mask.dim() == 1 else mask[i]).tolist()
            for t in range(v):
                if not words[t // 32] >> (t % 32) & 1:
                    x[i, t] = -math.inf
    return x


def infinities(cache, lengths):
    """Infinities of either sign in the V of every sequence's open block, each in a column (head, d) of its own: in its
    first and its last row, two of one sign in a column; and one of each sign in a column (their sum is NaN)."""
    t = cache.v_tail.shape[1]
    for b, n in enumerate(lengths):
        if n % t:
            last, v = n % t - 1, cache.v_tail[b]
            v[0, 0, 3], v[last, 0, 4], v[0, 0, 5], v[last, 0, 5] = math.inf, -math.inf, -math.inf, -math.inf
            if last:
                v[0, 0, 9], v[last, 0, 9] = math.inf, -math.inf
    return cache


def assert_close64_inf(got, want, off):
    """``assert_close64``, with infinities and NaN where (and of the sign that) the oracle has them."""
    fin = torch.isfinite(want)
    assert torch.equal(got.double()[~fin].nan_to_num(7.0), want[~fin].nan_to_num(7.0))
    assert_close64(got[fin], want[fin], off[fin])
