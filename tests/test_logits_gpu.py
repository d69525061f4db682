"""The logit-control kernel (csrc/logits.hip) against 64-bit oracles: sizes, types, strides, histories, masks, graphs."""
import math

import pytest
import torch

from kv8_oracle import logits64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ops():
    from distributed_pytorch_hpc_amd import ops

    return ops


def _check(got, want, dtype, size):
    """At most six 32-bit roundings of values below ``size``; bf16 outputs then round by half a step, 2^-8."""
    got, want = got.double().cpu(), want.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin].nan_to_num(7.0), want[~fin].nan_to_num(7.0))
    off = 6 * 2.0 ** -24 * size
    tol = off + (2.0 ** -8 * (want.abs() + off) if dtype == torch.bfloat16 else 0.0)
    err = (got - want).abs()
    assert not (err[fin] > (tol[fin] if torch.is_tensor(tol) else tol)).any(), err[fin].max()


def _case(n, v, length, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(n, v, generator=g)).to(dtype)
    few = torch.randint(0, min(v, 7), (n, length), generator=g)
    tokens = torch.where(torch.rand(n, length, generator=g) < 0.5, few, torch.randint(-3, v + 9, (n, length), generator=g))
    lens = torch.randint(0, length + 1, (n,), generator=g).int()
    lens[0] = length
    kw = dict(prompt_lengths=(lens // 2).int(), repetition=1 + torch.rand(n, generator=g),
              presence=torch.rand(n, generator=g), frequency=0.1 * torch.rand(n, generator=g),
              bias=torch.randn(n, v, generator=g), mask=_ops().pack_token_mask(torch.rand(n, v, generator=g) < 0.5))
    return x, tokens, lens, kw


def _want(x, tokens, lens, kw):
    return logits64(x, tokens, lens, *(kw.get(k) for k in ("prompt_lengths", "repetition", "presence", "frequency",
                                                           "bias", "mask")))


def _want_fast(x, tokens, lens, kw):
    """The oracle without its loop over the vocabulary: the mask in one step."""
    y = _want(x, tokens, lens, {k: t for k, t in kw.items() if k != "mask"})
    bits = (kw["mask"].long()[:, :, None] >> torch.arange(32)) & 1
    return y.masked_fill(bits.flatten(1)[:, :y.shape[1]] == 0, -math.inf)


def _run(x, tokens, lens, kw):
    d = lambda t: None if t is None else t.to(DEV)   # noqa: E731
    return _ops().process_logits(d(x), d(tokens), d(lens), **{k: d(t) for k, t in kw.items()})


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,length", [(1, 1, 1), (3, 31, 40), (2, 33, 0), (4, 4096, 300), (2, 4099, 1000),
                                        (1, 32000, 65), (5, 12345, 7), (1, 9000, 6500), (2, 8195, 7001),
                                        (17, 97000, 3)])
def test_all_controls(dph_native, dtype, n, v, length):
    x, tokens, lens, kw = _case(n, v, length, dtype, v)
    want = _want(x, tokens, lens, kw) if n * v < 10 ** 6 else _want_fast(x, tokens, lens, kw)
    _check(_run(x, tokens, lens, kw), want, dtype, 2.0 ** 6 + 0.1 * length)


@pytest.mark.parametrize("parts", ["", "repetition", "presence", "frequency", "prompt_lengths frequency", "bias", "mask",
                                   "repetition mask", "bias mask", "presence bias"])
def test_each_control_alone(dph_native, parts):
    x, tokens, lens, kw = _case(3, 1000, 90, torch.float32, 3)
    kw = {k: t for k, t in kw.items() if k in parts.split()}
    _check(_run(x, tokens, lens, kw), _want(x, tokens, lens, kw), torch.float32, 64)
    if not any(k in parts for k in ("rep", "pres", "freq")):   # without penalties the history may be left out
        _check(_run(x, None, None, kw), _want(x, None, None, kw), torch.float32, 64)


def test_shared_rows_strides_and_views(dph_native):
    """A bias and a mask for all rows, broadcast ones, and operands that are views into wider buffers."""
    ops = _ops()
    x, tokens, lens, kw = _case(4, 777, 50, torch.bfloat16, 8)
    shared = dict(kw, bias=kw["bias"][0], mask=kw["mask"][1])
    want = _want(x, tokens, lens, shared)
    _check(_run(x, tokens, lens, shared), want, torch.bfloat16, 64)
    wide = torch.zeros(4, 800, dtype=torch.bfloat16, device=DEV)
    wide[:, 5:782] = x.to(DEV)
    hist = torch.full((4, 61), 2, dtype=torch.int64, device=DEV)
    hist[:, 3:53] = tokens.to(DEV)
    kd = {k: t.to(DEV) for k, t in kw.items()}
    kd["bias"], kd["mask"] = kd["bias"][:1].expand(4, -1), kd["mask"][1:2].expand(4, -1)
    got = ops.process_logits(wide[:, 5:782], hist[:, 3:53], lens.to(DEV), **kd)
    assert got.is_contiguous()
    _check(got, want, torch.bfloat16, 64)
    odd = torch.zeros(4, 780, device=DEV)[:, 1:778]   # a bias at an odd row address
    odd.copy_(kw["bias"])
    _check(ops.process_logits(wide[:, 5:782], hist[:, 3:53], lens.to(DEV),
                              **{**kd, "bias": odd}), _want(x, tokens, lens, dict(kw, mask=kw["mask"][1])),
           torch.bfloat16, 64)


def test_extreme_values(dph_native):
    """Infinities and NaN keep the formula's result; masked places are -inf whatever stood there; a row may lose all."""
    x, tokens, lens, kw = _case(3, 300, 40, torch.float32, 9)
    tokens[0, :6] = torch.tensor([0, 1, 2, 3, 4, 5])
    x[0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, 3e38])
    x[1, 7], x[1, 8] = math.nan, torch.finfo(torch.float32).min
    x[0, 100], x[0, 101], x[0, 102] = math.inf, -math.inf, math.nan
    x = x.clamp(-1e30, 1e30).where(torch.isfinite(x) & (x.abs() < 1e30), x)
    kw["mask"][2] = 0
    kw["mask"][0, 0] = -1
    kw["bias"][1, 9] = -math.inf
    got = _run(x, tokens, lens, kw)
    assert (got[2] == -math.inf).all()
    want = _want(x.clone(), tokens, lens, kw)
    keep = x.abs() < 1e30
    _check(torch.where(keep.to(DEV), got, 0), torch.where(keep, want, 0), torch.float32, 64)
    for i, j in ((0, 0), (0, 1), (0, 2), (0, 5), (0, 100), (0, 101), (0, 102), (1, 7), (1, 8)):
        g, w = float(got[i, j]), float(want[i, j])
        assert g == pytest.approx(w, rel=2.0 ** -20, nan_ok=True), (i, j)


def test_negative_and_oversized_lengths(dph_native):
    """A length below zero is none, one past the buffer the buffer's; a prompt longer than the history leaves no
    generated token."""
    x, tokens, lens, kw = _case(3, 200, 20, torch.float32, 10)
    lens = torch.tensor([-5, 999, 20], dtype=torch.int32)
    kw["prompt_lengths"] = torch.tensor([0, 3, 50], dtype=torch.int32)
    _check(_run(x, tokens, lens, kw), _want(x, tokens, lens, kw), torch.float32, 64)


def test_one_token_many_times(dph_native):
    """100 000 copies of one id: an exact count, the same on every run."""
    n = 100000
    x = torch.zeros(1, 5000)
    tokens = torch.full((1, n), 4321, dtype=torch.int64)
    kw = dict(frequency=torch.tensor([2.0 ** -10]), presence=torch.tensor([0.5]))
    got = _run(x, tokens, torch.tensor([n], dtype=torch.int32), kw)
    assert float(got[0, 4321]) == -(n * 2.0 ** -10 + 0.5) and (got[0, :4321] == 0).all()


def test_no_rows_and_no_columns(dph_native):
    ops = _ops()
    assert ops.process_logits(torch.zeros(0, 50, device=DEV)).shape == (0, 50)
    assert ops.process_logits(torch.zeros(3, 0, device=DEV)).shape == (3, 0)


def test_graph_replays(dph_native):
    """A captured call follows the history as it grows on the device; replays with eager work between them equal eager."""
    ops = _ops()
    x, tokens, lens, kw = _case(2, 6000, 50, torch.float32, 11)
    xd, td, kd = x.to(DEV), tokens.to(DEV), {k: t.to(DEV) for k, t in kw.items()}
    ld = torch.tensor([3, 20], dtype=torch.int32, device=DEV)
    ops.process_logits(xd, td, ld, **kd)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.process_logits(xd, td, ld, **kd)
    for step in range(6):
        xd.copy_(x * (1 + step))
        g.replay()
        assert torch.equal(y, ops.process_logits(xd, td, ld, **kd))
        ld += 5
        torch.cuda.synchronize()


def test_more_rows_than_wide_workgroups(dph_native):
    """2^22 + 1 rows of four tokens with a history each: 1024 threads a row would be more than a launch takes.  Integers,
    so the result is exact."""
    ops = _ops()
    n = 2 ** 22 + 1
    x = (torch.arange(4 * n, device=DEV) % 97).float().view(n, 4)
    tokens = (torch.arange(n, device=DEV) % 4)[:, None]
    got = ops.process_logits(x, tokens, torch.ones(n, dtype=torch.int32, device=DEV),
                             presence=(torch.arange(n, device=DEV) % 5).float())
    want = x.scatter_add(1, tokens, -(torch.arange(n, device=DEV) % 5).float()[:, None])
    assert torch.equal(got, want)


@pytest.mark.parametrize("v", [64, 65])
def test_repetition_penalties_whose_reciprocal_leaves_32_bits(dph_native, v):
    """1 / r is infinite for r = 2^-140 and has lost digits for r = 1.3 * 2^127, x / r is neither: one rounding from it.
    A penalty of infinity leaves zero, one of zero infinity."""
    r = torch.tensor([2.0 ** -140, 1.3 * 2.0 ** 127, 2.0 ** -126, 2.0 ** 126, math.inf, 0.0])
    x = torch.linspace(1, 1000, v).repeat(6, 1)
    x[0] *= 2.0 ** -30
    x[2] *= 2.0 ** -30
    x[1] *= 2.0 ** 100
    x[3] *= 2.0 ** 100
    x[:4, ::3] *= -2.0 ** -20   # times r, not divided
    tokens = torch.arange(v).repeat(6, 1)
    got = _run(x, tokens, torch.full((6,), v, dtype=torch.int32), dict(repetition=r)).cpu()
    want = torch.where(x > 0, x.double() / r[:, None].double(), x.double() * r[:, None].double())
    assert (got[4] == 0).all() and (got[5] == math.inf).all()
    # half a step of the result (2^-24, and of the least subnormal), for the reciprocal a second rounding
    err = (got[:4].double() - want[:4]).abs()
    fits = want[:4].float().isfinite()
    assert (err <= 2 * 2.0 ** -24 * want[:4].abs() * (1 + 2.0 ** -20) + 2.0 ** -149)[fits].all()
    assert (got[:4].isinf() & (got[:4].sign() == want[:4].sign()))[~fits].all()
    assert fits[0].all() and fits[2].all()
