"""The HIP kernels of the 8-bit KV cache and the logit controls at the edges of their values and sizes."""
import pytest
import torch

from kv8_oracle import assert_close64_inf, attention64, filled, infinities, make_qkv

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]
DECODE = [(4, 4, 32, 16), (12, 4, 64, 32), (8, 1, 128, 64), (3, 3, 128, 128), (40, 2, 64, 16), (32, 1, 128, 32)]
DEV = "cuda"


def _ops():
    from distributed_pytorch_hpc_amd import ops

    return ops


def _pos(*p):
    return torch.tensor(p, dtype=torch.int32)


def _to(cache, dev):
    return type(cache)(*(t.to(dev) for t in cache))


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d,t", DECODE)
def test_decode_attention_infinities_in_the_open_block(dph_native, code, hq, hkv, d, t):
    """An infinity in V of the open block comes out as what it is, in the row's only share and in the last of several,
    whatever the number of open rows; the other columns keep their accuracy."""
    ops = _ops()
    cap = 1900
    pos = _pos(0, t // 2, t, t + 14, 200, cap - 3, cap - 2)
    c = infinities(filled(ops.kv8_cache(7, cap, hkv, d, code, t), 5), (pos + 1).tolist())
    qkv = make_qkv(7, 1, hq, hkv, d, 6, "cpu")
    want, off = attention64(qkv, c, pos, hq, hkv, d ** -0.5)
    assert torch.isinf(want).any() and want.isnan().any()
    c, pos, qkv = _to(c, DEV), pos.to(DEV), qkv.to(DEV)
    for bound in (100, cap):
        assert_close64_inf(ops.kv8_decode_attention(qkv, c, pos, hq, hkv, max_len=bound).cpu(), want, off)
    for b in (5, 6):   # alone: more shares of the row
        got = ops.kv8_decode_attention(qkv[b:b + 1], c.slot(b), pos[b:b + 1], hq, hkv)
        assert_close64_inf(got.cpu(), want[b:b + 1], off[b:b + 1])


def test_graph_replays_over_rows_shared_by_workgroups(dph_native):
    """Two captured append + attention steps whose rows several workgroups share (one of them with rows of fewer turns than
    workgroups, one with more), each with its workspace in its graph's memory.  Replayed in turn with eager work between
    them, across borders of turns (128 -> 129, 256 -> 257, 512 -> 513 keys) and of blocks, they equal eager steps bit for
    bit: those divide the same lengths over as many workgroups."""
    from kv8_oracle import tables

    ops = _ops()
    hq, d, t, cap = 8, 64, 16, 700
    cos, sin = tables(d, cap, DEV)
    hkv = [2, 4]
    start = [_pos(120, 251, 500).to(DEV), (torch.arange(60) * 11 % 660).int().to(DEV)]
    assert 60 * 4 * 6 > 512 > 3 * 2 * 6   # turns of 128 keys at the capacity against workgroups
    caches = [_to(filled(ops.kv8_cache(len(p), cap, h, d, block=t), 40 + h), DEV) for p, h in zip(start, hkv)]
    eager = [type(c)(*(x.clone(memory_format=torch.preserve_format) for x in c)) for c in caches]
    pos, epos = [p.clone() for p in start], [p.clone() for p in start]

    def step(x, c, p, h):
        ops.kv8_append_(x, c, p, cos, sin, hq, h)
        o = ops.kv8_decode_attention(x, c, p, hq, h)
        p += 1
        return o

    bufs = [torch.zeros(len(p), 1, (hq + 2 * h) * d, dtype=torch.bfloat16, device=DEV) for p, h in zip(start, hkv)]
    graphs, outs = [], []
    for i in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(bufs[i].clone(), type(caches[i])(*(x.clone() for x in caches[i])), pos[i].clone(), hkv[i])
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(bufs[i], caches[i], pos[i], hkv[i]))
        graphs.append(g)
    for k in range(36):
        x = [make_qkv(len(start[i]), 1, hq, hkv[i], d, 200 + 2 * k + i, DEV) for i in range(2)]
        for i in (0, 1) if k % 2 else (1, 0):
            bufs[i].copy_(x[i])
            graphs[i].replay()
        if k % 5 == 0:
            torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], step(x[i], eager[i], epos[i], hkv[i])), (k, i)
            assert torch.equal(bufs[i], x[i])
        if k in (0, 17, 35):   # and are the attention of the cache as it stands
            want, off = attention64(x[0].cpu(), _to(eager[0], "cpu"), epos[0].cpu() - 1, hq, hkv[0], d ** -0.5)
            assert_close64_inf(outs[0].cpu(), want, off)
    for i in range(2):
        for name, a, b in zip(caches[i]._fields, caches[i], eager[i]):
            assert torch.equal(a.float(), b.float()), name


@pytest.mark.parametrize("cap,t", [(1, 16), (10, 64), (127, 128)])
def test_capacity_below_one_block(dph_native, cap, t):
    """No block ever fills and there is no scale: everything lives in the open block."""
    from kv8_oracle import tables

    ops = _ops()
    cos, sin = tables(64, cap, "cpu")
    ref = ops.kv8_cache(2, cap, 2, 64, block=t)
    got = _to(ref, DEV)
    assert ref.k_scale.shape == (2, 0, 2)
    x = make_qkv(2, cap, 6, 2, 64, 3, "cpu")
    gx, pos = x.to(DEV), _pos(0, 0)
    ops.kv8_append_(x, ref, pos, cos, sin, 6, 2)
    ops.kv8_append_(gx, got, pos.to(DEV), cos.to(DEV), sin.to(DEV), 6, 2)
    assert torch.equal(gx.cpu(), x) and torch.equal(got.v_tail.cpu(), ref.v_tail) and torch.equal(got.k_tail.cpu(), ref.k_tail)
    pos += cap - 1
    want, off = attention64(x[:, -1:], ref, pos, 6, 2, 0.125)
    assert_close64_inf(ops.kv8_decode_attention(gx[:, -1:], got, pos.to(DEV), 6, 2).cpu(), want, off)
    assert torch.equal(ops.kv8_read(got, pos.to(DEV) + 1, cap)[0].cpu(), ops.kv8_read(ref, pos + 1, cap)[0])
