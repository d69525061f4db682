"""HIP kernels of the block-scaled 8-bit KV cache (csrc/kv8.hip): stored bits equal to the reference's, attention within
32-bit arithmetic and one bf16 rounding of 64-bit oracles, refusals, layouts, graphs and streams."""
import pytest
import torch

from kv8_oracle import assert_close64, attention64, filled, make_qkv, rows64, tables
from kv8_refusals import REFUSED

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]
DEV = "cuda"


def _ops():
    from distributed_pytorch_hpc_amd import ops

    return ops


def _bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype != torch.float32 else t.contiguous().view(torch.int32)


def _equal(a, b, what=""):
    assert a.shape == b.shape and a.dtype == b.dtype
    n = int((_bits(a.cpu()) != _bits(b.cpu())).sum())
    assert n == 0, f"{what}: {n} of {a.numel() * a.element_size()} bytes or words differ"


def _same(a, b):
    for name, x, y in zip(a._fields, a, b):
        _equal(x, y, name)


def _to(cache, dev):
    return type(cache)(*(t.to(dev) for t in cache))


def _pos(*p):
    return torch.tensor(p, dtype=torch.int32)


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refusals(dph_native, name):
    with pytest.raises((RuntimeError, ValueError)):
        REFUSED[name](DEV)


@pytest.mark.parametrize("part", ["strides", "alignment", "last dim", "devices", "overlap", "k is v", "head dim"])
def test_layout_refusals(dph_native, part):
    ops = _ops()
    c = ops.kv8_cache(2, 40, 2, 32, block=16, device=DEV)
    cos, sin = tables(32, 40, DEV)
    qkv, pos = make_qkv(2, 1, 4, 2, 32, 0, DEV), _pos(3, 5).to(DEV)
    if part == "strides":
        k, v = (torch.zeros(2, 40, 2, 40, dtype=torch.int8, device=DEV)[..., :32] for _ in range(2))
        c = c._replace(k=k, v=v)
    elif part == "alignment":
        c = c._replace(k=torch.zeros(2 * 40 * 2 * 32 + 8, dtype=torch.int8, device=DEV)[8:].view(2, 40, 2, 32),
                       v=torch.zeros(2, 40, 2, 32, dtype=torch.int8, device=DEV))
    elif part == "last dim":
        qkv = torch.zeros(2, 1, 2 * 8 * 32, dtype=torch.bfloat16, device=DEV)[..., ::2]
    elif part == "devices":
        c = c._replace(k_scale=c.k_scale.cpu())
    elif part == "overlap":
        c = c._replace(k=torch.zeros(40, 2, 32, dtype=torch.int8, device=DEV).expand(2, -1, -1, -1),
                       v=torch.zeros(40, 2, 32, dtype=torch.int8, device=DEV).expand(2, -1, -1, -1))
    elif part == "k is v":
        c = c._replace(v=c.k)
    else:
        c = ops.kv8_cache(2, 40, 2, 16, block=16, device=DEV)
        qkv, (cos, sin) = make_qkv(2, 1, 4, 2, 16, 0, DEV), tables(16, 40, DEV)
    with pytest.raises(RuntimeError):
        ops.kv8_append_(qkv, c, pos, cos, sin, 4, 2)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d,t", [(4, 4, 32, 16), (12, 4, 64, 32), (8, 1, 128, 64), (2, 2, 128, 128),
                                        (5, 5, 64, 16), (6, 3, 32, 128)])
@pytest.mark.parametrize("s", [1, 2, 17, 150])
def test_append_bitwise(dph_native, code, hq, hkv, d, t, s):
    """Ragged positions at and around block borders, capacities that no block divides: every stored bit, the rotated q
    and k, and nothing else is written."""
    ops = _ops()
    cap = 2 * t + s + 13
    pos = _pos(0, t - 1, t, 2 * t - min(s, t), 2 * t + 13)
    ref = filled(ops.kv8_cache(5, cap, hkv, d, code, t), 7)
    got = _to(ref, DEV)
    assert got.k.stride() == ref.k.stride()
    qkv = make_qkv(5, s, hq, hkv, d, 11, "cpu")
    gqkv = qkv.to(DEV)
    cos, sin = tables(d, cap, "cpu")
    ops.kv8_append_(qkv, ref, pos, cos, sin, hq, hkv)
    ops.kv8_append_(gqkv, got, pos.to(DEV), cos.to(DEV), sin.to(DEV), hq, hkv)
    _equal(gqkv, qkv)
    _same(got, ref)


@pytest.mark.parametrize("hkv,d,t", [(8, 32, 16), (4, 64, 16), (8, 32, 32), (2, 32, 64)])
def test_append_bitwise_many_small_blocks(dph_native, hkv, d, t):
    """Blocks of fewer chunks than a workgroup has threads: the spare threads, which read a chunk that its owner rotates in
    place meanwhile, have no part in the scale."""
    ops = _ops()
    s, cap = 900, 960
    qkv = make_qkv(6, s, hkv, hkv, d, 12, "cpu")
    ref = ops.kv8_cache(6, cap, hkv, d, block=t)
    got, x = _to(ref, DEV), qkv.to(DEV)
    cos, sin = tables(d, cap, "cpu")
    pos = _pos(0, 1, 15, 16, 40, 60)
    ops.kv8_append_(qkv, ref, pos, cos, sin, hkv, hkv)
    ops.kv8_append_(x, got, pos.to(DEV), cos.to(DEV), sin.to(DEV), hkv, hkv)
    _equal(x, qkv)
    _same(got, ref)


@pytest.mark.parametrize("code", CODES)
def test_append_values_at_the_edges(dph_native, code):
    """Blocks of zeros, of the least and the largest bf16 numbers, and with infinities or NaN."""
    ops = _ops()
    hq, hkv, d, t = 2, 2, 64, 16
    x = make_qkv(1, 6 * t, hq, hkv, d, 5, "cpu")
    v = x.view(1, 6, t, hq + 2 * hkv, d)[:, :, :, hq + hkv:]
    v[:, 0] = 0
    v[:, 1] *= 1e-38
    v[:, 2] *= 2.0 ** 125
    v[:, 3, 2, 0, 7] = float("inf")
    v[:, 4, 3, 1, 9] = float("nan")
    cos, sin = tables(d, 6 * t, "cpu")
    ref = ops.kv8_cache(1, 6 * t, hkv, d, code, t)
    got, gx = _to(ref, DEV), x.to(DEV)
    ops.kv8_append_(x, ref, _pos(0), cos, sin, hq, hkv)
    ops.kv8_append_(gx, got, _pos(0).to(DEV), cos.to(DEV), sin.to(DEV), hq, hkv)
    for a, b in zip(got, ref):
        a = a.cpu()
        if a.dtype == torch.float32:
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
        else:
            _equal(a, b)
    assert got.v_scale[0, 3, 0].isnan() and not got.v_scale[0, 3, 1].isnan() and got.v_scale[0, 4, 1].isnan()
    k, v = ops.kv8_read(got, _pos(6 * t).to(DEV), 6 * t)
    assert v[0, 3 * t:4 * t, 0].isnan().all() and torch.isfinite(v[0, :3 * t]).all() and torch.isfinite(k).all()


def test_append_past_the_capacity_is_dropped(dph_native):
    """A replayed graph may run past the end: tokens from Smax on, and sequences at negative positions, write nothing."""
    ops = _ops()
    hq, hkv, d, t, cap = 2, 2, 32, 16, 40
    c = filled(ops.kv8_cache(4, cap, hkv, d, block=t), 3)
    got = _to(c, DEV)
    qkv = make_qkv(4, 5, hq, hkv, d, 1, DEV)
    before = qkv.clone()
    cos, sin = tables(d, cap, DEV)
    ops.kv8_append_(qkv, got, _pos(38, 40, 2 ** 31 - 3, -7).to(DEV), cos, sin, hq, hkv)
    want, ref = before[:1, :2].cpu(), c.slot(0)
    ops.kv8_append_(want, ref, _pos(38), cos.cpu(), sin.cpu(), hq, hkv)
    _same(got, c)
    assert torch.equal(qkv[:1, :2].cpu(), want) and torch.equal(qkv[:1, 2:], before[:1, 2:])
    assert torch.equal(qkv[1:], before[1:])


DECODE = [(4, 4, 32, 16), (12, 4, 64, 32), (8, 1, 128, 64), (3, 3, 128, 128), (40, 2, 64, 16), (32, 1, 128, 32)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d,t", DECODE)
def test_decode_attention(dph_native, code, hq, hkv, d, t):
    """Lengths of one token, of a block and one more or less, of an odd capacity, and none; rows behind each sequence's
    end hold NaN, which must not be read into the output."""
    ops = _ops()
    cap = 333
    pos = _pos(0, t - 2, t - 1, t, 200, cap - 1, -1).to(DEV)
    c = _to(filled(ops.kv8_cache(7, cap, hkv, d, code, t), 5), DEV)
    for b, p in enumerate(pos.tolist()):
        n = p + 1
        for scale, tail in ((c.k_scale, c.k_tail), (c.v_scale, c.v_tail)):
            scale[b, n // t:] = float("nan")
            tail[b, n % t:] = float("nan")
    qkv = 2 * make_qkv(7, 1, hq, hkv, d, 6, DEV)
    want, off = attention64(qkv, c, pos, hq, hkv, d ** -0.5)
    for bound in (None, cap):
        got = ops.kv8_decode_attention(qkv, c, pos, hq, hkv, max_len=bound)
        assert got.shape == (7, hq * d) and (got[6] == 0).all()
        assert_close64(got, want, off)


@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0])
def test_decode_attention_scale_and_tight_bound(dph_native, scale):
    ops = _ops()
    c = _to(filled(ops.kv8_cache(3, 900, 2, 64, block=32), 8), DEV)
    pos = _pos(30, 31, 470).to(DEV)
    qkv = make_qkv(3, 1, 6, 2, 64, 9, DEV)
    want, off = attention64(qkv, c, pos, 6, 2, scale)
    for bound in (471, 900):
        assert_close64(ops.kv8_decode_attention(qkv, c, pos, 6, 2, scale=scale, max_len=bound), want, off)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("batch,n", [(1, 5000), (1, 16384), (3, 2999)])
def test_decode_attention_long(dph_native, code, batch, n):
    """Lengths that are split over many workgroups; one key far above the others late in the sequence."""
    ops = _ops()
    hq, hkv, d, t = 8, 2, 128, 64
    c = _to(filled(ops.kv8_cache(batch, n, hkv, d, code, t), 12), DEV)
    pos = torch.tensor([n - 1 - 700 * b for b in range(batch)], dtype=torch.int32, device=DEV)
    c.k_scale[:, n // t - 20] *= 6
    c.v_scale[:, 3] *= 1e-6
    qkv = 3 * make_qkv(batch, 1, hq, hkv, d, 13, DEV)
    want, off = [], []
    for b in range(batch):   # dequantised rows, vectorised: the oracle's loop over rows is for the short tests
        m = int(pos[b]) + 1
        f = m // t
        kv = [torch.cat([x[b, :f * t].double() * s[b, :f].double().repeat_interleave(t, 0)[..., None],
                         y[b, :m % t].double()])
              for x, s, y in ((c.k, c.k_scale, c.k_tail), (c.v, c.v_scale, c.v_tail))]
        k, v = (x.transpose(0, 1) for x in kv)
        q = qkv[b, 0, :hq * d].double().view(hkv, hq // hkv, d)
        s = (q @ k.transpose(1, 2)) * d ** -0.5
        mag = (q.abs() @ k.abs().transpose(1, 2)) * d ** -0.5
        w = torch.softmax(s, -1)
        ds = (d + 4) * 2.0 ** -24 * mag
        dw = w * ds + w * (w * ds).sum(-1, keepdim=True) + w * (2.0 ** -22 + 2.0 ** -16 + 96 * 2.0 ** -24)
        want.append((w @ v).reshape(-1))
        off.append((dw @ v.abs()).reshape(-1))
    got = ops.kv8_decode_attention(qkv, c, pos, hq, hkv)
    assert_close64(got, torch.stack(want), torch.stack(off))
    again = ops.kv8_decode_attention(qkv, c, pos, hq, hkv)
    assert torch.equal(got, again)


def test_decode_attention_non_finite(dph_native):
    """A block with a scale of NaN makes every head that reads it NaN, others and other sequences stay clean; queries of
    infinity give NaN."""
    ops = _ops()
    hq, hkv, d, t = 4, 2, 64, 16
    c = _to(filled(ops.kv8_cache(3, 100, hkv, d, block=t), 2), DEV)
    pos = _pos(99, 99, 99).to(DEV)
    qkv = make_qkv(3, 1, hq, hkv, d, 3, DEV)
    clean = ops.kv8_decode_attention(qkv, c, pos, hq, hkv).view(3, hq, d)
    c.k_scale[0, 2, 0] = float("nan")
    c.v_scale[1, 3, 1] = float("nan")
    qkv[2, 0, 0] = float("inf")
    got = ops.kv8_decode_attention(qkv, c, pos, hq, hkv).view(3, hq, d)
    assert got[0, :2].isnan().all() and torch.equal(got[0, 2:], clean[0, 2:])
    assert got[1, 2:].isnan().all() and torch.equal(got[1, :2], clean[1, :2])
    assert got[2, 0].isnan().all() and torch.equal(got[2, 1:], clean[2, 1:])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hkv,d,t", [(4, 32, 16), (3, 64, 32), (1, 128, 64), (2, 128, 128)])
@pytest.mark.parametrize("count", [0, 1, 33, 300])
def test_read(dph_native, code, hkv, d, t, count):
    """Bits of the reference, zeros before the first token; an ``out`` view is written and its surroundings are not."""
    ops = _ops()
    ref = filled(ops.kv8_cache(4, 300, hkv, d, code, t), 4)
    got, pos = _to(ref, DEV), _pos(0, 5, 2 * t, 299)
    want = ops.kv8_read(ref, pos, count)
    for a, b in zip(ops.kv8_read(got, pos.to(DEV), count), want):
        _equal(a, b)
    room = [torch.full((4, count + 9, hkv + 2, d), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    view = tuple(r[:, 4:4 + count, 1:1 + hkv] for r in room)
    ops.kv8_read(got, pos.to(DEV), count, view)
    for r, a, b in zip(room, view, want):
        assert torch.equal(a.cpu(), b)
        a.fill_(7.0)
        assert (r == 7.0).all()


@pytest.mark.parametrize("layout", ["rows first", "interleaved", "padded", "qkv view"])
def test_layouts(dph_native, layout):
    """Caches and qkv whose strides are not those of kv8_cache."""
    ops = _ops()
    hq, hkv, d, t, cap, s = 6, 2, 64, 16, 50, 20
    base = filled(ops.kv8_cache(2, cap, hkv, d, block=t), 9)
    qkv = make_qkv(2, s, hq, hkv, d, 10, "cpu")
    x = qkv.to(DEV)
    if layout == "rows first":
        c = base._replace(**{n: v.contiguous().to(DEV) for n, v in zip(base._fields, base)})
    elif layout == "interleaved":   # keys and values next to each other in one buffer
        both = torch.stack([base.k, base.v], 3).to(DEV)
        sc = torch.stack([base.k_scale, base.v_scale], 3).to(DEV)
        c = _to(base, DEV)._replace(k=both[:, :, :, 0], v=both[:, :, :, 1], k_scale=sc[..., 0], v_scale=sc[..., 1])
    elif layout == "padded":
        def pad(v):
            r = torch.zeros(3, v.shape[1] + 1, v.shape[2] + 1, v.shape[3] + 16, dtype=v.dtype, device=DEV)
            r = r[1:, 1:, 1:, 16:]
            r.copy_(v)
            return r
        c = _to(base, DEV)._replace(k=pad(base.k), v=pad(base.v), k_tail=pad(base.k_tail), v_tail=pad(base.v_tail))
    else:
        c = _to(base, DEV)
        x = torch.zeros(2, s + 3, qkv.shape[2] + 8, dtype=torch.bfloat16, device=DEV)[:, 2:-1, 8:]
        x.copy_(qkv)
    cos, sin = tables(d, cap, "cpu")
    pos = _pos(3, 28)
    ops.kv8_append_(qkv, base, pos, cos, sin, hq, hkv)
    ops.kv8_append_(x, c, pos.to(DEV), cos.to(DEV), sin.to(DEV), hq, hkv)
    assert torch.equal(x.cpu(), qkv)
    _same(c, base)
    pos = _pos(22, 47)
    one = x[:, -1:]
    want, off = attention64(one.cpu(), base, pos, hq, hkv, d ** -0.5)
    assert_close64(ops.kv8_decode_attention(one, c, pos.to(DEV), hq, hkv).cpu(), want, off)
    for a, b in zip(ops.kv8_read(c, pos.to(DEV) + 1, 31), ops.kv8_read(base, pos + 1, 31)):
        assert torch.equal(a.cpu(), b)


def _step(ops, qkv, c, pos, cos, sin, hq, hkv):
    ops.kv8_append_(qkv, c, pos, cos, sin, hq, hkv)
    o = ops.kv8_decode_attention(qkv, c, pos, hq, hkv)
    pos += 1
    return o


def test_graph_replays_with_the_cache_advancing(dph_native):
    """A captured append + attention step, replayed across two block borders with eager work in between, equals eager
    steps bit for bit; a second graph over another cache shares no state with it."""
    ops = _ops()
    hq, hkv, d, t, cap = 8, 2, 64, 16, 64
    cos, sin = tables(d, cap, DEV)
    caches = [_to(filled(ops.kv8_cache(3, cap, hkv, d, block=t), 20 + i), DEV) for i in range(2)]
    eager = [type(c)(*(x.clone(memory_format=torch.preserve_format) for x in c)) for c in caches]
    start = [_pos(0, 14, 30).to(DEV), _pos(5, 31, 2).to(DEV)]
    pos, epos = [p.clone() for p in start], [p.clone() for p in start]
    bufs = [torch.zeros(3, 1, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    graphs, outs = [], []
    for i in range(2):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):   # warm-up on clones
            w = type(caches[i])(*(x.clone() for x in caches[i]))
            _step(ops, bufs[i].clone(), w, pos[i].clone(), cos, sin, hq, hkv)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(ops, bufs[i], caches[i], pos[i], cos, sin, hq, hkv))
        graphs.append(g)
    for k in range(33):
        x = [make_qkv(3, 1, hq, hkv, d, 100 + 2 * k + i, DEV) for i in range(2)]
        for i in range(2):
            bufs[i].copy_(x[i])
            graphs[i].replay()
        if k % 5 == 0:
            torch.cuda.synchronize()
        for i in range(2):
            want = _step(ops, x[i], eager[i], epos[i], cos, sin, hq, hkv)
            assert torch.equal(outs[i], want), (k, i)
            assert torch.equal(bufs[i], x[i])
    for i in range(2):
        _same(caches[i], eager[i])


def test_two_streams(dph_native):
    """Steps on a side stream and on the current one at once, each with its own cache."""
    ops = _ops()
    hq, hkv, d, t, cap = 8, 8, 128, 64, 2048
    cos, sin = tables(d, cap, DEV)
    c = [_to(filled(ops.kv8_cache(2, cap, hkv, d, block=t), 30 + i), DEV) for i in range(2)]
    pos = [_pos(1999, 700).to(DEV), _pos(63, 1407).to(DEV)]
    x = [make_qkv(2, 1, hq, hkv, d, 40 + i, DEV) for i in range(2)]
    want = []
    for i in range(2):
        w = type(c[i])(*(y.clone(memory_format=torch.preserve_format) for y in c[i]))
        want.append(_step(ops, x[i].clone(), w, pos[i].clone(), cos, sin, hq, hkv))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = _step(ops, x[0], c[0], pos[0], cos, sin, hq, hkv)
    b = _step(ops, x[1], c[1], pos[1], cos, sin, hq, hkv)
    torch.cuda.synchronize()
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_offsets_past_32_bits(dph_native):
    """A cache whose last sequences lie more than 2^32 bytes behind its start."""
    ops = _ops()
    hq, hkv, d, t, cap, batch = 2, 2, 128, 64, 32768, 520
    cos, sin = tables(d, cap, DEV)
    c = ops.kv8_cache(batch, cap, hkv, d, block=t, device=DEV)   # 4.4 GB of codes each
    assert c.k.numel() > 2 ** 32
    pos = torch.zeros(batch, dtype=torch.int32, device=DEV)
    pos[-1] = cap - 100
    qkv = make_qkv(1, 100, hq, hkv, d, 50, DEV).expand(batch, -1, -1).contiguous()
    ops.kv8_append_(qkv, c, pos, cos, sin, hq, hkv)
    ref = ops.kv8_cache(1, cap, hkv, d, block=t)
    x = make_qkv(1, 100, hq, hkv, d, 50, "cpu")
    ops.kv8_append_(x, ref, _pos(cap - 100), cos.cpu(), sin.cpu(), hq, hkv)
    _same(c.slot(batch - 1), ref)
    pos += 99
    one = qkv[:, -1:].contiguous()
    got = ops.kv8_decode_attention(one, c, pos, hq, hkv)
    small = type(c)(*(y[-1:].clone(memory_format=torch.preserve_format) for y in c))
    assert torch.equal(got[-1:], ops.kv8_decode_attention(one[-1:], small, pos[-1:].clone(), hq, hkv))
    k, v = ops.kv8_read(c.slot(batch - 1), pos[-1:].clone() + 1, 120)
    assert torch.equal(v[0, -100:].cpu(), ops.kv8_read(ref, _pos(cap), 100)[1][0])


def test_read_refuses_outputs_over_the_cache(dph_native):
    ops = _ops()
    c = ops.kv8_cache(2, 40, 2, 32, block=16, device=DEV)
    pos = _pos(3, 5).to(DEV)
    a = torch.zeros(2, 4, 2, 32, dtype=torch.bfloat16, device=DEV)
    for out in ((a, a), (c.k_tail[:, :4], a), (a, a.clone()[:1].expand(2, -1, -1, -1))):
        with pytest.raises(RuntimeError):
            ops.kv8_read(c, pos, 4, out)


def test_no_sequences_and_no_tokens(dph_native):
    ops = _ops()
    cos, sin = tables(32, 40, DEV)
    c = ops.kv8_cache(0, 40, 2, 32, block=16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    ops.kv8_append_(torch.zeros(0, 3, 256, dtype=torch.bfloat16, device=DEV), c, none, cos, sin, 4, 2)
    one = torch.zeros(0, 1, 256, dtype=torch.bfloat16, device=DEV)
    assert ops.kv8_decode_attention(one, c, none, 4, 2).shape == (0, 128)
    assert ops.kv8_read(c, none, 7)[1].shape == (0, 7, 2, 32)
    c = _to(filled(ops.kv8_cache(2, 40, 2, 32, block=16), 1), DEV)
    before = type(c)(*(t.clone() for t in c))
    ops.kv8_append_(torch.zeros(2, 0, 256, dtype=torch.bfloat16, device=DEV), c, _pos(3, 5).to(DEV), cos, sin, 4, 2)
    _same(c, before)


@pytest.mark.parametrize("batch", [63, 64, 65, 130])
def test_decode_attention_many_sequences(dph_native, batch):
    """Lengths from none to the capacity, more sequences than lanes: every one equals itself in a batch of one, up to how
    its sum is divided (compared with the oracle)."""
    ops = _ops()
    hq, hkv, d, t, cap = 4, 2, 32, 16, 700
    c = _to(filled(ops.kv8_cache(batch, cap, hkv, d, block=t), 15), DEV)
    pos = (torch.arange(batch) * 37 % (cap + 1) - 1).int()
    qkv = make_qkv(batch, 1, hq, hkv, d, 16, DEV)
    got = ops.kv8_decode_attention(qkv, c, pos.to(DEV), hq, hkv)
    some = [0, 1, batch // 2, batch - 2, batch - 1]
    small = type(c)(*(x[some] for x in c))
    want, off = attention64(qkv[some], small, pos[some], hq, hkv, d ** -0.5)
    assert_close64(got[some], want, off)
    for i in range(batch):   # the kernel's own sums of one sequence, one rounding of each side apart
        alone = ops.kv8_decode_attention(qkv[i:i + 1], c.slot(i), pos[i:i + 1].to(DEV), hq, hkv)
        torch.testing.assert_close(got[i:i + 1].float(), alone.float(), rtol=2 * 2.0 ** -8, atol=2.0 ** -12)


@pytest.mark.parametrize("max_len", [1, 100, 128, 129, 333])
def test_decode_attention_max_len_only_splits_the_work(dph_native, max_len):
    """A bound that is too low, too high or right gives the same attention."""
    ops = _ops()
    c = _to(filled(ops.kv8_cache(4, 333, 2, 64, block=32), 18), DEV)
    pos = _pos(-1, 40, 128, 332).to(DEV)
    qkv = make_qkv(4, 1, 6, 2, 64, 19, DEV)
    want, off = attention64(qkv, c, pos, 6, 2, 0.125)
    assert_close64(ops.kv8_decode_attention(qkv, c, pos, 6, 2, scale=0.125, max_len=max_len), want, off)


def test_decode_attention_past_the_capacity(dph_native):
    """Positions at and past Smax (a replayed graph run too far) see the rows that exist."""
    ops = _ops()
    c = _to(filled(ops.kv8_cache(3, 70, 2, 64, block=32), 21), DEV)
    pos = _pos(69, 70, 2 ** 31 - 1).to(DEV)
    qkv = make_qkv(1, 1, 4, 2, 64, 22, DEV).expand(3, -1, -1)
    same = type(c)(*(x[:1].expand_as(x).contiguous() for x in c))
    got = ops.kv8_decode_attention(qkv, same, pos, 4, 2)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    for a, b in zip(ops.kv8_read(same, pos + torch.tensor([1, 0, 0], device=DEV, dtype=torch.int32), 30), range(2)):
        assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


def test_decode_attention_scales_far_apart(dph_native):
    """One block of V 2^-40 of the others' size with all of the weight on it: its digits are not lost."""
    ops = _ops()
    hq, hkv, d, t, n = 2, 2, 128, 16, 600
    c = _to(filled(ops.kv8_cache(1, n, hkv, d, block=t), 23), DEV)
    c.v_scale[:, 20] *= 2.0 ** -40
    c.k_scale[:, :20] *= 1e-3
    c.k_scale[:, 21:] *= 1e-3
    c.k[:, 20 * t:21 * t] = 64
    c.k_scale[:, 20] = 1.0
    c.k_tail.mul_(1e-3)
    qkv = make_qkv(1, 1, hq, hkv, d, 24, DEV)
    qkv[:, :, :hq * d] = 1.0
    pos = _pos(n - 1).to(DEV)
    want, off = attention64(qkv, c, pos, hq, hkv, d ** -0.5)
    got = ops.kv8_decode_attention(qkv, c, pos, hq, hkv)
    assert float(want.abs().max()) < 2.0 ** -36
    assert_close64(got, want, off)
