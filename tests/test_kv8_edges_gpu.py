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
