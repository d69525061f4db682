"""The 8-bit KV cache and the logit controls at the edges of their values and sizes, on the CPU."""
import pytest
import torch

from kv8_oracle import assert_close64_inf, attention64, filled, infinities, make_qkv

CODES = [torch.int8, torch.float8_e4m3fn]


def _ops():
    from distributed_pytorch_hpc_amd import ops

    return ops


@pytest.mark.parametrize("code", CODES)
def test_decode_reference_with_infinities_in_the_open_block(code):
    ops = _ops()
    cache = infinities(filled(ops.kv8_cache(4, 75, 2, 64, code, 32), 1), [1, 33, 50, 75])
    pos = torch.tensor([0, 32, 49, 74], dtype=torch.int32)
    qkv = make_qkv(4, 1, 8, 2, 64, 2, "cpu")
    want, off = attention64(qkv, cache, pos, 8, 2, 0.125)
    assert torch.isinf(want).any() and want.isnan().any()
    assert_close64_inf(ops.kv8_decode_attention(qkv, cache, pos, 8, 2), want, off)


def test_a_refused_append_leaves_everything_as_it_was():
    """The second sequence has no room: the first one's open block is not quantised away under its unchanged position."""
    from kv8_oracle import tables

    ops = _ops()
    cos, sin = tables(32, 40, "cpu")
    cache, x = filled(ops.kv8_cache(2, 40, 2, 32, block=16), 1), make_qkv(2, 3, 4, 2, 32, 0, "cpu")
    before = [t.clone() for t in (*cache, x)]
    for pos in ([14, 38], [14, -1]):
        with pytest.raises(ValueError, match="overflow"):
            ops.kv8_append_(x, cache, torch.tensor(pos, dtype=torch.int32), cos, sin, 4, 2)
        assert all(torch.equal(a.float(), b.float()) for a, b in zip((*cache, x), before))
