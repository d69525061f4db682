"""Calls that the 8-bit KV cache and the logit operators refuse, each a function of a device: run on the CPU by
test_kv8.py and on the GPU by test_kv8_gpu.py."""
import torch

from kv8_oracle import make_qkv, tables


def _case(dev, **over):
    from distributed_pytorch_hpc_amd import ops

    hq, hkv, d = 4, 2, 32
    cache = ops.kv8_cache(2, 40, hkv, d, block=16, device=dev)._replace(**over.pop("parts", {}))
    cos, sin = tables(d, 40, dev)
    a = dict(qkv=make_qkv(2, 1, hq, hkv, d, 0, dev), cache=cache,
             pos=torch.tensor([3, 5], dtype=torch.int32, device=dev), cos=cos, sin=sin, n_heads=hq, n_kv_heads=hkv)
    a.update(over)
    return a


def _append(dev, **over):
    from distributed_pytorch_hpc_amd import ops

    ops.kv8_append_(**_case(dev, **over))


def _decode(dev, max_len=None, **over):
    from distributed_pytorch_hpc_amd import ops

    a = _case(dev, **over)
    ops.kv8_decode_attention(a["qkv"], a["cache"], a["pos"], a["n_heads"], a["n_kv_heads"], max_len=max_len)


def _read(dev, count, out=None, **over):
    from distributed_pytorch_hpc_amd import ops

    a = _case(dev, **over)
    ops.kv8_read(a["cache"], a["pos"], count, out)


def _logits(dev, n=3, v=50, **over):
    from distributed_pytorch_hpc_amd import ops

    a = dict(logits=torch.zeros(n, v, device=dev), tokens=torch.zeros(n, 4, dtype=torch.int64, device=dev),
             lengths=torch.full((n,), 4, dtype=torch.int32, device=dev), repetition=torch.ones(n, device=dev))
    a.update(over)
    ops.process_logits(**{k: t for k, t in a.items() if t is not None})


def _t(dev, *shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device=dev)


BF, I8 = torch.bfloat16, torch.int8
REFUSED = {
    "append_grad": lambda d: _append(d, qkv=make_qkv(2, 1, 4, 2, 32, 0, d).requires_grad_()),
    "append_heads": lambda d: _append(d, n_heads=3),
    "append_kv_heads": lambda d: _append(d, n_kv_heads=1),
    "append_width": lambda d: _append(d, qkv=_t(d, 2, 1, 8 * 32 - 8, dtype=BF)),
    "append_batch": lambda d: _append(d, qkv=_t(d, 3, 1, 8 * 32, dtype=BF)),
    "append_pos_type": lambda d: _append(d, pos=torch.zeros(2, dtype=torch.int64, device=d)),
    "append_pos_size": lambda d: _append(d, pos=torch.zeros(3, dtype=torch.int32, device=d)),
    "append_short_table": lambda d: _append(d, cos=_t(d, 39, 16), sin=_t(d, 39, 16)),
    "append_table_width": lambda d: _append(d, cos=_t(d, 40, 32), sin=_t(d, 40, 32)),
    "append_too_many": lambda d: _append(d, qkv=_t(d, 2, 41, 8 * 32, dtype=BF)),
    "cache_code_type": lambda d: _append(d, parts=dict(k=_t(d, 2, 40, 2, 32, dtype=BF))),
    "cache_mixed_types": lambda d: _decode(d, parts=dict(v=_t(d, 2, 40, 2, 32, dtype=torch.float8_e4m3fn))),
    "cache_scale_type": lambda d: _decode(d, parts=dict(k_scale=_t(d, 2, 2, 2, dtype=BF))),
    "cache_scale_blocks": lambda d: _decode(d, parts=dict(k_scale=_t(d, 2, 3, 2), v_scale=_t(d, 2, 3, 2))),
    "cache_tail_block": lambda d: _decode(d, parts=dict(k_tail=_t(d, 2, 20, 2, 32, dtype=BF),
                                                        v_tail=_t(d, 2, 20, 2, 32, dtype=BF))),
    "cache_tail_type": lambda d: _read(d, 4, parts=dict(k_tail=_t(d, 2, 16, 2, 32), v_tail=_t(d, 2, 16, 2, 32))),
    "decode_grad": lambda d: _decode(d, qkv=make_qkv(2, 1, 4, 2, 32, 0, d).requires_grad_()),
    "decode_two_tokens": lambda d: _decode(d, qkv=_t(d, 2, 2, 8 * 32, dtype=BF)),
    "decode_max_len_0": lambda d: _decode(d, max_len=0),
    "decode_max_len_big": lambda d: _decode(d, max_len=41),
    "read_negative": lambda d: _read(d, -1),
    "read_too_many": lambda d: _read(d, 41),
    "read_out_shape": lambda d: _read(d, 4, out=(_t(d, 2, 5, 2, 32, dtype=BF), _t(d, 2, 5, 2, 32, dtype=BF))),
    "logits_grad": lambda d: _logits(d, logits=torch.zeros(3, 50, device=d, requires_grad=True)),
    "logits_type": lambda d: _logits(d, logits=_t(d, 3, 50, dtype=torch.float64)),
    "logits_shape": lambda d: _logits(d, logits=_t(d, 1, 3, 50)),
    "logits_no_tokens": lambda d: _logits(d, tokens=None),
    "logits_no_lengths": lambda d: _logits(d, lengths=None),
    "logits_token_type": lambda d: _logits(d, tokens=_t(d, 3, 4, dtype=torch.int32)),
    "logits_token_rows": lambda d: _logits(d, tokens=_t(d, 2, 4, dtype=torch.int64)),
    "logits_length_type": lambda d: _logits(d, lengths=_t(d, 3, dtype=torch.int64)),
    "logits_penalty_size": lambda d: _logits(d, presence=_t(d, 2)),
    "logits_bias_size": lambda d: _logits(d, bias=_t(d, 49)),
    "logits_bias_type": lambda d: _logits(d, bias=_t(d, 50, dtype=BF)),
    "logits_mask_words": lambda d: _logits(d, mask=_t(d, 3, 1, dtype=torch.int32)),
    "logits_mask_type": lambda d: _logits(d, mask=_t(d, 3, 2, dtype=torch.int64)),
}
