"""Calls of the 8-bit KV cache and logit operators with one operand that requires grad, each a function of a device: none
has a backward, so every one is refused where a graph is recorded (test_kv8_grads.py, test_kv8_grads_gpu.py)."""
import torch

from kv8_oracle import make_qkv, tables

PENALTIES = ("repetition", "presence", "frequency")


def kv8_call(op, dev, need=None):
    from distributed_pytorch_hpc_amd import ops

    hq, hkv, d = 4, 2, 32
    cos, sin = tables(d, 40, dev)
    cache = ops.kv8_cache(2, 40, hkv, d, block=16, device=dev)
    out = tuple(torch.zeros(2, 5, hkv, d, dtype=torch.bfloat16, device=dev) for _ in range(2))
    named = dict(cache._asdict(), qkv=make_qkv(2, 1, hq, hkv, d, 0, dev), cos=cos, sin=sin, out0=out[0], out1=out[1])
    if need is not None:
        named[need].requires_grad_()
    pos = torch.tensor([3, 5], dtype=torch.int32, device=dev)
    if op == "append":
        return ops.kv8_append_(named["qkv"], cache, pos, cos, sin, hq, hkv)
    if op == "decode":
        return ops.kv8_decode_attention(named["qkv"], cache, pos, hq, hkv)
    return ops.kv8_read(cache, pos, 5, out if op == "read_into" else None)


def logits_call(dev, need=None):
    from distributed_pytorch_hpc_amd import ops

    a = dict(logits=torch.zeros(3, 50, device=dev), bias=torch.zeros(50, device=dev),
             **{k: torch.ones(3, device=dev) for k in PENALTIES})
    if need is not None:
        a[need].requires_grad_()
    return ops.process_logits(tokens=torch.zeros(3, 4, dtype=torch.int64, device=dev),
                              lengths=torch.full((3,), 4, dtype=torch.int32, device=dev), **a)


PARTS = ("k_scale", "v_scale", "k_tail", "v_tail")
CASES = [("append", n) for n in ("qkv", *PARTS, "cos", "sin")] + [("decode", n) for n in ("qkv", *PARTS)] + \
    [("read", n) for n in PARTS] + [("read_into", n) for n in (*PARTS, "out0", "out1")] + \
    [("logits", n) for n in ("logits", "bias", *PENALTIES)]


def call(op, dev, need=None):
    return logits_call(dev, need) if op == "logits" else kv8_call(op, dev, need)
