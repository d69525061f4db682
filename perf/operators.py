"""Serving operators of the Llama decoder and what each has to compute: the block-scaled 8-bit KV cache (append, decode
attention, read-back) and the control of logits before sampling.

``own`` False computes them with elementary torch operations, True through ``distributed_pytorch_hpc_amd.ops``.

An 8-bit cache of a layer holds, for sequences of pos[b] tokens and blocks of T tokens,
  k, v               [B, Smax, Hkv, D]    codes (int8 or e4m3) of the blocks that are full
  k_scale, v_scale   [B, Smax // T, Hkv]  fp32, value = code * scale
  k_tail, v_tail     [B, T, Hkv, D]       bf16 rows of the block that is still open (row t % T)
with scale = max(amax / QMAX, 2^-126) over the T x D entries of a block and KV head, code = round(x * (1 / scale)).
"""
import math

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TINY = 2.0 ** -126
DEV = "cuda"
STATE = ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")

# (query heads, KV heads, head dim): the decoder's presets, a grouped 64-wide form and the small test model
HEADS = {"7b": (32, 32, 128), "70b": (64, 8, 128), "1b": (16, 16, 128), "13b": (40, 40, 128), "gqa64": (12, 4, 64),
         "tiny": (4, 4, 32), "mqa": (8, 1, 128)}


# ------------------------------------------------------------------------------------------------------- cases
def _kv(op, name, batch, heads, block, code, cap, lo, hi, new=0):
    hq, hkv, d = HEADS[heads]
    return {"name": name, "op": op, "batch": batch, "hq": hq, "hkv": hkv, "d": d, "block": block, "code": code,
            "cap": cap, "lo": lo, "hi": hi, "new": new}


def _logits(name, rows, vocab, dtype, length, penalties, bias, mask):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "dtype": dtype, "len": length,
            "penalties": penalties, "bias": bias, "mask": mask}


def listed():
    return [
        # one decode step's append in the middle of generation: 16 sequences, a few of them filling their block
        _kv("append", "append_step_7b_b16", 16, "7b", 64, "int8", 4096, 200, 3900, 1),
        # a speculative or chunked continuation of ragged sequences
        _kv("append", "append_chunk_70b_b4", 4, "70b", 32, "e4m3", 4096, 0, 2500, 333),
        # the prefill of one long prompt
        _kv("append", "append_prompt_7b", 1, "7b", 64, "int8", 4608, 0, 0, 4096),
        # first tokens of a small model: latency only
        _kv("decode", "decode_tiny_b2", 2, "tiny", 16, "int8", 512, 5, 60),
        # one user, a middling context
        _kv("decode", "decode_7b_b1", 1, "7b", 64, "int8", 4096, 2345, 2345),
        # a served batch at ragged lengths
        _kv("decode", "decode_7b_b16", 16, "7b", 64, "int8", 4096, 1000, 4000),
        # grouped heads, a large batch at long context: the largest read
        _kv("decode", "decode_70b_b32", 32, "70b", 32, "e4m3", 8192, 4000, 8100),
        # one very long sequence: only the split over its length fills the card
        _kv("decode", "decode_70b_long", 1, "70b", 128, "int8", 32768, 32001, 32001),
        # the prefix of a chunked prefill
        _kv("read", "read_prefix_7b", 1, "7b", 64, "int8", 4096, 3500, 3500),
        # the last tokens of ragged sequences of grouped 64-wide heads
        _kv("read", "read_window_gqa64_b8", 8, "gqa64", 16, "e4m3", 2048, 40, 2000, 512),
        # one user's penalties over a short history
        _logits("logits_b1", 1, 32000, "float32", 300, True, False, False),
        # a served batch with long histories, biases and a grammar
        _logits("logits_b64", 64, 32000, "bfloat16", 4000, True, True, True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "read", "logits"])
    if op == "logits":
        rows = _log(rng, 1, 64)
        return {"op": op, "rows": rows, "vocab": _log(rng, 500, 131072 if rows < 16 else 33000),
                "dtype": rng.choice(["float32", "bfloat16"]), "len": _log(rng, 1, 4096),
                "penalties": True, "bias": rng.random() < 0.5, "mask": rng.random() < 0.5}
    hq, hkv, d = HEADS[rng.choice(sorted(HEADS))]
    block, code = rng.choice([16, 32, 64, 128]), rng.choice(["int8", "e4m3"])
    cap = _log(rng, 300, 32768)
    # no more cache than the largest listed case reads
    batch = _log(rng, 1, max(1, min(32, (1 << 28) // (cap * hkv * d))))
    new = 0
    if op == "append":
        new = 1 if rng.random() < 0.4 else min(_log(rng, 2, 2048), cap // 2, max(2, (1 << 24) // (batch * hq * d)))
    if op == "read":
        new = _log(rng, 1, max(1, min(cap, (1 << 24) // (batch * hkv * d))))
    hi = rng.randint(0, cap - new - 2 * block - 1) if cap > new + 2 * block + 1 else 0
    return {"op": op, "batch": batch, "hq": hq, "hkv": hkv, "d": d, "block": block, "code": code, "cap": cap,
            "lo": min(hi, rng.randint(0, hi)), "hi": hi, "new": new}


def _lengths(case):
    """pos[b] of the case: spread evenly over lo .. hi, the same for every seed (the work is the case's)."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi if n == 1 else lo + (hi - lo) * b // (n - 1) for b in range(n)]


def work(case):
    if case["op"] == "logits":
        n, e = case["rows"] * case["vocab"], 4 if case["dtype"] == "float32" else 2
        total = 2 * n * e + 8 * case["rows"] * case["len"] * case["penalties"]
        return {"bytes": total + 4 * n * case["bias"] + n / 8 * case["mask"], "flops": 4 * n}
    b, hq, hkv, d, t = (case[k] for k in ("batch", "hq", "hkv", "d", "block"))
    row = hkv * (2 * d + 8 / t)   # codes and scales of one token's key and value
    if case["op"] == "decode":
        n = sum(p + 1 for p in _lengths(case))
        return {"bytes": n * row + 4 * b * hq * d, "flops": 4.0 * n * hq * d}
    if case["op"] == "read":
        n = sum(min(p, case["new"] or p) for p in _lengths(case))
        return {"bytes": n * row + 4 * b * (case["new"] or case["hi"]) * hkv * d, "flops": 2.0 * n * hkv * d}
    n, back = b * case["new"], b * _window(case)
    move = n * ((hq + 2 * hkv) * 2 * d + (hq + hkv) * 2 * d + row)
    return {"bytes": move + back * (row + 4 * hkv * d), "flops": 6.0 * n * (hq + 2 * hkv) * d}


def _window(case):
    """Rows read back after an append: the new ones and at least the block that the last of them may have filled."""
    return max(case["new"], case["block"])


# ------------------------------------------------------------------------------------------------------ inputs
def _codes(x, block, code):
    """bf16 [B, H, N * T, D] -> codes and scales [B, H, N] of whole blocks, in 32 bits."""
    b, h, n, d = x.shape
    w = x.float().view(b, h, n // block, block * d)
    s = (w.abs().amax(-1) / QMAX[code]).clamp_min(TINY)
    q = w * s.reciprocal()[..., None]
    q = q.round().clamp(-127, 127) if code == "int8" else q.clamp(-448, 448)
    return q.to(CODE[code]).view(b, h, n, d), s


def _tables(d, n):
    f = 10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * f
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if case["op"] == "logits":
        n, v, length = case["rows"], case["vocab"], case["len"]
        dt = getattr(torch, case["dtype"])
        st = {"op": "logits", "logits": (3.0 * randn(n, v)).to(dt)}
        # a history repeats itself: half of it comes from a few dozen tokens
        ids = torch.randint(0, v, (n, length), device=DEV, generator=g)
        few = torch.randint(0, min(v, 40), (n, length), device=DEV, generator=g)
        st["tokens"] = torch.where(torch.rand(n, length, device=DEV, generator=g) < 0.5, ids, few)
        lens = torch.randint(max(1, length // 2), length + 1, (n,), device=DEV, generator=g)
        st["lengths"] = lens.int()
        st["prompt"] = (lens // 3).int()
        st["rep"] = 1.0 + 0.3 * torch.rand(n, device=DEV, generator=g)
        st["pres"] = torch.rand(n, device=DEV, generator=g)
        st["freq"] = 0.2 * torch.rand(n, device=DEV, generator=g)
        st["bias"] = randn(n, v) if case["bias"] else None
        st["mask"] = None
        if case["mask"]:   # a grammar leaves few tokens or most of them; bit v % 32 of word v / 32
            words = torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), device=DEV, generator=g, dtype=torch.int64)
            more = torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), device=DEV, generator=g, dtype=torch.int64)
            keep = torch.rand(n, 1, device=DEV, generator=g) < 0.5
            st["mask"] = torch.where(keep, words | more, words & more).int()
        return st

    b, hq, hkv, d, t = (case[k] for k in ("batch", "hq", "hkv", "d", "block"))
    cap, new = case["cap"], case["new"]
    full = cap // t * t
    st = {"op": case["op"], "block": t, "code": case["code"], "hq": hq, "hkv": hkv, "d": d, "cap": cap,
          "max_len": min(max(_lengths(case)) + 1, cap)}
    # keys have a few channels that are far larger than the others, values do not
    loud = 1.0 + 4.0 * (torch.rand(1, hkv, 1, d, device=DEV, generator=g) < 0.05).float()
    for name, gain in (("k", loud), ("v", 1.0)):
        codes, scales = _codes((randn(b, hkv, full, d) * gain).bfloat16(), t, case["code"])
        room = torch.zeros(b, hkv, cap, d, dtype=CODE[case["code"]], device=DEV)
        room[:, :, :full] = codes
        st[name] = room.transpose(1, 2)   # [B, Smax, Hkv, D], each head's rows next to each other in memory
        st[name + "_scale"] = scales.transpose(1, 2)
        st[name + "_tail"] = (randn(b, hkv, t, d) * gain).bfloat16().transpose(1, 2)
    st["pos"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    st["count"] = new or max(1, case["hi"])
    if case["op"] != "read":
        st["qkv"] = randn(b, new or 1, (hq + 2 * hkv) * d).bfloat16()
    if case["op"] == "append":
        st["cos"], st["sin"] = _tables(d, cap)
        st["count"] = _window(case)
        st["pos_after"] = st["pos"] + new
    return st


# --------------------------------------------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, at):
    """Interleaved pairs of x [B, S, H, D] rotated by the angles of positions at [B, S]: products in 64 bits."""
    co, si = (c[at].double()[:, :, None] for c in (cos, sin))
    a, b = x.double().unflatten(-1, (-1, 2)).unbind(-1)
    return torch.stack([a * co - b * si, a * si + b * co], -1).flatten(-2).float().bfloat16()


def _split(st):
    hq, hkv, d = st["hq"], st["hkv"], st["d"]
    b, s, _ = st["qkv"].shape
    x = st["qkv"].view(b, s, hq + 2 * hkv, d)
    return x[:, :, :hq], x[:, :, hq:hq + hkv], x[:, :, hq + hkv:]


def _append(st):
    t, code, pos = st["block"], st["code"], st["pos"].long()
    q, k, v = _split(st)
    b, s = q.shape[:2]
    at = pos[:, None] + torch.arange(s, device=DEV)
    q.copy_(_rotate(q, st["cos"], st["sin"], at))
    k.copy_(_rotate(k, st["cos"], st["sin"], at))
    row = torch.arange(b, device=DEV)[:, None]
    first, end = pos // t * t, pos + s
    blocks = (s + t - 2) // t + 1   # blocks that the new rows can touch
    win = first[:, None] + torch.arange(blocks * t, device=DEV)   # absolute rows of the window
    is_new = (win >= pos[:, None])[..., None, None]
    done = (first[:, None] + t * (1 + torch.arange(blocks, device=DEV)) <= end[:, None])[..., None, None]
    inside = (win - pos[:, None]).clamp(0, s - 1)
    slots = torch.arange(t, device=DEV)
    last = (end // t * t)[:, None] + slots   # absolute rows of the open block after the append
    put = ((last >= pos[:, None]) & (last < end[:, None]))[..., None, None]
    there = (last - pos[:, None]).clamp(0, s - 1)
    bi = first[:, None] // t + torch.arange(blocks, device=DEV)
    bi_in = bi.clamp_max(st["k_scale"].shape[1] - 1)
    win_in = win.clamp_max(st["cap"] - 1)
    for name, x in (("k", k), ("v", v)):
        tail = st[name + "_tail"]
        w = torch.where(is_new, x[row, inside], tail[:, slots.repeat(blocks)]).float()
        w = w.unflatten(1, (blocks, t)).transpose(2, 3).flatten(3)   # [B, blocks, Hkv, T * D]
        sc = (w.abs().amax(-1) / QMAX[code]).clamp_min(TINY)
        c = w * sc.reciprocal()[..., None]
        c = c.round().clamp(-127, 127) if code == "int8" else c.clamp(-448, 448)
        c = c.unflatten(3, (t, -1)).transpose(2, 3).to(CODE[code])
        old = st[name].view(torch.uint8)
        c = torch.where(done[..., None], c.view(torch.uint8), old[row, win_in].unflatten(1, (blocks, t)))
        old[row, win_in] = c.flatten(1, 2)
        scales = st[name + "_scale"]
        scales[row, bi_in] = torch.where(done[..., 0], sc, scales[row, bi_in])
        tail.copy_(torch.where(put, x[row, there], tail))


def _values(st, name, at, n):
    """fp32 rows at [B, R] of the cache that holds n [B] tokens."""
    t = st["block"]
    row = torch.arange(at.shape[0], device=DEV)[:, None]
    stored = st[name][row, at].float() * st[name + "_scale"][row, (at // t).clamp_max(st["cap"] // t - 1)][..., None]
    is_open = (at >= (n // t * t)[:, None])[..., None, None]
    return torch.where(is_open, st[name + "_tail"][row, at % t].float(), stored)


def _read(st, pos):
    n = pos.long()
    at = n[:, None] - st["count"] + torch.arange(st["count"], device=DEV)
    real = (at >= 0)[..., None, None]
    return [torch.where(real, _values(st, name, at.clamp_min(0), n), 0.0).bfloat16() for name in ("k", "v")]


def _decode(st):
    n = st["pos"].long() + 1
    q = _split(st)[0].float()
    b, _, hq, d = q.shape
    hkv = st["hkv"]
    at = torch.arange(st["max_len"], device=DEV).expand(b, -1)
    k = _values(st, "k", at, n).permute(0, 2, 3, 1)   # [B, Hkv, D, n]
    s = (q.view(b, hkv, hq // hkv, d) / math.sqrt(d)) @ k
    del k
    s = s.masked_fill((at >= n[:, None])[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return (p @ _values(st, "v", at, n).transpose(1, 2)).reshape(b, hq * d).bfloat16()


def _process(st):
    x = st["logits"].float()
    n, v = x.shape
    at = torch.arange(st["tokens"].shape[1], device=DEV)
    valid = at < st["lengths"][:, None]
    made = valid & (at >= st["prompt"][:, None])
    seen = torch.zeros(n, v, device=DEV).scatter_add_(1, st["tokens"], valid.float()) > 0
    count = torch.zeros(n, v, device=DEV).scatter_add_(1, st["tokens"], made.float())
    rep = st["rep"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (st["freq"][:, None] * count + st["pres"][:, None] * (count > 0))
    if st["bias"] is not None:
        x = x + st["bias"]
    if st["mask"] is not None:
        ids = torch.arange(v, device=DEV)
        x = torch.where((st["mask"][:, ids // 32] >> (ids % 32)) & 1 == 1, x, -math.inf)
    return x.to(st["logits"].dtype)


def run(state):
    op = state["op"]
    if own:
        from distributed_pytorch_hpc_amd import ops

        if op == "logits":
            return ops.process_logits(state["logits"], state["tokens"], state["lengths"], state["prompt"],
                                      repetition=state["rep"], presence=state["pres"], frequency=state["freq"],
                                      bias=state["bias"], mask=state["mask"])
        cache = ops.KV8Cache(*(state[name] for name in STATE))
        if op == "decode":
            return ops.kv8_decode_attention(state["qkv"], cache, state["pos"], state["hq"], state["hkv"],
                                            max_len=state["max_len"])
        if op == "read":
            return ops.kv8_read(cache, state["pos"], state["count"])
        ops.kv8_append_(state["qkv"], cache, state["pos"], state["cos"], state["sin"], state["hq"], state["hkv"])
        return [state["qkv"], *ops.kv8_read(cache, state["pos_after"], state["count"])]
    if op == "logits":
        return _process(state)
    if op == "decode":
        return _decode(state)
    if op == "read":
        return _read(state, state["pos"])
    _append(state)
    return [state["qkv"], *_read(state, state["pos_after"])]


# -------------------------------------------------------------------------------------------------------- exact
def _exact_rows(st, name, b, n, tail=None, codes=None):
    """The n rows of sequence b as 64-bit values [n, Hkv, D]; ``codes`` a dict of blocks quantised meanwhile."""
    t = st["block"]
    full = n // t
    rows = st[name][b, :full * t].double().unflatten(0, (full, t)) * st[name + "_scale"][b, :full].double()[:, None, :, None]
    rows = rows.flatten(0, 1)
    return torch.cat([rows, (st[name + "_tail"][b] if tail is None else tail)[:n - full * t].double()])


def _exact_append(st):
    t, lim = st["block"], QMAX[st["code"]]
    b, s, width = st["qkv"].shape
    hq, hkv, d = st["hq"], st["hkv"], st["d"]
    x = st["qkv"].double().view(b, s, hq + 2 * hkv, d // 2, 2).clone()
    outs = ([], [])
    for i, p in enumerate(st["pos"].tolist()):
        z = torch.complex(st["cos"][p:p + s].double(), st["sin"][p:p + s].double())[:, None]
        x[i, :, :hq + hkv] = torch.view_as_real(torch.view_as_complex(x[i, :, :hq + hkv]) * z)
        rows = x[i].flatten(-2)
        for out, name, h in ((outs[0], "k", hq), (outs[1], "v", hq + hkv)):
            first = p // t
            fresh = rows[:, h:h + hkv].bfloat16().double()   # stored values are bf16 before they are quantised
            held = _exact_rows(st, name, i, p)
            body = torch.cat([held[first * t:], fresh])
            whole = body.shape[0] // t
            w = body[:whole * t].unflatten(0, (whole, t))
            sc = (w.abs().amax((1, 3), keepdim=True) / lim).clamp_min(TINY)
            c = (w / sc).round() if st["code"] == "int8" else (w / sc).float().to(CODE["e4m3"]).double()
            kept = torch.cat([held[:first * t], (c * sc).flatten(0, 1), body[whole * t:]])
            pad = torch.zeros(st["count"], hkv, d, dtype=torch.float64, device=DEV)
            out.append(torch.cat([pad, kept])[-st["count"]:])
    return [x.reshape(b, s, width), torch.stack(outs[0]), torch.stack(outs[1])]


def exact(case, seed):
    st = prepare(case, seed)
    if st["op"] == "logits":
        x = st["logits"].double()
        n, v = x.shape
        for i in range(n):
            m, p = int(st["lengths"][i]), int(st["prompt"][i])
            ids = st["tokens"][i]
            said = torch.bincount(ids[:m], minlength=v)
            made = torch.bincount(ids[p:m], minlength=v)
            r, f, a = (st[key][i].double() for key in ("rep", "freq", "pres"))
            y = torch.where(said > 0, torch.minimum(x[i] * r, x[i] / r), x[i])   # r >= 1: the smaller of the two
            x[i] = y - f * made - a * (made > 0)
            if st["bias"] is not None:
                x[i] += st["bias"][i].double()
            if st["mask"] is not None:
                bits = (st["mask"][i].long()[:, None] >> torch.arange(32, device=DEV)) % 2
                x[i][bits.flatten()[:v] == 0] = -math.inf
        return x
    if st["op"] == "append":
        return _exact_append(st)
    lens = st["pos"].tolist()
    if st["op"] == "read":
        outs = []
        for name in ("k", "v"):
            pad = torch.zeros(st["count"], st["hkv"], st["d"], dtype=torch.float64, device=DEV)
            outs.append(torch.stack([torch.cat([pad, _exact_rows(st, name, i, n)])[-st["count"]:]
                                     for i, n in enumerate(lens)]))
        return outs
    outs = []
    for i, p in enumerate(lens):
        q = st["qkv"][i, 0, :st["hq"] * st["d"]].double().view(st["hkv"], -1, st["d"])
        k, v = (_exact_rows(st, name, i, p + 1).transpose(0, 1) for name in ("k", "v"))
        w = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(st["d"]), -1)
        outs.append((w @ v).reshape(-1))
    return torch.stack(outs)
