"""The block-scaled 8-bit cache and the logit controls in the serving loops, on the CPU (references of the kernels)."""
import math

import pytest
import torch

from dist_utils import run_distributed
from test_inference import _model

CODES = [torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("block", [16, 32])
def test_block_scaled_cache_tracks_the_full_forward(dtype, block):
    """Prefill, decode over a block border, a chunked append and further steps; logits stay close to the exact forward.
    The same bound as the one-scale e4m3 cache's test."""
    from distributed_pytorch_hpc_amd.models.llama2 import KVCache

    m = _model()
    t = torch.randint(0, 97, (2, 50), generator=torch.Generator().manual_seed(1))
    full = m(t)
    c = KVCache(m, 2, 60, dtype=dtype, kv_block=block)
    assert not c.fp8 and c.k[0].dtype == dtype and len(c.blocks) == 2
    got = [m.forward_inference(t[:, :10], c)]
    got += [m.forward_inference(t[:, i:i + 1], c) for i in range(10, 20)]
    got.append(m.forward_inference(t[:, 20:45], c, last_only=False)[:, -1])
    got += [m.forward_inference(t[:, i:i + 1], c) for i in range(45, 50)]
    got = torch.stack(got, 1)
    ref = torch.stack([full[:, i] for i in [*range(9, 20), *range(44, 50)]], 1)
    assert c.pos.tolist() == [50, 50]
    assert (got - ref).norm() / ref.norm() < 0.05


def test_block_scaled_cache_slots_and_refusals():
    from distributed_pytorch_hpc_amd.inference import ContinuousBatcher, Generator
    from distributed_pytorch_hpc_amd.models.llama2 import KVCache

    m = _model()
    with pytest.raises(ValueError, match="kv_block"):
        KVCache(m, 1, 32, dtype=torch.int8)
    with pytest.raises(ValueError, match="kv_scale"):
        KVCache(m, 1, 32, dtype=torch.int8, kv_block=16, kv_scale=0.5)
    with pytest.raises(ValueError, match="dtype"):
        KVCache(m, 1, 32, kv_block=16)
    c = KVCache(m, 2, 32, dtype=torch.int8, kv_block=16)
    m.forward_inference(torch.tensor([[1, 2, 3]]), c.slot(0))
    with pytest.raises(RuntimeError, match="same, host-known length"):
        m.forward_inference(torch.tensor([[1, 2], [3, 4]]), c)
    # requests of different lengths on two slots equal each one generated alone over such a cache
    reqs = [([1, 2, 3], 20), ([4, 5, 6, 7, 8, 9], 3), ([10], 25), ([11, 12], 1), ([13, 14, 15, 16] * 5, 9)]
    cb = ContinuousBatcher(Generator(m, 2, 40, dtype=torch.int8, kv_block=16))
    hs = [cb.submit(p, n) for p, n in reqs]
    cb.run()
    solo = Generator(m, 1, 40, dtype=torch.int8, kv_block=16)
    for h, (p, n) in zip(hs, reqs):
        assert h.prompt + h.output == solo.generate([p], n)[0]


def _naive(m, prompt, n, c, bias=None):
    """Greedy generation by full forwards with the controls written out."""
    x, made = list(prompt), []
    for _ in range(n):
        z = m(torch.tensor([x]))[0, -1].double()
        for t in set(x):
            z[t] = z[t] / c.repetition_penalty if z[t] > 0 else z[t] * c.repetition_penalty
        for t in set(made):
            z[t] -= c.frequency_penalty * made.count(t) + c.presence_penalty
        if bias is not None:
            z += bias.double()
        if c.allowed is not None:
            a = c.allowed(made)
            if a is not None:
                z[~a] = -math.inf
        t = int(z.argmax())
        x.append(t)
        made.append(t)
    return x


def _controls():
    from distributed_pytorch_hpc_amd.inference import LogitControls

    bias = torch.zeros(97)
    bias[5], bias[6] = 3.0, -math.inf

    def grammar(made):   # even and odd tokens in turns, anything for the first
        return None if not made else torch.arange(97) % 2 == len(made) % 2

    return [LogitControls(repetition_penalty=1.5), LogitControls(presence_penalty=0.7, frequency_penalty=0.4),
            LogitControls(bias={5: 3.0, 6: -math.inf}), LogitControls(allowed=grammar),
            LogitControls(1.3, 0.2, 0.1, bias, grammar)], [None, None, bias, None, bias]


def test_generate_with_controls_matches_naive():
    from distributed_pytorch_hpc_amd.inference import Generator

    m = _model()
    cs, biases = _controls()
    prompts = [[1, 2, 3, 4, 5], [7, 8, 9], [5], [3, 3, 3, 4], [1, 5, 6]]
    want = [_naive(m, p, 12, c, b) for p, c, b in zip(prompts, cs, biases)]
    g = Generator(m, 5, 32)
    assert g.generate(prompts, 12, controls=cs) == want
    one = Generator(m, 5, 32).generate(prompts, 6, controls=[cs[0], None, None, None, None])
    assert one[0] == want[0][:11] and one[1:] == Generator(m, 5, 32).generate(prompts, 6)[1:]
    assert g.generate(prompts, 3, controls=cs[0])[0] == want[0][:8]


def test_continuous_batching_with_controls_matches_one_request_at_a_time():
    from distributed_pytorch_hpc_amd.inference import ContinuousBatcher, Generator

    m = _model()
    cs, _ = _controls()
    reqs = [([1, 2, 3], 9, cs[0]), ([4, 5, 6], 3, None), ([10], 6, cs[4]), ([11, 12], 1, cs[1]), ([3, 3], 8, cs[3]),
            ([13, 14], 7, None), ([5], 5, cs[2])]
    cb = ContinuousBatcher(Generator(m, 2, 16))
    hs = [cb.submit(p, n, controls=c) for p, n, c in reqs]
    assert len(cb.run()) == len(reqs)
    solo = Generator(m, 1, 16)
    for h, (p, n, c) in zip(hs, reqs):
        assert h.prompt + h.output == solo.generate([p], n, controls=c)[0]


def test_a_grammar_that_fails_drops_its_request_alone():
    from distributed_pytorch_hpc_amd.inference import ContinuousBatcher, Generator, LogitControls

    m = _model()
    none = LogitControls(allowed=lambda made: torch.zeros(97, dtype=torch.bool) if len(made) == 2 else None)
    cb = ContinuousBatcher(Generator(m, 2, 16))
    a, b, c = cb.submit([1, 2, 3], 6), cb.submit([4, 5], 6, controls=none), cb.submit([7], 4)
    done = []
    with pytest.raises(ValueError, match="no token"):
        while cb.queue or cb.active:
            done += cb.step()
    done += cb.run()
    assert not b.done and len(b.output) == 2 and a.done and c.done and {id(r) for r in done} == {id(a), id(c)}
    solo = Generator(m, 1, 16)
    assert a.output == solo.generate([[1, 2, 3]], 6)[0][3:] and c.output == solo.generate([[7]], 4)[0][1:]
    with pytest.raises(ValueError, match="no token"):
        Generator(m, 1, 16).generate([[1]], 5, controls=none)


def test_control_refusals():
    from distributed_pytorch_hpc_amd.inference import ContinuousBatcher, Generator, LogitControls

    m = _model()
    for kw in (dict(repetition_penalty=0.0), dict(repetition_penalty=math.inf), dict(presence_penalty=math.nan)):
        with pytest.raises(ValueError):
            LogitControls(**kw)
    g = Generator(m, 1, 16)
    for bias in ({97: 1.0}, torch.zeros(5), torch.full((97,), -math.inf), {3: math.nan}, {3: math.inf}):
        with pytest.raises(ValueError):
            g.generate([[1]], 2, controls=LogitControls(bias=bias))
        with pytest.raises(ValueError):
            ContinuousBatcher(g).submit([1], 2, controls=LogitControls(bias=bias))
    for a in (torch.ones(96, dtype=torch.bool), torch.ones(97)):
        with pytest.raises(ValueError, match="bool tensor"):
            g.generate([[1]], 2, controls=LogitControls(allowed=lambda made, a=a: a))
    ban = torch.zeros(97)
    ban[:50] = -math.inf
    with pytest.raises(ValueError, match="no token"):
        g.generate([[1]], 2, controls=LogitControls(bias=ban, allowed=lambda made: torch.arange(97) < 50))
    with pytest.raises(ValueError, match="controls for"):
        g.generate([[1]], 2, controls=[None, None])


def test_temperature_sampling_stays_inside_the_mask():
    from distributed_pytorch_hpc_amd.inference import Generator, LogitControls

    m = _model()
    few = torch.zeros(97, dtype=torch.bool)
    few[[3, 50, 96]] = True
    out = Generator(m, 2, 32).generate([[1], [2, 3]], 20, temperature=2.0, top_k=10, controls=LogitControls(allowed=lambda _: few),
                                       generator=torch.Generator().manual_seed(0))
    assert set(out[0][1:]) | set(out[1][2:]) <= {3, 50, 96}


def _tp_worker(rank, world):
    import torch.distributed as dist

    from distributed_pytorch_hpc_amd.inference import Generator, LogitControls
    from distributed_pytorch_hpc_amd.parallel.tensor_parallel import parallelize_llama

    m = _model(vocab=96)
    if world > 1:
        parallelize_llama(m, dist.group.WORLD, sequence_parallel=False, loss_parallel=False)
    return Generator(m, 2, 40, dtype=torch.int8, kv_block=16).generate(
        [[1, 2, 3, 4, 5], [7, 8, 9, 10, 11]], 20, controls=LogitControls(repetition_penalty=1.3, frequency_penalty=0.1))


def test_tensor_parallel_block_scaled_cache_with_controls():
    """A scale belongs to one KV head, so sharding the heads over two ranks changes neither codes nor tokens."""
    ref = _tp_worker(0, 1)
    for out in run_distributed(_tp_worker, 2):
        assert out == ref


def test_example_runs_with_block_scaled_cache_and_penalty():
    import json
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, os.path.join(root, "examples", "08_serving", "generate_llama.py"), "--model",
                          "tiny", "--batch", "2", "--prompt-len", "20", "--max-new", "18", "--kv-dtype", "int8",
                          "--kv-block", "16", "--repetition-penalty", "1.3"], capture_output=True, text=True, timeout=300,
                         env=dict(os.environ, MASTER_ADDR="127.0.0.1"))
    assert out.returncode == 0, out.stderr[-2000:]
    s = json.loads([ln for ln in out.stdout.splitlines() if ln.startswith("{")][-1])
    assert s["kv_dtype"] == "int8" and len(s["first_sequence_new_ids"]) == 16
