"""The serving loops over a block-scaled 8-bit cache with logit controls, on the MI355X: graph replays equal eager steps,
logits stay close to the full forward, histories follow the tokens on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CODES = [torch.int8, torch.float8_e4m3fn]


def _tiny_llama(seed=0):
    from distributed_pytorch_hpc_amd.models.llama2 import ModelArgs, build_llama

    args = ModelArgs(dim=512, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, multiple_of=64, max_seq_len=256)
    return build_llama(args, device="cuda", dtype=torch.bfloat16, seed=seed)


@pytest.mark.parametrize("dtype", CODES)
@pytest.mark.parametrize("block", [16, 64])
def test_block_scaled_cache_matches_full_forward(dph_native, dtype, block):
    """Prefill, decode, a chunked append over a prefix that ends inside a block, decode: the 5 % of the one-scale cache."""
    from distributed_pytorch_hpc_amd.models.llama2 import KVCache

    m = _tiny_llama()
    t = torch.randint(0, 512, (2, 150), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    with torch.no_grad():
        full = m(t)
    c = KVCache(m, 2, 160, dtype=dtype, kv_block=block)
    got = [m.forward_inference(t[:, :61], c)]
    got += [m.forward_inference(t[:, i:i + 1], c) for i in range(61, 75)]
    got.append(m.forward_inference(t[:, 75:130], c))
    got += [m.forward_inference(t[:, i:i + 1], c) for i in range(130, 150)]
    got = torch.stack(got, 1)
    ref = full[:, [60, *range(61, 75), 129, *range(130, 150)]]
    assert (got - ref).norm() / ref.norm() < 0.05


def _controls():
    from distributed_pytorch_hpc_amd.inference import LogitControls

    ids = torch.arange(512)
    return [LogitControls(repetition_penalty=1.3, frequency_penalty=0.2),
            LogitControls(bias={7: 2.0}, allowed=lambda made: ids % 3 == len(made) % 3),
            None, LogitControls(1.1, 0.3, 0.1, torch.linspace(-1, 1, 512))]


@pytest.mark.parametrize("dtype", CODES)
def test_generate_graphed_equals_eager(dph_native, dtype):
    from distributed_pytorch_hpc_amd.inference import Generator

    m = _tiny_llama(seed=3)
    prompts = [[5, 6, 7, 8, 9, 10], [11, 12, 13], [1] * 20, [2]]
    eager = Generator(m, 4, 80, graphs=False, dtype=dtype, kv_block=16).generate(prompts, 50, controls=_controls())
    g = Generator(m, 4, 80, graphs=True, dtype=dtype, kv_block=16)
    assert g.generate(prompts, 50, controls=_controls()) == eager and g._graph is not None
    assert g.generate(prompts, 50, controls=_controls()) == eager   # replays after a reset
    assert all((t % 3) == i % 3 for i, t in enumerate(eager[1][3:]))


def test_continuous_batching_graphed_equals_eager(dph_native):
    """Six requests on two slots, with and without controls: a captured step gives what eager steps give."""
    from distributed_pytorch_hpc_amd.inference import ContinuousBatcher, Generator

    m = _tiny_llama(seed=9)
    cs = _controls()
    reqs = [([5, 6, 7], 9, cs[0]), ([8, 9, 10, 11, 12, 13, 14], 4, None), ([15], 30, cs[1]), ([16, 17], 2, None),
            ([18, 19, 20, 21], 17, cs[3]), ([22] * 18, 20, cs[0])]

    def serve(graphs):
        cb = ContinuousBatcher(Generator(m, 2, 48, graphs=graphs, dtype=torch.int8, kv_block=16))
        hs = [cb.submit(p, n, controls=c) for p, n, c in reqs]
        cb.run()
        return [h.output for h in hs]

    eager = serve(False)
    assert serve(True) == eager
    assert [len(o) for o in eager] == [n for _, n, _ in reqs]
    assert all((t % 3) == i % 3 for i, t in enumerate(eager[2]))


def test_processor_keeps_history_on_the_device(dph_native):
    """push / start / stop / push_one leave the history that the controls then see, compared with the CPU's."""
    from distributed_pytorch_hpc_amd.inference import LogitControls, LogitProcessor

    outs = []
    for dev in ("cuda", "cpu"):
        p = LogitProcessor(3, 6, 512, dev)
        p.start(0, [3, 4], LogitControls(2.0, 0.5, 0.25))
        p.start(2, [7], LogitControls(presence_penalty=1.0))
        p.push(torch.tensor([4, 9, 8], device=dev))
        p.stop(2)
        p.start(1, [1, 1, 1], LogitControls(frequency_penalty=0.5))
        p.push_one(1, 2)
        for t in ([4, 2, 5], [6, 2, 5], [6, 5, 5], [6, 5, 5]):   # row 0 and 1 run past the room of 6
            p.push(torch.tensor(t, device=dev))
        z = torch.linspace(-2, 2, 3 * 512).view(3, 512).to(dev)
        outs.append((p.tokens.cpu(), p.lengths.cpu(), p(z).cpu(), p(z[1:2], row=1).cpu()))
    for a, b in zip(*outs):
        torch.testing.assert_close(a, b, rtol=0, atol=8 * 2.0 ** -24 * 4)   # eight roundings of values below 4


def test_unsupported_head_dim_is_refused_with_the_cache(dph_native):
    """Not at the first append: a model with heads of 16 gets no block-scaled cache on the GPU, and keeps its bf16 one."""
    from distributed_pytorch_hpc_amd.inference import Generator
    from distributed_pytorch_hpc_amd.models.llama2 import KVCache, ModelArgs, build_llama

    m = build_llama(ModelArgs(dim=64, n_layers=1, n_heads=4, n_kv_heads=2, vocab_size=96, multiple_of=32, max_seq_len=64),
                    device="cuda", dtype=torch.bfloat16)
    for make in (KVCache, Generator):
        with pytest.raises(ValueError, match="head dim"):
            make(m, 2, 32, dtype=torch.int8, kv_block=16)
    KVCache(m, 2, 32)
