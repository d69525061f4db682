"""Edges of the logit controls in the serving loops, on the CPU."""
import pytest
import torch

from test_inference import _model


def test_processor_hands_over_the_history_in_use(monkeypatch):
    """However much room there is, the operator gets as many columns as the longest history it has to look at holds, and
    the logits are those of the whole buffer."""
    from distributed_pytorch_hpc_amd import ops
    from distributed_pytorch_hpc_amd.inference import LogitControls, LogitProcessor

    widths, plain = [], ops.process_logits

    def spy(logits, tokens=None, lengths=None, **kw):
        widths.append(tokens.shape[1])
        whole = proc.tokens if logits.shape[0] > 1 else proc.tokens[1:2]
        y = plain(logits, tokens, lengths, **kw)
        assert torch.equal(y, plain(logits, whole, lengths, **kw))
        assert int(lengths.max()) == tokens.shape[1]
        return y

    monkeypatch.setattr(ops, "process_logits", spy)
    proc = LogitProcessor(3, 9, 20, "cpu")
    z = torch.linspace(-2, 2, 60).view(3, 20)
    c = LogitControls(1.5, 0.5, 0.25)
    proc.start(0, [3, 4], c)
    proc(z)
    proc.start(1, [5, 6, 7, 8], c)
    proc(z)
    proc.push_one(1, 2)
    proc(z[1:2], row=1)
    proc.push(torch.tensor([1, 2, 3]))
    proc(z)
    proc.stop(1)
    proc(z)
    for _ in range(8):   # past the room
        proc.push(torch.tensor([1, 2, 3]))
    proc(z)
    proc.push_one(0, 4)
    proc(z)
    proc.start(2, [], c)
    proc.stop(0)
    proc(z)
    assert widths == [2, 4, 5, 6, 3, 9, 9, 0]


LOWEST = [torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min, -1e39, -1e300]


@pytest.mark.parametrize("low", LOWEST)
@pytest.mark.parametrize("temperature", [0.0, 0.5])
def test_a_bias_of_the_lowest_value_bans_a_token(low, temperature):
    """As -inf does: the others are sampled, and where none is left the call is refused before it has sampled."""
    from distributed_pytorch_hpc_amd.inference import ContinuousBatcher, Generator, LogitControls

    m = _model()
    g = Generator(m, 1, 16)
    for bias in ({t: low for t in range(50)}, low * (torch.arange(97) < 50).double()):
        out = g.generate([[1]], 8, temperature=temperature, controls=LogitControls(bias=bias, presence_penalty=1.0),
                         generator=torch.Generator().manual_seed(0))
        assert min(out[0][1:]) >= 50
        with pytest.raises(ValueError, match="no token"):
            g.generate([[1]], 2, temperature=temperature,
                       controls=LogitControls(bias=bias, allowed=lambda made: torch.arange(97) < 50))
    for c in (g.generate, ContinuousBatcher(g).submit):
        with pytest.raises(ValueError, match="no token"):
            c([[1]] if c == g.generate else [1], 2, controls=LogitControls(bias=torch.full((97,), low, dtype=torch.float64)))


@pytest.mark.parametrize("kw", [dict(repetition_penalty=1e-50), dict(repetition_penalty=1e39), dict(repetition_penalty=1e-30),
                                dict(presence_penalty=1e39), dict(frequency_penalty=-1e39), dict(presence_penalty=-1e300),
                                dict(frequency_penalty=3e38)])
def test_penalties_that_leave_32_bits_are_refused(kw):
    """1e-50 is zero in 32 bits, 1e39 infinite, and a few copies of a token times 3e38 are."""
    from distributed_pytorch_hpc_amd.inference import LogitControls

    with pytest.raises(ValueError, match="LogitControls"):
        LogitControls(**kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_controls_leave_finite_logits(dtype):
    from distributed_pytorch_hpc_amd.inference import LogitControls, LogitProcessor

    z = torch.linspace(-2.0 ** 35, 2.0 ** 35, 20)[None].to(dtype)
    for sign in (1, -1):
        for rep in (2.0 ** 64, 2.0 ** -64):
            p = LogitProcessor(1, 40, 20, "cpu")
            p.start(0, list(range(20)), LogitControls(rep, sign * 2.0 ** 64, sign * 2.0 ** 64,
                                                      torch.full((20,), -sign * 2.0 ** 100)))
            for t in range(20):
                p.push(torch.tensor([t]))
            y = p(z)
            assert torch.isfinite(y).all() and torch.isfinite(y.float() / 2.0 ** -25).all()
    with pytest.raises(ValueError, match="biases"):
        LogitProcessor(1, 4, 20, "cpu").start(0, [1], LogitControls(bias={3: 2.0 ** 101}))
