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
