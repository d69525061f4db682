"""No operator of the 8-bit KV cache or of the logits loses a gradient silently (CPU references)."""
import pytest
import torch

from kv8_grads import CASES, call


@pytest.mark.parametrize("op,need", CASES)
def test_operands_that_require_grad_are_refused(op, need):
    with pytest.raises(RuntimeError, match="no backward"):
        call(op, "cpu", need)
    with torch.no_grad():
        call(op, "cpu", need)
    call(op, "cpu")
