"""No operator of the 8-bit KV cache or of the logits loses a gradient silently (HIP kernels)."""
import pytest
import torch

from kv8_grads import CASES, call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op,need", CASES)
def test_operands_that_require_grad_are_refused(dph_native, op, need):
    with pytest.raises(RuntimeError, match="no backward"):
        call(op, "cuda", need)
    with torch.no_grad():
        call(op, "cuda", need)
    call(op, "cuda")
