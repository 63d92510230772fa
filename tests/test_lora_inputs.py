"""What ``ops.LoraBank`` and ``ops.linear_lora`` accept and refuse beside ``test_linear_lora``'s cases."""

import pytest
import torch

from difflet_b200 import ops
from test_linear_lora import _compare, _make, _ref

BF = torch.bfloat16


def _gradients_are_refused(device, dtype):
    x, w, b, A, B, scale = _make(5, 24, 32, [4, 4], device, dtype)
    bank = ops.LoraBank(A, B, scale)
    ids = torch.zeros(5, dtype=torch.long, device=device)
    ask = lambda t: t.clone().requires_grad_()  # noqa: E731
    with pytest.raises(RuntimeError, match="no backward"):
        ops.linear_lora(x, ask(w), b, bank=bank, ids=ids)
    for args in (([ask(A[0]), A[1]], B), (A, [B[0], ask(B[1])]), (A, B, torch.ones(2, device=device, requires_grad=True))):
        with pytest.raises(RuntimeError, match="no backward"):
            ops.LoraBank(*args)
    want = ops.linear_lora(x, w, b, bank=bank, ids=ids)
    with torch.no_grad():
        got = ops.linear_lora(x, ask(w), b, bank=ops.LoraBank([ask(a) for a in A], B, scale), ids=ids)
    assert torch.equal(got, want) and not got.requires_grad


def test_gradients_are_refused():
    _gradients_are_refused("cpu", torch.float32)


@pytest.mark.gpu
def test_gradients_are_refused_on_cuda(native):
    _gradients_are_refused("cuda", BF)
