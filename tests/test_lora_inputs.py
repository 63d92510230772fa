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


@pytest.mark.gpu
def test_one_row_of_any_pitch(native):
    """A single row cut from a tensor whose rows are no whole 16-byte pieces apart: a row has no stride to speak of."""
    K, N = 512, 256
    x, w, b, A, B, scale = _make(4, N, K, [16, 8], "cuda")
    bank, ids = ops.LoraBank(A, B, scale), torch.tensor([1], device="cuda")
    y, err = _ref(x[:1], w, b, A, B, scale, ids, 2.0 ** -8)
    for pad in (3, 4, 8):
        wide = torch.zeros(4, K + pad, device="cuda", dtype=BF)
        wide[:, :K] = x
        got = ops.linear_lora(wide[:1, :K], w, b, bank=bank, ids=ids)
        _compare(got, y, err, None, 2.0 ** -8)
        out, resid = torch.zeros(4, N + pad, device="cuda", dtype=BF), torch.ones(4, N + pad, device="cuda", dtype=BF)
        gate = torch.ones(1, N + pad, device="cuda")[:, :N]
        assert torch.equal(ops.linear_lora(wide[:1, :K], w, b, bank=bank, ids=ids, out=out[:1, :N]), got)
        assert torch.equal(out[:1, :N], got) and bool((out[1:] == 0).all() and (out[:, N:] == 0).all())
        gated = ops.linear_lora(wide[:1, :K], w, b, bank=bank, ids=ids, gate=gate, resid=resid[:1, :N])
        assert torch.equal(gated, ops.linear_lora(x[:1], w, b, bank=bank, ids=ids, gate=gate, resid=torch.ones(1, N, device="cuda", dtype=BF)))
