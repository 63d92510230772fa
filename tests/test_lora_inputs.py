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


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 40, 300])
def test_gate_and_residual_of_any_alignment(native, M):
    """Rows that 16-byte accesses do not reach are laid out first, whatever kernel the number of rows selects."""
    K, N = 128, 264
    x, w, b, A, B, scale = _make(M, N, K, [16, 8], "cuda")
    bank = ops.LoraBank(A, B, scale)
    ids = torch.tensor([1, 0], device="cuda")
    rpb = -(-M // 2)
    gate, resid = torch.randn(2, N, device="cuda"), torch.randn(M, N, device="cuda", dtype=BF)
    kw = dict(bank=bank, ids=ids, rows_per_batch=rpb)
    want = ops.linear_lora(x, w, b, gate=gate, resid=resid, **kw)
    for off, pad in ((1, 2), (0, 3), (4, 5)):
        g, r = torch.zeros(2, N + pad + off, device="cuda"), torch.zeros(M, N + pad + off, device="cuda", dtype=BF)
        g[:, off:off + N], r[:, off:off + N] = gate, resid
        assert torch.equal(ops.linear_lora(x, w, b, gate=g[:, off:off + N], resid=r[:, off:off + N], **kw), want)
    columns = resid.t().contiguous().t()  # a residual of another order, and a gate shared by all rows
    assert torch.equal(ops.linear_lora(x, w, b, gate=gate.t().contiguous().t(), resid=columns, **kw), want)
    one = torch.zeros(3, N + 1, device="cuda")[:1, :N]
    got = ops.linear_lora(x, w, b, gate=one, resid=resid, gate_rows_per_batch=M, **kw)
    assert torch.equal(got, resid)
    with pytest.raises(ValueError):
        ops.linear_lora(x, torch.zeros(N * K + 1, device="cuda", dtype=BF)[1:].view(N, K), b, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 300])
def test_results_whose_rows_overlap_are_refused(native, M):
    x, w, b, A, B, scale = _make(M, 64, 128, [16], "cuda")
    bank, ids = ops.LoraBank(A, B, scale), torch.zeros(M, device="cuda", dtype=torch.int32)
    for bad in (torch.empty(1, 64, device="cuda", dtype=BF).expand(M, 64), torch.empty(M * 64, device="cuda", dtype=BF).as_strided((M, 64), (32, 1))):
        with pytest.raises(ValueError):
            ops.linear_lora(x, w, b, bank=bank, ids=ids, out=bad)


def _shape_refusals(device, dtype):
    """A bias, gate or residual that would only broadcast is refused on every device."""
    x, w, b, A, B, scale = _make(6, 24, 32, [4, 4], device, dtype)
    bank, ids = ops.LoraBank(A, B, scale), torch.zeros(6, dtype=torch.long, device=device)
    gate, resid = torch.ones(6, 24, device=device), torch.ones(6, 24, device=device, dtype=dtype)
    kw = dict(bank=bank, ids=ids)
    for bad in (dict(gate=gate[:1], resid=resid, gate_rows_per_batch=1), dict(gate=gate[:, :16], resid=resid), dict(gate=gate[0], resid=resid),
                dict(gate=gate[:1], resid=resid[:1]), dict(gate=gate[:1], resid=resid[:, :1]), dict(gate=gate[:2], resid=resid, gate_rows_per_batch=2)):
        with pytest.raises(ValueError):
            ops.linear_lora(x, w, b, **kw, **bad)
    for bad in (b[:1], b[None]):
        with pytest.raises(ValueError):
            ops.linear_lora(x, w, bad, **kw)
    ops.linear_lora(x, w, b, gate=gate[:1], resid=resid, **kw)


def test_shapes_that_only_broadcast_are_refused():
    _shape_refusals("cpu", torch.float32)


@pytest.mark.gpu
def test_shapes_that_only_broadcast_are_refused_on_cuda(native):
    _shape_refusals("cuda", BF)
