"""The scaled embedding lookup and the table's gradient against the formula in 64 bits."""

import pytest
import torch

from difflet_b200 import _native, ops
from difflet_b200.ops import fused as F

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _make(n, V, D, dtype, device, kind="uniform", seed=0):
    g = torch.Generator().manual_seed(seed)
    w = (0.5 * torch.randn(V, D, generator=g)).to(device, dtype)
    dy = torch.randn(n, D, generator=g).to(device, dtype)
    ids = torch.randint(0, V, (n,), generator=g)
    if kind == "one":
        ids[:] = V // 2
    elif kind == "skewed":  # few ids hold most tokens
        ids = (torch.rand(n, generator=g, dtype=torch.float64).pow(8) * V).long().clamp(max=V - 1)
    elif kind == "runs":
        ids = (torch.arange(n) // 33).clamp(max=V - 1)
    return ids.to(device), w, dy


def _grad(ids, dy, V, scale, pad=-1):
    """The gradient, the sum of its terms' sizes and the number of terms of each row."""
    real = ids != pad
    z = torch.zeros(V, dy.shape[1], dtype=torch.float64, device=dy.device)
    want = z.clone().index_add_(0, ids[real], dy[real].double()) * scale
    size = z.index_add_(0, ids[real], dy[real].double().abs()) * abs(scale)
    return want, size, torch.bincount(ids[real], minlength=V)[:, None]


def _check_grad(got, ids, dy, scale, pad=-1):
    """Sums of c terms in f32 (2^-24 a term), the product with the scale (f32 itself rounded) and the rounding to the type."""
    want, size, c = _grad(ids, dy, got.shape[0], scale, pad)
    r = torch.finfo(got.dtype).eps / 2
    tol = (c + 2) * 2.0 ** -24 * size * (1 + r) + r * want.abs() + torch.finfo(got.dtype).smallest_normal * r
    assert got.dtype == dy.dtype and bool(((got.double() - want).abs() <= tol).all())
    assert bool((got[(c == 0)[:, 0]] == 0).all())


# ----------------------------------------------------------------------------- CPU
def test_lookup_and_gradient_on_cpu():
    ids, w, dy = _make(40, 13, 7, torch.float64, "cpu")
    ids = ids.view(5, 8)
    assert torch.equal(ops.embedding(ids, w, scale=3.0), w[ids] * 3.0)
    w.requires_grad_()
    assert torch.autograd.gradcheck(lambda t: ops.embedding(ids, t, scale=3.0), (w,))
    got = torch.autograd.grad(ops.embedding(ids, w, scale=3.0, padding_idx=-12), w, dy.view(5, 8, 7))[0]
    want, _, _ = _grad(ids.reshape(-1), dy, 13, 3.0, 1)
    assert torch.allclose(got, want) and not bool(got[1].any())
    assert torch.allclose(F.embedding_grad(dy, ids, 13, 3.0, 1), want)


def test_refusals():
    ids, w, _ = _make(6, 9, 4, FF, "cpu")
    assert ops.embedding(ids.int()[:0], w).shape == (0, 4) and ops.embedding(ids[0], w).shape == (4,)
    for bad in (lambda: ops.embedding(ids.float(), w), lambda: ops.embedding(ids > 2, w), lambda: ops.embedding(ids, w[0]),
                lambda: ops.embedding(ids, w.long()), lambda: ops.embedding(ids, w, padding_idx=9),
                lambda: ops.embedding(ids, w, padding_idx=-10)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(IndexError):
        ops.embedding(ids + 100, w)


# ----------------------------------------------------------------------------- kernels
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (3, 5, 8), (77, 1000, 771), (1000, 33, 4096), (600, 7, 24), (33000, 600, 40), (5, 256384, 16)])
def test_lookup(native, n, V, D, dtype):
    ids, w, _ = _make(n, V, D, dtype, "cuda")
    for scale in (1.0, D ** 0.5, -0.3):
        want = w.double()[ids] * scale
        got = ops.embedding(ids, w, scale=scale)
        r = torch.finfo(dtype).eps / 2
        # the factor and the product in f32, then the type
        tol = (r + 2.0 ** -22) * want.abs() + torch.finfo(dtype).smallest_normal * r
        assert got.dtype == dtype and bool(((got.double() - want).abs() <= tol).all())
        assert torch.equal(got, ops.embedding(ids.int(), w, scale=scale))
    assert torch.equal(ops.embedding(ids, w), w[ids])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("kind", ["uniform", "one", "skewed", "runs"])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (5, 3, 8), (64, 2, 264), (65, 2, 33), (616, 5000, 771), (4097, 100, 512), (20000, 12, 72), (9000, 30000, 64), (30000, 60, 8), (70000, 150, 4)])
def test_gradient(native, n, V, D, kind, dtype):
    ids, w, dy = _make(n, V, D, dtype, "cuda", kind)
    w.requires_grad_()
    for scale, pad in ((1.0, None), (D ** 0.5, V // 2)):
        y = ops.embedding(ids, w, scale=scale, padding_idx=pad)
        got = torch.autograd.grad(y, w, dy)[0]
        _check_grad(got, ids, dy, scale, -1 if pad is None else pad)
        again = torch.autograd.grad(ops.embedding(ids.int(), w, scale=scale, padding_idx=pad), w, dy)[0]
        assert torch.equal(got, again)  # no atomic's order shows


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, FF])
@pytest.mark.parametrize("D", [2, 6, 12, 255, 770, 772, 1030, 2052])
def test_widths(native, D, dtype):
    """Rows that pieces of 8, 4 or 2 bytes fit, and tables and gradients that start at any value."""
    ids, w, dy = _make(333, 90, D, dtype, "cuda", "skewed")
    want, grad = ops.embedding(ids, w, scale=0.7), F.embedding_grad(dy, ids, 90, 0.7)
    assert torch.equal(want, (w[ids].float() * 0.7).to(dtype))
    _check_grad(grad, ids, dy, 0.7)
    for off in (1, 2, 4):
        flat_w, flat_d = (torch.zeros(off + t.numel(), device="cuda", dtype=dtype)[off:].view(t.shape) for t in (w, dy))
        flat_w.copy_(w)
        flat_d.copy_(dy)
        assert torch.equal(ops.embedding(ids, flat_w, scale=0.7), want)
        assert torch.equal(F.embedding_grad(flat_d, ids, 90, 0.7), grad)


@pytest.mark.gpu
def test_gradient_of_many_tokens(native):
    """More tokens than one bitmap holds, of few ids: the order is found window by window."""
    n = 300_001
    ids, w, dy = _make(n, 3, 8, FF, "cuda")
    got = F.embedding_grad(dy, ids, 3)
    _check_grad(got, ids, dy, 1.0)
    assert torch.equal(got, F.embedding_grad(dy, ids, 3))


@pytest.mark.gpu
def test_sums_are_in_the_order_of_the_ids(native):
    """Up to 64 tokens of an id are added one after another, in ascending order."""
    ids, w, dy = _make(700, 20, 40, FF, "cuda")
    got = F.embedding_grad(dy, ids, 20)
    for v in range(20):
        s = torch.zeros(40, device="cuda")
        at = (ids == v).nonzero()[:, 0]
        assert 0 < len(at) <= 64
        for i in at.tolist():
            s += dy[i]
        assert torch.equal(got[v], s)


@pytest.mark.gpu
def test_layouts(native):
    ids, w, dy = _make(48, 30, 64, BF, "cuda")
    want = ops.embedding(ids, w, scale=2.0)
    assert torch.equal(ops.embedding(ids.view(4, 12).t(), w, scale=2.0), want.view(4, 12, 64).transpose(0, 1))
    wide = torch.zeros(30, 100, device="cuda", dtype=BF)
    for off in (0, 5, 8):
        wide[:, off:off + 64] = w
        assert torch.equal(ops.embedding(ids, wide[:, off:off + 64], scale=2.0), want)
    assert torch.equal(ops.embedding(ids, w.t().contiguous().t(), scale=2.0), want)
    assert torch.equal(ops.embedding(ids, w[:1].expand(30, 64), scale=2.0), w[:1].expand(48, 64) * 2)
    for small in (torch.int8, torch.int16, torch.uint8):
        assert torch.equal(ops.embedding(ids.to(small), w, scale=2.0), want)
    w.requires_grad_()
    a = torch.autograd.grad(ops.embedding(ids, w).sum(), w)[0]
    b = torch.autograd.grad(ops.embedding(ids, w), w, torch.ones_like(dy))[0]
    assert torch.equal(a, b)
    odd = torch.zeros(1 + dy.numel(), device="cuda", dtype=BF)[1:].view(48, 64)
    odd.copy_(dy)
    for d in (odd, dy.t().contiguous().t()):
        assert torch.equal(torch.autograd.grad(ops.embedding(ids, w), w, d)[0], torch.autograd.grad(ops.embedding(ids, w), w, dy)[0])


@pytest.mark.gpu
def test_empty(native):
    ids, w, dy = _make(4, 6, 8, BF, "cuda")
    w.requires_grad_()
    y = ops.embedding(ids[:0], w)
    assert y.shape == (0, 8) and not bool(torch.autograd.grad(y, w, dy[:0])[0].any())
    assert ops.embedding(ids, w[:, :0]).shape == (4, 0)


@pytest.mark.gpu
def test_ids_outside_the_table(native):
    """Zeros and no gradient for them, and the device error word says so."""
    ids, w, dy = _make(50, 20, 72, BF, "cuda")
    torch.cuda.synchronize()
    _native.check_device_errors()
    bad = ids.clone()
    bad[3], bad[7], bad[11] = -1, 20, 2 ** 40
    got = ops.embedding(bad, w, scale=3.0)
    torch.cuda.synchronize()
    from difflet_b200.utils.errors import DeviceError

    with pytest.raises(DeviceError):
        _native.check_device_errors()
    keep = torch.ones(50, dtype=torch.bool, device="cuda")
    keep[[3, 7, 11]] = False
    assert not bool(got[~keep].any()) and torch.equal(got[keep], ops.embedding(ids, w, scale=3.0)[keep])
    _check_grad(F.embedding_grad(dy, bad, 20), ids[keep], dy[keep], 1.0)
    _native.check_device_errors()


@pytest.mark.gpu
def test_off_the_kernel(native):
    ids, w, _ = _make(9, 12, 8, torch.float64, "cuda")
    assert torch.equal(ops.embedding(ids, w, scale=2.0), w[ids] * 2)
    w = w.float()
    y, t = torch.func.jvp(lambda v: ops.embedding(ids, v, scale=2.0), (w,), (w,))
    assert torch.equal(y, t)
    with pytest.raises(ValueError):
        ops.embedding(ids.cpu(), w)


@pytest.mark.gpu
def test_captured(native):
    ids, w, dy = _make(3000, 500, 128, BF, "cuda", "skewed")
    w.requires_grad_()

    def step():
        y = ops.embedding(ids, w, scale=2.0, padding_idx=1)
        return y.detach(), torch.autograd.grad(y, w, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    ids.copy_(ids.flip(0) // 2)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
    _check_grad(got[1], ids, dy, 2.0, 1)
