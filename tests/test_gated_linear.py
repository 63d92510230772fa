"""The gated projection ``act(x Wg^T) * (x Wu^T)`` and its gradients against the formula in 64 bits."""

import pytest
import torch
import torch.nn.functional as TF

from difflet_b200 import ops
from difflet_b200.ops import fused as F

BF, HF = torch.bfloat16, torch.float16
ACTS = ("silu", "gelu", "gelu_erf")


def _make(M, K, N, dtype, device, seed=0, lead=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(device, dtype)  # noqa: E731
    return r(*(lead or (M,)), K), r(N, K, std=1.5 * K ** -0.5), r(N, K, std=K ** -0.5), r(*(lead or (M,)), N)


def _act(g, act):
    """act(g) and its derivative, written out."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if act == "gelu_erf":
        s = 0.5 * torch.erfc(-g / 2 ** 0.5)
        return g * s, s + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _check(got, want, tol, name):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def _forward_tol(x, wg, wu, act, dtype):
    """The result's rounding, the f32 sums (2^-23 a step where the adder truncates; |act'| < 1.13) and the activation in f32 (its
    exponential is off by a few units of 2^-24 for each unit of an argument below 64: 2^-16)."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    a, _ = _act(g, act)
    step = x.shape[-1] * 2.0 ** -23
    eg, eu = step * (x.abs() @ wg.abs().t()), step * (x.abs() @ wu.abs().t())
    r = torch.finfo(dtype).eps / 2
    least = torch.finfo(dtype).smallest_normal * r
    sums = 1.13 * eg * u.abs() + a.abs() * eu + eg * eu + 2.0 ** -16 * (a * u).abs()
    return a * u, (1 + r) * sums + r * (a * u).abs() + least


def _grad_tols(x, wg, wu, dh, act, dtype):
    """Gradients and bounds: g and u are kept rounded (r each; |act'| < 1.13, |act''| < 1.2), dg and du are rounded (r), then
    the sums over their products in f32 and the results' rounding."""
    x, wg, wu, dh = (t.double() for t in (x.reshape(-1, x.shape[-1]), wg, wu, dh.reshape(-1, dh.shape[-1])))
    g, u = x @ wg.t(), x @ wu.t()
    a, d = _act(g, act)
    dg, du = dh * u * d, dh * a
    fi = torch.finfo(dtype)
    r, least = fi.eps / 2, fi.smallest_normal * fi.eps / 2
    step = x.shape[1] * 2.0 ** -23
    eg, eu = step * (x.abs() @ wg.abs().t()) * (1 + r) + r * g.abs() + least, step * (x.abs() @ wu.abs().t()) * (1 + r) + r * u.abs() + least
    f = 2.0 ** -16
    e_dg = dh.abs() * ((u.abs() + eu) * (d.abs() * f + 1.2 * eg * (1 + f)) + eu * d.abs())
    e_du = dh.abs() * (a.abs() * f + 1.13 * eg * (1 + f))
    e_dg, e_du = e_dg * (1 + r) + r * dg.abs() + least, e_du * (1 + r) + r * du.abs() + least
    M, N = dg.shape
    out = {}
    for name, want, err, size, n in (
            ("dx", dg @ wg + du @ wu, e_dg @ wg.abs() + e_du @ wu.abs(), (dg.abs() + e_dg) @ wg.abs() + (du.abs() + e_du) @ wu.abs(), 2 * N),
            ("dwg", dg.t() @ x, e_dg.t() @ x.abs(), (dg.abs() + e_dg).t() @ x.abs(), M),
            ("dwu", du.t() @ x, e_du.t() @ x.abs(), (du.abs() + e_du).t() @ x.abs(), M)):
        err = err + n * 2.0 ** -23 * size
        out[name] = (want, err * (1 + r) + r * want.abs() + least)
    return out


# ----------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("act", ACTS + ("gelu_tanh",))
def test_oracle_and_gradients_on_cpu(act):
    x, wg, wu, dh = _make(5, 24, 13, torch.float64, "cpu")
    want = _act(x @ wg.t(), "gelu" if act == "gelu_tanh" else act)[0] * (x @ wu.t())
    assert torch.allclose(ops.gated_linear(x, wg, wu, act=act), want, rtol=1e-12, atol=1e-12)
    for t in (x, wg, wu):
        t.requires_grad_()
    assert torch.autograd.gradcheck(lambda *t: ops.gated_linear(*t, act=act), (x, wg, wu))
    got = torch.autograd.grad(ops.gated_linear(x, wg, wu, act=act), (x, wg, wu), dh)
    for name, t in zip(("dx", "dwg", "dwu"), got):
        want, _ = _grad_tols(x.detach(), wg.detach(), wu.detach(), dh, "gelu" if act == "gelu_tanh" else act, torch.float64)[name]
        assert torch.allclose(t, want, rtol=1e-10, atol=1e-12)


def test_shapes_and_refusals():
    x, wg, wu, _ = _make(6, 16, 9, torch.float32, "cpu", lead=(2, 3))
    assert ops.gated_linear(x, wg, wu).shape == (2, 3, 9)
    assert ops.gated_linear(x[:, :0], wg, wu).shape == (2, 0, 9)
    assert ops.gated_linear(x[0, 0], wg, wu).shape == (9,)
    with pytest.raises(ValueError):
        ops.gated_linear(x, wg, wu, act="tanh")
    with pytest.raises(ValueError):
        ops.gated_linear(x, wg, wu[:-1])
    with pytest.raises(ValueError):
        ops.gated_linear(x[..., :-1], wg, wu)
    with pytest.raises(ValueError):
        ops.gated_linear(x, wg, wu.to(BF))
    with pytest.raises(ValueError):
        ops.gated_linear(x.long(), wg.long(), wu.long())


# ----------------------------------------------------------------------------- kernels
SHAPES = [(1, 8, 1), (1, 64, 8), (4, 512, 1000), (7, 136, 65), (16, 1024, 333), (17, 40, 128), (33, 96, 129), (127, 256, 511), (129, 72, 64),
          (300, 1032, 257), (1000, 264, 1031), (2049, 64, 1280), (515, 2048, 2564), (70, 4096, 333), (257, 1024, 4099), (600, 520, 1), (40, 8, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_forward(native, M, K, N, dtype):
    x, wg, wu, _ = _make(M, K, N, dtype, "cuda")
    for act in ACTS:
        want, tol = _forward_tol(x, wg, wu, act, dtype)
        _check(ops.gated_linear(x, wg, wu, act=act), want, tol, act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gradients(native, M, K, N, dtype):
    x, wg, wu, dh = _make(M, K, N, dtype, "cuda")
    for act in ACTS:
        want = _grad_tols(x, wg, wu, dh, act, dtype)
        leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
        h = ops.gated_linear(*leaves, act=act)
        fw, tol = _forward_tol(x, wg, wu, act, dtype)
        _check(h.detach(), fw, tol, act)
        for name, t in zip(("dx", "dwg", "dwu"), torch.autograd.grad(h, leaves, dh)):
            assert t.dtype == dtype
            _check(t, *want[name], f"{act} {name}")


@pytest.mark.gpu
def test_gradient_against_differences(native):
    x, wg, wu, dh = _make(70, 128, 90, BF, "cuda")
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    got = torch.autograd.grad(ops.gated_linear(*leaves), leaves, dh)
    g = torch.Generator().manual_seed(9)
    tols = _grad_tols(x, wg, wu, dh, "silu", BF)
    for i, name in enumerate(("dx", "dwg", "dwu")):
        v = torch.randn(leaves[i].shape, generator=g).to("cuda", torch.float64)

        def loss(e):
            t = [u.double() for u in (x, wg, wu)]
            t[i] = t[i] + e * v
            return (F.gated_linear(*t) * dh.double()).sum()

        step = 1e-4  # (a third derivative times step^2: 1e-8 of the sum's size)
        want = (loss(step) - loss(-step)) / (2 * step)
        bound = (tols[name][1] * v.abs()).sum() + 1e-5 * (tols[name][0] * v).abs().sum()
        assert abs(float((got[i].double() * v).sum() - want)) <= float(bound)


@pytest.mark.gpu
@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)])
def test_some_gradients_only(native, need):
    x, wg, wu, dh = _make(65, 128, 130, BF, "cuda")
    full = [t.clone().requires_grad_() for t in (x, wg, wu)]
    want = torch.autograd.grad(ops.gated_linear(*full), full, dh)
    some = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, wg, wu), need)]
    got = torch.autograd.grad(ops.gated_linear(*some), [t for t in some if t.requires_grad], dh)
    assert all(torch.equal(a, b) for a, b in zip(got, [w for w, n in zip(want, need) if n]))


@pytest.mark.gpu
def test_layouts(native):
    """Rows of any pitch and start, one tensor that holds both weights, leading axes, gradients that are broadcast."""
    x, wg, wu, dh = _make(40, 64, 72, BF, "cuda")
    want = ops.gated_linear(x, wg, wu)
    both = torch.cat([wg, wu])
    assert torch.equal(ops.gated_linear(x, *both.chunk(2)), want)
    assert torch.equal(ops.gated_linear(x.view(5, 8, 64).transpose(0, 1).contiguous().transpose(0, 1), wg, wu).reshape(40, 72), want)
    assert torch.equal(ops.gated_linear(x.t().contiguous().t(), wg.t().contiguous().t(), wu), want)
    wide = torch.zeros(40, 200, device="cuda", dtype=BF)
    for off in (0, 8, 3):
        wide[:, off:off + 64] = x
        assert torch.equal(ops.gated_linear(wide[:, off:off + 64], wg, wu), want)
    odd = torch.zeros(1 + wg.numel(), device="cuda", dtype=BF)[1:].view(72, 64)
    odd.copy_(wg)
    assert torch.equal(ops.gated_linear(x, odd, wu), want)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]
    a = torch.autograd.grad(ops.gated_linear(*leaves).sum(), leaves)
    b = torch.autograd.grad(ops.gated_linear(*leaves), leaves, torch.ones_like(want))
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    col = dh[:, :1].expand(40, 72)
    a = torch.autograd.grad(ops.gated_linear(*leaves), leaves, col)
    b = torch.autograd.grad(ops.gated_linear(*leaves), leaves, col.contiguous())
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    same = x.new_empty(40, 72)[:, :].copy_(dh).t().contiguous().t()
    a = torch.autograd.grad(ops.gated_linear(*leaves), leaves, same)
    b = torch.autograd.grad(ops.gated_linear(*leaves), leaves, dh)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    one = x.new_zeros(3, 3, 64)
    assert torch.equal(ops.gated_linear(one[:, 1], wg, wu), torch.zeros(3, 72, device="cuda", dtype=BF))


@pytest.mark.gpu
def test_off_the_kernel(native):
    """Widths and types without a kernel, no rows, tangents: torch operations or an empty result."""
    x, wg, wu, _ = _make(9, 20, 12, BF, "cuda")
    assert torch.equal(ops.gated_linear(x, wg, wu), F.gated_linear(x, wg, wu))
    x, wg, wu, dh = _make(9, 32, 12, torch.float32, "cuda")
    assert torch.equal(ops.gated_linear(x, wg, wu), F.gated_linear(x, wg, wu))
    x, wg, wu = (t.to(BF).requires_grad_() for t in (x, wg, wu))
    none = torch.autograd.grad(ops.gated_linear(x[:0], wg, wu), (wg, wu), dh.to(BF)[:0])
    assert ops.gated_linear(x[:0], wg, wu).shape == (0, 12) and not any(bool(t.any()) for t in none)
    assert ops.gated_linear(x, wg[:0], wu[:0]).shape == (9, 0)
    a, b = (t.detach() for t in (wg, wu))
    y, t = torch.func.jvp(lambda v: ops.gated_linear(v, a, b), (x.detach(),), (x.detach(),))
    assert y.shape == t.shape == (9, 12) and bool((t != 0).any())
    v = torch.func.vmap(lambda v: ops.gated_linear(v, a, b))(x.detach())
    assert v.shape == (9, 12)
    with pytest.raises(ValueError):
        ops.gated_linear(x, wg.cpu(), wu.cpu())


@pytest.mark.gpu
def test_infinities_stay_in_their_rows(native):
    x, wg, wu, _ = _make(140, 64, 90, BF, "cuda")
    want = ops.gated_linear(x, wg, wu)
    x2 = x.clone()
    x2[3] = float("nan")
    x2[130, 5] = float("inf")
    got = ops.gated_linear(x2, wg, wu)
    keep = torch.ones(140, dtype=torch.bool, device="cuda")
    keep[[3, 130]] = False
    assert torch.equal(got[keep], want[keep]) and bool(got[3].isnan().all())
    big = torch.full((1, 64), 30.0, device="cuda", dtype=BF)  # g = -+ 1920: far tails are 0 or u
    h = ops.gated_linear(big, torch.full((8, 64), -1.0, device="cuda", dtype=BF), torch.ones(8, 64, device="cuda", dtype=BF))
    assert bool((h == 0).all())


@pytest.mark.gpu
def test_repeatable_and_captured(native):
    x, wg, wu, dh = _make(150, 256, 300, BF, "cuda")
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu)]

    def step():
        h = ops.gated_linear(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        leaves[0].copy_(x.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    new = step()
    assert all(torch.equal(a, b) for a, b in zip(got, new)) and not torch.equal(got[0], want[0])


@pytest.mark.gpu
def test_backward_twice_and_refused_second_order(native):
    x, wg, wu, dh = _make(20, 64, 48, BF, "cuda")
    x.requires_grad_()
    h = ops.gated_linear(x, wg, wu)
    a = torch.autograd.grad(h, x, dh, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(h, x, dh)[0])
    with pytest.raises(RuntimeError):
        g = torch.autograd.grad(ops.gated_linear(x, wg, wu), x, dh.clone().requires_grad_(), create_graph=True)[0]
        torch.autograd.grad(g.sum(), x)


def test_matches_torch_module_form():
    """The form that encoder checkpoints use: down(act(gate(x)) * up(x))."""
    x, wg, wu, _ = _make(6, 32, 24, torch.float32, "cpu")
    want = TF.silu(TF.linear(x, wg)) * TF.linear(x, wu)
    assert torch.allclose(ops.gated_linear(x, wg, wu), want, atol=1e-5)
