"""What ``ops.attention`` and ``ops.cross_attention`` accept: one meaning of a call on every device, type and path.

Kernel results are compared with the 64-bit formula and the tolerances of ``test_cross_attention``."""

import math

import pytest
import torch

from difflet_b200 import ops
from test_cross_attention import _check, _inputs, _ref

BOTH = (ops.attention, ops.cross_attention)


# ----------------------------------------------------------------------------- integer masks are added to the scores
def _int_mask(B, Sq, Sk, dtype, device):
    g = torch.Generator().manual_seed(4)
    low = -100 if dtype == torch.int8 else -10000
    return torch.where(torch.rand(B, 1, Sq, Sk, generator=g) < 0.6, 0, low).to(device, dtype)


@pytest.mark.parametrize("fn", BOTH)
@pytest.mark.parametrize("dtype", [torch.int8, torch.int32, torch.int64])
def test_integer_masks_are_additive(fn, dtype):
    q, k, v = _inputs(2, 4, 4, 6, 9, 16, torch.float32, "cpu")
    m = _int_mask(2, 6, 9, dtype, "cpu")
    want = fn(q, k, v, scale=0.25, attention_mask=m.float())
    assert torch.allclose(fn(q, k, v, scale=0.25, attention_mask=m), want, atol=1e-6)
    assert torch.allclose(want.double(), _ref(q, k, v, 0.25, m.float())[0], atol=1e-5)
    got = fn(q.clone().requires_grad_(), k, v, scale=0.25, attention_mask=m)
    assert torch.allclose(got.detach(), want, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("fn", BOTH)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Sq,D", [(3, 64), (150, 64), (150, 128)])
def test_integer_masks_are_additive_on_cuda(native, fn, dtype, Sq, D):
    q, k, v = _inputs(2, 4, 4, Sq, 70, D, dtype, "cuda")
    m = _int_mask(2, Sq, 70, torch.int32, "cuda")
    o = fn(q, k, v, scale=0.1, attention_mask=m)
    if dtype != torch.float32:  # the kernels; -10000 masks whatever the scores are
        _check(o, _ref(q, k, v, 0.1, m.float()), dtype, D, 70, v.abs().max().item())
    keep = fn(q, k, v, scale=0.1, attention_mask=m == 0)
    grad = fn(q.clone().requires_grad_(), k, v, scale=0.1, attention_mask=m).detach()
    for other in (keep, grad):  # the library's own roundings: a few of the largest value
        assert (o.double() - other.double()).abs().max() <= 4 * torch.finfo(dtype).eps * v.abs().max()


@pytest.mark.gpu
def test_masks_and_lengths_of_other_types(native):
    """Lengths of any integer type and device, f64 masks at their lowest value, a mask of no dimension, many batch rows, and
    the result in place of the queries."""
    B, H, Sq, Sk, D = 2, 2, 40, 50, 64
    q, k, v = _inputs(B, H, H, Sq, Sk, D, torch.bfloat16, "cuda")
    all_keys = ops.cross_attention(q, k, v, scale=0.1)
    for lens in (torch.tensor([1 << 40, 50]), torch.tensor([50, 99], dtype=torch.int16)):
        assert torch.equal(ops.cross_attention(q, k, v, scale=0.1, kv_lens=lens), all_keys)
    assert bool((ops.cross_attention(q, k, v, scale=0.1, kv_lens=torch.tensor([-3, 0])) == 0).all())
    m = torch.rand(B, 1, Sq, Sk, device="cuda") < 0.5
    want = ops.cross_attention(q, k, v, scale=0.1, attention_mask=m)
    low = torch.zeros(m.shape, device="cuda", dtype=torch.float64).masked_fill(~m, torch.finfo(torch.float64).min)
    low[:, :, 3] = torch.finfo(torch.float64).min  # a row at the lowest value everywhere: the mean of the values
    o = ops.cross_attention(q, k, v, scale=0.1, attention_mask=low)
    mean = v.double().mean(2)
    assert bool(((o[:, :, 3].double() - mean).abs() <= 2.0 ** -7 * (mean.abs() + v.double().abs().mean(2))).all())
    keep = torch.arange(Sq, device="cuda") != 3
    assert torch.allclose(o[:, :, keep].float(), want[:, :, keep].float(), atol=2.0 ** -6)
    assert torch.equal(ops.cross_attention(q, k, v, scale=0.1, attention_mask=torch.tensor(True, device="cuda")), all_keys)
    big = _inputs(70000, 1, 1, 1, 3, 64, torch.bfloat16, "cuda")  # more batch rows than a grid axis holds
    _check(ops.cross_attention(*big, scale=0.1), _ref(*big, 0.1), q.dtype, 64, 3, big[2].abs().max().item())
    same = q.contiguous()
    got = ops.cross_attention(same, k, v, scale=0.1, out=same)
    assert got is same and torch.equal(got, all_keys)


# ----------------------------------------------------------------------------- gradients
@pytest.mark.parametrize("fn", BOTH)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_inputs_that_ask_for_gradients_stay_off_the_kernels(fn, which):
    """Shapes and dispatch alone (tensors without data): no kernel is called, and the result has a history."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        qkv = [torch.empty(2, 2, 20, 128, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
        qkv[which].requires_grad_()
        o = fn(*qkv, scale=0.1)
        assert o.shape == qkv[0].shape and o.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("fn", BOTH)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", [None, "bounds", "mask"])
def test_gradients(native, fn, D, kind):
    q, k, v = (t.detach().requires_grad_() for t in _inputs(2, 2, 2, 20, 33, D, torch.bfloat16, "cuda"))
    keep = torch.ones(2, 1, 20, 33, device="cuda", dtype=torch.bool)
    kw = {}
    if kind == "bounds":
        hi = torch.tensor([33, 12], device="cuda").view(2, 1, 1, 1)
        kw = dict(bound_min=torch.zeros_like(hi), bound_max=hi)
        keep = keep & (torch.arange(33, device="cuda") < hi)
    elif kind == "mask":
        keep = (torch.rand(2, 1, 20, 33, device="cuda") < 0.7) | (torch.arange(33, device="cuda") == 0)
        kw = dict(attention_mask=keep)
    w = torch.randn(2, 2, 20, D, device="cuda")
    ref = [t.detach().double().requires_grad_() for t in (q, k, v)]
    z = (ref[0] @ ref[1].transpose(2, 3) * 0.1).masked_fill(~keep, -math.inf)
    want = torch.autograd.grad(((z.softmax(-1) @ ref[2]) * w.double()).sum(), ref)
    got = torch.autograd.grad((fn(q, k, v, scale=0.1, **kw) * w).sum(), (q, k, v))
    for a, b in zip(got, want):  # the library's bf16 products: a few roundings (2^-8) of the largest value
        assert (a.double() - b).abs().max() <= 2.0 ** -5 * b.abs().max()


# ----------------------------------------------------------------------------- shapes
def _wide(B, H, Hk, Sq, Sk, D, Dv, dtype, device):
    q, k, _ = _inputs(B, H, Hk, Sq, Sk, D, dtype, device)
    return q, k, _inputs(B, H, Hk, Sq, Sk, Dv, dtype, device, 1)[2]


@pytest.mark.parametrize("Hk", [4, 2])
def test_values_of_another_width(Hk):
    q, k, v = _wide(2, 4, Hk, 6, 9, 16, 24, torch.float32, "cpu")
    lens = torch.tensor([9, 3])
    m = torch.rand(2, 1, 6, 9) < 0.6
    for kw, ref in (({}, {}), (dict(attention_mask=m), dict(mask=m)), (dict(kv_lens=lens), dict(lens=lens))):
        want = _ref(q, k, v, 0.25, **ref)[0]
        o, out = ops.cross_attention(q, k, v, scale=0.25, **kw), torch.empty(2, 4, 6, 24)
        assert o.shape == (2, 4, 6, 24) and torch.allclose(o.double(), want, atol=1e-5)
        assert torch.equal(ops.cross_attention(q, k, v, scale=0.25, out=out, **kw), o) and torch.equal(out, o)
    with pytest.raises(ValueError):
        ops.cross_attention(q, k, v, out=torch.empty_like(q))
    if Hk == 4:
        assert torch.allclose(ops.attention(q, k, v, scale=0.25, attention_mask=m).double(), _ref(q, k, v, 0.25, m)[0], atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,Dv", [(64, 32), (64, 128), (128, 64), (48, 64)])
def test_values_of_another_width_on_cuda(native, D, Dv, dtype):
    q, k, v = _wide(2, 4, 4, 30, 41, D, Dv, dtype, "cuda")
    m = torch.rand(2, 1, 30, 41, device="cuda") < 0.6
    lens = torch.tensor([41, 7], device="cuda")
    for fn in BOTH:
        for kw in ({}, dict(mask=m)):
            o = fn(q, k, v, scale=0.1, attention_mask=kw.get("mask"))
            want, _, size, _ = _ref(q, k, v, 0.1, **kw)
            assert o.shape == want.shape  # the library's form: P and the result in the type
            assert bool(((o.double() - want).abs() <= 2 * torch.finfo(dtype).eps * (size + want.abs()) + 1e-6).all())
    o = ops.cross_attention(q, k, v, scale=0.1, kv_lens=lens, out=torch.empty(2, 4, 30, Dv, device="cuda", dtype=dtype))
    want, _, size, _ = _ref(q, k, v, 0.1, lens=lens)
    assert bool(((o.double() - want).abs() <= 2 * torch.finfo(dtype).eps * (size + want.abs()) + 1e-6).all())


SHARED = [((1, 4), (3, 4)), ((3, 4), (1, 4)), ((3, 4), (1, 1)), ((3, 1), (3, 4)), ((1, 1), (3, 4))]


def _shared(q_rows, k_rows, device, dtype, D=16, Sq=6, Sk=9):
    """q, k, v of one batch row or head for all of the other side, and q, k, v written out."""
    q, k, v = _inputs(3, 4, 4, Sq, Sk, D, dtype, device)
    q, k, v = (t[:r[0], :r[1]] for t, r in zip((q, k, v), (q_rows, k_rows, k_rows)))
    return (q, k, v), [t.expand(3, 4, *t.shape[2:]) for t in (q, k, v)]


@pytest.mark.parametrize("rows", SHARED)
def test_one_batch_row_or_head_for_all(rows):
    (q, k, v), (fq, fk, fv) = _shared(*rows, "cpu", torch.float32)
    m = torch.rand(3, 1, 6, 9) < 0.6
    lens = torch.tensor([9, 3, 0])
    for kw, ref in (({}, {}), (dict(attention_mask=m), dict(mask=m)), (dict(kv_lens=lens), dict(lens=lens))):
        o = ops.cross_attention(q, k, v, scale=0.25, **kw)
        assert o.shape == (3, 4, 6, 16) and torch.allclose(o.double(), _ref(fq, fk, fv, 0.25, **ref)[0], atol=1e-5)
    for bad in (((q[:, :, :, :8], k, v)), ((fq[:2], fk, fv)), ((fq, fk[:, :3], fv[:, :3])), ((fq, fk[:1, :2], fv[:1, :2]))):
        with pytest.raises(ValueError):
            ops.cross_attention(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", SHARED)
def test_one_batch_row_or_head_for_all_on_cuda(native, rows, D):
    (q, k, v), (fq, fk, fv) = _shared(*rows, "cuda", torch.bfloat16, D, 40, 70)
    m = torch.rand(3, 1, 40, 70, device="cuda") < 0.6
    vmax = v.abs().max().item()
    for kw, ref in (({}, {}), (dict(attention_mask=m), dict(mask=m)), (dict(kv_lens=torch.tensor([70, 9, 0], device="cuda")),) * 2):
        lse = torch.empty(3, 4, 40, device="cuda")
        o = ops.cross_attention(q, k, v, scale=0.1, lse=lse, **kw)
        _check(o, _ref(fq, fk, fv, 0.1, ref.get("mask"), ref.get("kv_lens")), q.dtype, D, 70, vmax, lse)
    if rows in (((3, 4), (1, 4)), ((1, 4), (3, 4))):  # as ``attention`` takes them
        o = ops.attention(q, k, v, scale=0.1, attention_mask=m)
        want, _, size, _ = _ref(fq, fk, fv, 0.1, m)
        assert bool(((o.double() - want).abs() <= 2 * torch.finfo(q.dtype).eps * (size + want.abs()) + 1e-6).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fn", BOTH)
def test_masks_of_the_host(native, fn):
    q, k, v = _inputs(2, 4, 4, 40, 70, 64, torch.bfloat16, "cuda")
    g = torch.Generator().manual_seed(0)
    for m in (torch.rand(2, 1, 40, 70, generator=g) < 0.6, torch.randn(70, generator=g), torch.randn(40, 70, generator=g).bfloat16()):
        assert torch.equal(fn(q, k, v, scale=0.1, attention_mask=m), fn(q, k, v, scale=0.1, attention_mask=m.cuda()))


# ----------------------------------------------------------------------------- tensors without data, transforms
def test_meta_tensors():
    q, k, v = _inputs(2, 4, 4, 6, 9, 16, torch.float32, "meta")
    m, lens = torch.ones(2, 1, 1, 9, dtype=torch.bool, device="meta"), torch.ones(2, dtype=torch.long, device="meta")
    for kw in ({}, dict(attention_mask=m), dict(attention_mask=m.float()), dict(kv_lens=lens)):
        o = ops.cross_attention(q, k[:, :2], v[:, :2], **kw)
        assert o.shape == q.shape and o.is_meta
    x, mod = torch.empty(6, 32, device="meta"), torch.empty(2, 32, device="meta")
    y, s = ops.add_rms_norm(x, x, scale=mod, shift=mod, rows_per_batch=3)
    assert y.shape == s.shape == x.shape and y.is_meta


def test_fake_tensors():
    """Tracing sees the library path: no kernel is given a tensor without data."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
        for D in (64, 128):
            q, k, v = e(2, 4, 6, D), e(2, 4, 9, D), e(2, 4, 9, D)
            for fn in BOTH:
                for m in (e(6, 9, dtype=torch.bool), e(2, 1, 1, 9)):
                    o = fn(q, k, v, attention_mask=m)
                    assert o.shape == q.shape and o.is_cuda
            o = ops.cross_attention(q, k[:, :2], v[:, :2], kv_lens=e(2, dtype=torch.int32))
            assert o.shape == q.shape and o.is_cuda
        o = ops.dequantize_mx(e(4, 64, dtype=torch.float8_e4m3fn), e(4, 2, dtype=torch.uint8))
        assert o.shape == (4, 64) and o.is_cuda


def test_forward_mode_is_refused_where_no_tangent_is_carried():
    import torch.autograd.forward_ad as fwAD

    x = torch.randn(3, 32)
    bank = ops.LoraBank([torch.randn(4, 32)], [torch.randn(24, 4)])
    with fwAD.dual_level():
        d = fwAD.make_dual(x, torch.randn(3, 32))
        with pytest.raises(RuntimeError, match="no backward"):
            ops.add_rms_norm(d)
        with pytest.raises(RuntimeError, match="no backward"):
            ops.linear_lora(d, torch.randn(24, 32), bank=bank, ids=torch.zeros(3, dtype=torch.long))
        ops.add_rms_norm(x)


@pytest.mark.gpu
@pytest.mark.parametrize("fn", BOTH)
def test_transforms_and_tangents(native, fn):
    import torch.autograd.forward_ad as fwAD

    q, k, v = _inputs(2, 4, 4, 20, 33, 64, torch.bfloat16, "cuda")
    m = torch.rand(20, 33, device="cuda") < 0.7
    m[:, 0] = True
    call = lambda q, k, v: fn(q, k, v, scale=0.1, attention_mask=m)  # noqa: E731
    want, _, size, _ = _ref(q, k, v, 0.1, m)
    got = torch.vmap(call)(*(torch.stack([t, t]) for t in (q, k, v)))
    assert bool(((got[1].double() - want).abs() <= 2 * torch.finfo(q.dtype).eps * (size + want.abs())).all())
    t = torch.randn_like(q)
    f64 = lambda q: ((q @ k.double().transpose(2, 3) * 0.1).masked_fill(~m, -math.inf)).softmax(-1) @ v.double()  # noqa: E731
    _, ref = torch.func.jvp(f64, (q.double(),), (t.double(),))
    with torch.nn.attention.sdpa_kernel(torch.nn.attention.SDPBackend.MATH), fwAD.dual_level():
        tangent = fwAD.unpack_dual(call(fwAD.make_dual(q, t), k, v)).tangent
    assert tangent is not None  # bf16 throughout: a few roundings (2^-8) of the largest value
    assert (tangent.double() - ref).abs().max() <= 2.0 ** -5 * ref.abs().max()


# ----------------------------------------------------------------------------- excluded keys and empty rows off the kernels
def _excluded(kind, dtype, device, Sk=33):
    """Arguments that exclude keys, and which keys every batch row keeps."""
    n = torch.tensor([Sk, 12, 0], device=device)
    keep = torch.arange(Sk, device=device) < n[:, None]
    if kind == "lens":
        return dict(kv_lens=n), keep, torch.ones(1, 1, 20, Sk, dtype=torch.bool, device=device)
    if kind == "keys":
        keep = keep & (torch.arange(Sk, device=device) % 3 != 1)
        return dict(attention_mask=keep[:, None, None]), keep, torch.ones(1, 1, 20, Sk, dtype=torch.bool, device=device)
    own = torch.rand(1, 1, 20, Sk, generator=torch.Generator().manual_seed(0)).to(device) < 0.5
    own[:, :, 3] = False
    m = own if kind == "lens+bool" else torch.where(own, 0.0, -math.inf).to(dtype)
    return dict(kv_lens=n, attention_mask=m), keep, own


def _excluded_keys(kind, D, dtype, device, tol):
    q, k, v = _inputs(3, 4, 2, 20, 33, D, dtype, device)
    kw, keep, own = _excluded(kind, dtype, device)
    gone = ~keep[:, None, :, None]
    k, v = k.masked_fill(gone, math.nan).requires_grad_(), v.masked_fill(gone, math.inf).requires_grad_()
    q = q.detach().requires_grad_()
    lse = torch.empty(3, 4, 20, device=device)
    o = ops.cross_attention(q, k, v, scale=0.1, lse=lse, **kw)
    full = own & keep[:, None, None]
    some = full.any(-1, keepdim=True)
    ref = [t.detach().double().masked_fill(g, 0.0).requires_grad_() for t, g in ((q, torch.zeros_like(q).bool()), (k, gone), (v, gone))]
    z = (ref[0] @ ref[1].repeat_interleave(2, 1).transpose(2, 3) * 0.1).masked_fill(~full & some, -math.inf)
    want = z.softmax(-1) @ ref[2].repeat_interleave(2, 1) * some
    assert (o.double() - want).abs().max() <= tol * want.abs().max()
    lse_ref = torch.logsumexp(z, -1).masked_fill(~some[..., 0], -math.inf)
    assert torch.allclose(lse.double(), lse_ref, atol=10 * tol)
    w = torch.randn(want.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64).to(device)
    got = torch.autograd.grad((ops.cross_attention(q, k, v, scale=0.1, **kw).double() * w).sum(), (q, k, v))
    for a, b in zip(got, torch.autograd.grad((want * w).sum(), ref)):
        assert (a.double() - b).abs().max() <= tol * b.abs().max()
    out = torch.empty_like(o)
    with torch.no_grad():
        assert ops.cross_attention(q, k, v, scale=0.1, out=out, **kw) is out
    assert (out.double() - want).abs().max() <= tol * want.abs().max() and bool((out[2] == 0).all())


KINDS = ["lens", "keys", "lens+bool", "lens+bias"]


@pytest.mark.parametrize("kind", KINDS)
def test_excluded_keys_and_empty_rows(kind):
    _excluded_keys(kind, 16, torch.float32, "cpu", 2.0 ** -18)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype,tol", [(64, torch.float32, 2.0 ** -16), (40, torch.float32, 2.0 ** -16), (64, torch.bfloat16, 2.0 ** -5),
                                         (128, torch.bfloat16, 2.0 ** -5)])
@pytest.mark.parametrize("kind", KINDS)
def test_excluded_keys_and_empty_rows_off_the_kernels(native, kind, D, dtype, tol):
    """f32, other head dims and gradients take the library path on CUDA, with the same rules."""
    _excluded_keys(kind, D, dtype, "cuda", tol)


# ----------------------------------------------------------------------------- the library baseline
@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_library_baseline(native, monkeypatch, D):
    """DIFFLET_KERNEL_ATTN=sdpa: no attention entry launches a kernel of this framework, and the results agree."""
    from difflet_b200.ops import fused as F

    q, k, v = _inputs(2, 4, 2, 40, 70, D, torch.bfloat16, "cuda")
    fk, fv = (t.repeat_interleave(2, 1) for t in (k, v))
    m = torch.rand(2, 1, 40, 70, device="cuda") < 0.6
    lens = torch.tensor([70, 0], device="cuda")
    calls = [lambda: ops.cross_attention(q, k, v, scale=0.1), lambda: ops.cross_attention(q, k, v, scale=0.1, attention_mask=m),
             lambda: ops.cross_attention(q, k, v, scale=0.1, kv_lens=lens, attention_mask=m), lambda: ops.attention(q, fk, fv, scale=0.1),
             lambda: ops.attention(q, fk, fv, scale=0.1, attention_mask=m), lambda: F.attention(q, fk, fv, 0.1),
             lambda: ops.cross_attention(q[:, :, :2], k, v, scale=0.1, kv_lens=lens)]
    kernels = [f() for f in calls]
    monkeypatch.setenv("DIFFLET_KERNEL_ATTN", "sdpa")
    n = F.LAUNCHES[0]
    library = [f() for f in calls]
    assert F.LAUNCHES[0] == n
    for a, b in zip(kernels, library):  # both round P and the result
        assert (a.double() - b.double()).abs().max() <= 2.0 ** -6 * v.abs().max()


# ----------------------------------------------------------------------------- LSE and windows: f32 up to the result
def _check_precise(o, ref, dtype, D, Sk, vmax, lse=None):
    """As ``_check``, with P in two terms of the type: off by u^2 (u: half a step), in fp16 by 2^-25 absolutely."""
    want, lse_ref, size, bound = ref
    u = torch.finfo(dtype).eps / 2
    d = 2.0 ** -24 * (D + 4) * bound + 2.0 ** -20
    tol = (u * u + 2 * d) * size + u * want.abs() + 1e-30
    if dtype == torch.float16:
        tol = tol + Sk * 2.0 ** -25 * vmax + 2.0 ** -25
    err = (o.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol).nan_to_num(1e9).max().item():.3g} of the tolerance"
    if lse is not None:
        fine = torch.isfinite(lse_ref)
        assert torch.equal(fine, torch.isfinite(lse.double()))
        assert bool(((lse.double() - lse_ref).abs()[fine] <= d + 2.0 ** -20 * (1 + lse_ref.abs()[fine])).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,Sq,Sk,D", [(1, 1, 1, 1, 64), (2, 3, 5, 77, 64), (2, 4, 129, 128, 64), (2, 2, 501, 1024, 64), (3, 24, 1100, 130, 64),
                                         (2, 40, 300, 2000, 64), (1, 1, 3, 200, 128), (2, 3, 257, 129, 128), (3, 20, 600, 300, 128)])
def test_lse_and_windows_keep_f32(native, B, H, Sq, Sk, D, dtype):
    """Head dim 64 (and fp16) with LSE or a key window was f32 up to the result: P may not be rounded to the type once."""
    from difflet_b200.ops import fused as F
    from difflet_b200.ops.attn import attention_with_lse

    q, k, v = _inputs(B, H, H, Sq, Sk, D, dtype, "cuda", Sq + Sk)
    vmax = v.abs().max().item()
    lse = torch.empty(B, H, Sq, device="cuda")
    ref = _ref(q, k, v, D ** -0.5)
    if D == 64:
        _check_precise(F.attention(q, k, v, D ** -0.5, lse=lse), ref, dtype, D, Sk, vmax, lse)
        hi = torch.tensor([(Sk, 2 * Sk // 3, 0)[b] for b in range(B)], device="cuda", dtype=torch.int32)
        lo = (hi // 5).int()
        keep = (torch.arange(Sk, device="cuda") >= lo[:, None]) & (torch.arange(Sk, device="cuda") < hi[:, None])
        win = _ref(q, k, v, D ** -0.5, keep[:, None, None])
        clean = F.attention(q, k, v, D ** -0.5, kv_lo=lo, kv_hi=hi)
        _check_precise(clean, win, dtype, D, Sk, vmax)
        gone = ~keep[:, None, :, None]
        dirty = F.attention(q, k.masked_fill(gone, math.nan), v.masked_fill(gone, math.inf), D ** -0.5, kv_lo=lo, kv_hi=hi)
        assert torch.equal(dirty, clean)
    if D == 64 or dtype == torch.float16:
        o, lse = attention_with_lse(q, k, v, scale=D ** -0.5)
        _check_precise(o, ref, dtype, D, Sk, vmax, lse)
    m = torch.rand(B, 1, Sq, Sk, device="cuda") < 0.7
    lse = torch.empty(B, H, Sq, device="cuda")
    o = ops.attention(q, k, v, scale=D ** -0.5, attention_mask=m, lse=lse)
    _check_precise(o, _ref(q, k, v, D ** -0.5, m), dtype, D, Sk, vmax, lse)
    from difflet_b200 import _native

    _native.check_device_errors()


@pytest.mark.gpu
def test_precise_p_comes_without_a_mask(native):
    from difflet_b200.ops import fused as F

    q, k, v = _inputs(1, 2, 2, 3, 5, 64, torch.bfloat16, "cuda")
    with pytest.raises(ValueError):
        F.cross_attention(q, k, v, 1.0, mask=torch.ones(3, 5, device="cuda", dtype=torch.bool), precise_p=True)


# ----------------------------------------------------------------------------- LSE of any type and layout
def _lse_kinds(B, H, Sq, device):
    return [torch.empty(B, H, Sq, dtype=torch.float64, device=device), torch.empty(B, Sq, H, device=device).transpose(1, 2),
            torch.empty(B * H, Sq, dtype=torch.bfloat16, device=device), torch.empty(B, H, Sq, 2, device=device)[..., 1]]


def _any_lse(D, dtype, device):
    from difflet_b200.ops import fused as F

    B, H, Sq, Sk = 2, 4, 30, 41
    q, k, v = _inputs(B, H, H, Sq, Sk, D, dtype, device)
    m = torch.rand(B, 1, Sq, Sk, generator=torch.Generator().manual_seed(0)).to(device) < 0.7
    lens = torch.tensor([41, 7], device=device)
    calls = [lambda t: ops.cross_attention(q, k, v, scale=0.1, lse=t), lambda t: ops.cross_attention(q, k, v, scale=0.1, attention_mask=m, lse=t),
             lambda t: ops.cross_attention(q, k, v, scale=0.1, kv_lens=lens, lse=t), lambda t: ops.attention(q, k, v, scale=0.1, lse=t),
             lambda t: ops.attention(q, k, v, scale=0.1, attention_mask=m, lse=t), lambda t: F.attention(q, k, v, 0.1, lse=t)]
    for i, call in enumerate(calls if (D, dtype) != (128, torch.bfloat16) else calls[:3]):
        want = torch.empty(B, H, Sq, device=device)
        o = call(want)
        for t in _lse_kinds(B, H, Sq, device):
            if i in (3, 5) and t.dim() != 3:  # (plain attention takes the full shape)
                continue
            assert torch.equal(call(t), o) and torch.equal(t.reshape(B, H, Sq), want.to(t.dtype))
    for bad in (torch.empty(B, H, Sq + 1, device=device), torch.empty(B, H, 2, dtype=torch.float64, device=device)):
        with pytest.raises(ValueError):
            calls[0](bad)


def test_any_lse():
    _any_lse(16, torch.float32, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16), (64, torch.float32)])
def test_any_lse_on_cuda(native, D, dtype):
    _any_lse(D, dtype, "cuda")


# ----------------------------------------------------------------------------- lengths and bounds past the ends
def _past_the_ends(D, dtype, device):
    q, k, v = _inputs(2, 4, 4, 6, 9, D, dtype, device)
    big = torch.iinfo(torch.int64).max
    same = lambda a, b: torch.equal(a, b)  # noqa: E731
    every = ops.cross_attention(q, k, v, scale=0.25, kv_lens=torch.tensor([9, 9], device=device))
    for lens in (torch.tensor([1 << 40, big]), torch.tensor([(1 << 32) + 3, 1 << 31]), torch.tensor([9, 127], dtype=torch.int8)):
        assert same(ops.cross_attention(q, k, v, scale=0.25, kv_lens=lens.to(device)), every)
    assert bool((ops.cross_attention(q, k, v, scale=0.25, kv_lens=torch.tensor([-big, -(1 << 32) + 5], device=device)) == 0).all())
    edge = lambda *n: torch.tensor(n, device=device).view(2, 1, 1, 1)  # noqa: E731
    want = ops.cross_attention(q, k, v, scale=0.25, bound_min=edge(2, 0), bound_max=edge(9, 9))
    for lo, hi in ((edge(2, -big), edge(big, 1 << 32)), (edge(1.5, -0.5), edge(8.5, 1e30))):
        assert same(ops.cross_attention(q, k, v, scale=0.25, bound_min=lo, bound_max=hi), want)
        if q.is_cuda:
            m = (torch.arange(9, device=device) >= edge(2, 0)) & (torch.arange(9, device=device) < 9)
            o = ops.attention(q, k, v, scale=0.25, bound_min=lo, bound_max=hi)
            assert (o.double() - _ref(q, k, v, 0.25, m)[0]).abs().max() <= 2 * torch.finfo(dtype).eps * v.abs().max()
    with pytest.raises(ValueError):
        ops.cross_attention(q, k, v, kv_lens=torch.tensor([True, False], device=device))


def test_lengths_and_bounds_past_the_ends():
    _past_the_ends(16, torch.float32, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16), (40, torch.bfloat16), (64, torch.float32)])
def test_lengths_and_bounds_past_the_ends_on_cuda(native, D, dtype):
    _past_the_ends(D, dtype, "cuda")


@pytest.mark.gpu
def test_the_binding_refuses_what_it_would_not_differentiate(native, monkeypatch):
    from difflet_b200.ops import fused as F

    q, k, v = _inputs(1, 2, 2, 3, 5, 64, torch.bfloat16, "cuda")
    n = F.LAUNCHES[0]
    with pytest.raises(ValueError):
        F.cross_attention(q.clone().requires_grad_(), k, v, 1.0)
    monkeypatch.setenv("DIFFLET_KERNEL_ATTN", "sdpa")
    with pytest.raises(ValueError):
        F.cross_attention(q, k, v, 1.0)
    assert F.LAUNCHES[0] == n  # (a refused call is no launch)
    monkeypatch.delenv("DIFFLET_KERNEL_ATTN")
    F.cross_attention(q, k, v, 1.0)
    assert F.LAUNCHES[0] == n + 1


# ----------------------------------------------------------------------------- layouts
@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 200])
@pytest.mark.parametrize("off", [1, 3, 4])
def test_contiguous_from_an_odd_start(native, Sq, off):
    """Contiguous q, k, v and out that start where no copy engine can address them."""
    q, k, v = (t.contiguous() for t in _inputs(2, 4, 2, Sq, 300, 64, torch.bfloat16, "cuda"))
    want = ops.cross_attention(q, k, v, scale=0.1)

    def moved(t):
        u = torch.empty(t.numel() + off, device="cuda", dtype=t.dtype)[off:].view(t.shape)
        return u.copy_(t)

    for args in ((moved(q), k, v), (q, moved(k), v), (q, k, moved(v)), (moved(q), moved(k), moved(v))):
        assert torch.equal(ops.cross_attention(*args, scale=0.1), want)
    out = moved(torch.zeros_like(q))
    assert ops.cross_attention(q, k, v, scale=0.1, out=out) is out and torch.equal(out, want)
    one = torch.empty(3, 64 + off, device="cuda", dtype=q.dtype)[:1, :64].view(1, 1, 1, 64).copy_(q[:1, :1, :1])
    assert torch.equal(ops.cross_attention(one, k[:1, :1], v[:1, :1], scale=0.1), ops.cross_attention(q[:1, :1, :1], k[:1, :1], v[:1, :1], scale=0.1))


# ----------------------------------------------------------------------------- lengths beside masks
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["bool", "bias", "bias32", "key bias", "keys"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", [(4, 32, 4, 94, 1429, 128), (3, 12, 3, 473, 1402, 128), (2, 48, 6, 123, 1231, 128), (3, 12, 12, 700, 900, 128),
                                            (4, 32, 8, 104, 906, 64), (2, 6, 2, 5, 3000, 128)])
def test_lengths_beside_masks(native, B, H, Hk, Sq, Sk, D, kind, dtype):
    """Both exclude keys; many key tiles for one query tile a CTA, whose copies land in any order."""
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, dtype, "cuda")
    lens = torch.tensor([Sk, Sk // 2, 1, 0][:B], device="cuda")
    if kind == "key bias":
        m = torch.randn(1, Sk, generator=torch.Generator().manual_seed(0)).to("cuda", dtype)
    else:
        from test_cross_attention import _mask

        m = _mask(kind, B, H, Sq, Sk, "cuda", dtype)
    gone = (torch.arange(Sk, device="cuda") >= lens[:, None])[:, None, :, None]
    k, v = k.masked_fill(gone, math.nan), v.masked_fill(gone, math.inf)
    lse = torch.empty(B, H, Sq, device="cuda")
    o = ops.cross_attention(q, k, v, scale=D ** -0.5, attention_mask=m, kv_lens=lens, lse=lse)
    _check(o, _ref(q, k, v, D ** -0.5, m, lens), dtype, D, Sk, v[v.isfinite()].abs().max().item(), lse)
    for _ in range(20):
        assert torch.equal(ops.cross_attention(q, k, v, scale=D ** -0.5, attention_mask=m, kv_lens=lens), o)
    from difflet_b200 import _native

    _native.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_compiled_calls_trace_the_library_path(native, D):
    """A whole-graph trace (no code generation) meets no opaque native call."""
    q, k, v = _inputs(2, 4, 4, 20, 33, D, torch.bfloat16, "cuda")
    m = torch.rand(20, 33, device="cuda") < 0.7
    m[:, 0] = True
    for fn in BOTH:
        call = torch.compile(lambda q, k, v: fn(q, k, v, scale=0.1, attention_mask=m), backend="eager", fullgraph=True)  # noqa: B023
        want, _, size, _ = _ref(q, k, v, 0.1, m)
        assert bool(((call(q, k, v).double() - want).abs() <= 2 * torch.finfo(q.dtype).eps * (size + want.abs())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fused_attention_keeps_what_it_took(native, dtype):
    """``ops.fused.attention`` at head dim 64: values of another width, one batch row of keys, a result of another type."""
    from difflet_b200.ops import fused as F

    q, k, v = _inputs(3, 4, 4, 30, 41, 64, dtype, "cuda")
    wide = _inputs(3, 4, 4, 30, 41, 32, dtype, "cuda", 1)[2]
    hi = torch.tensor([41, 7, 30], device="cuda", dtype=torch.int32)
    lo = torch.zeros_like(hi)
    eps = torch.finfo(dtype).eps
    for args, full in (((q, k, wide), (q, k, wide)), ((q, k[:1], v[:1]), (q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)))):
        for kw, ref in (({}, {}), (dict(kv_lo=lo, kv_hi=hi), dict(lens=hi))):
            o = F.attention(*args, 0.1, **kw)
            want, _, size, _ = _ref(*full, 0.1, **ref)
            assert bool(((o.double() - want).abs() <= 2 * eps * (size + want.abs()) + 1e-6).all())
    want = F.attention(q, k, v, 0.1)
    out = torch.empty(3, 4, 30, 64, device="cuda")
    assert F.attention(q, k, v, 0.1, out=out) is out and torch.equal(out, want.float())


@pytest.mark.gpu
@pytest.mark.parametrize("fn", BOTH)
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.bfloat16), (40, torch.float32)])
def test_bounds_of_one_edge_per_batch_row_off_the_kernels(native, fn, D, dtype):
    """[B], [B, 1] and scalar bounds mean the same with and without gradients, at head dims with and without a kernel."""
    q, k, v = _inputs(3, 2, 2, 20, 33, D, dtype, "cuda")
    lo, hi = torch.tensor([0, 3, 5], device="cuda"), torch.tensor([33, 12, 5 + 28], device="cuda")
    keep = (torch.arange(33, device="cuda") >= lo[:, None]) & (torch.arange(33, device="cuda") < hi[:, None])
    want, _, size, _ = _ref(q, k, v, 0.1, keep[:, None, None])
    tol = 2 * torch.finfo(dtype).eps * (size + want.abs()) + 2.0 ** -20
    for shape in ((3,), (3, 1), (3, 1, 1, 1)):
        kw = dict(bound_min=lo.view(shape), bound_max=hi.view(shape))
        for grad in (False, True):
            o = fn(q.detach().clone().requires_grad_(grad), k, v, scale=0.1, **kw)
            assert o.requires_grad == grad and bool(((o.double() - want).abs() <= tol).all())
    one = dict(bound_min=torch.tensor(2, device="cuda"), bound_max=torch.tensor(30, device="cuda"))
    want, _, size, _ = _ref(q, k, v, 0.1, ((torch.arange(33, device="cuda") >= 2) & (torch.arange(33, device="cuda") < 30))[None, None, None])
    for grad in (False, True):
        o = fn(q.detach().clone().requires_grad_(grad), k, v, scale=0.1, **one)
        assert bool(((o.double() - want).abs() <= 2 * torch.finfo(dtype).eps * (size + want.abs()) + 2.0 ** -20).all())
