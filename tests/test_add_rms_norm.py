"""Residual RMSNorm (``ops.add_rms_norm``) and the MX dequantiser against the formula in 64 bits.

Tolerances: one rounding to the output type is half a step (``finfo.eps / 2`` of the value); the f32
arithmetic before it (a sum of at most 2^14 squares, pairwise over >= 32 threads, one rsqrt, three
products and a sum) is within 2^-18 of the terms it adds.
"""

import pytest
import torch

from difflet_b200 import ops
from difflet_b200.ops import fused as F

F32 = 2.0 ** -18


def _ref(x, resid, w, eps, scale, shift, batch_of):
    s = x.double() + (resid.double() if resid is not None else 0)
    a = s / (s.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if w is not None:
        a = a * w.double()
    if scale is not None:
        a = a * (1 + scale.double()[batch_of])
    size = a.abs()
    if shift is not None:
        a = a + shift.double()[batch_of]
        size = size + shift.double()[batch_of].abs()
    return s, a, size


def _check(y, ref, size, dtype):
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # one subnormal step
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + F32 * size + tiny
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol.clamp_min(1e-300)).max().item():.3g} of the tolerance"


def _inputs(M, D, dtype, device, seed=0, batch=0, w_dtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, resid = r(M, D).to(dtype), (3 * r(M, D)).to(dtype)
    w = (1 + 0.1 * r(D)).to(w_dtype or dtype)
    scale, shift = (0.2 * r(batch, D), 0.2 * r(batch, D)) if batch else (None, None)
    return [t if t is None else t.to(device) for t in (x, resid, w, scale, shift)]


def _case(M, D, dtype, device, batch=0, w_dtype=None):
    x, resid, w, scale, shift = _inputs(M, D, dtype, device, M * 31 + D, batch, w_dtype)
    rpb = -(-M // batch) if batch else 0
    bo = torch.arange(M, device=device) // rpb if batch else None
    y, s = ops.add_rms_norm(x, resid, w, eps=1e-5, scale=scale, shift=shift, rows_per_batch=rpb)
    rs, ry, size = _ref(x, resid, w, 1e-5, scale, shift, bo)
    assert y.dtype == s.dtype == dtype and y.shape == s.shape == x.shape
    _check(s, rs, x.double().abs() + resid.double().abs(), dtype)
    _check(y, ry, size, dtype)


@pytest.mark.parametrize("D", [32, 100])
def test_oracle(D):
    _case(5, D, torch.float32, "cpu", batch=2)


def test_refusals():
    x = torch.randn(4, 96)
    for kw in (dict(resid=torch.randn(4, 95)), dict(resid=torch.randn(4, 96).double()), dict(weight=torch.ones(95)),
               dict(weight=torch.ones(96).half()), dict(scale=torch.ones(96)), dict(shift=torch.ones(2, 95)),
               dict(resid_out=torch.empty(4, 96)), dict(out=torch.empty(4, 95)), dict(blocked=True),
               dict(quantize="float8_e4m3fn", blocked=True), dict(quantize="float8_e4m3fn", out=torch.empty(4, 96)),
               dict(row_map=torch.zeros(3, dtype=torch.int32)), dict(row_map=torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(ValueError):
            ops.add_rms_norm(x, **kw)
    with pytest.raises(ValueError):
        ops.add_rms_norm(torch.randn(2, 16385))
    with pytest.raises(ValueError):
        ops.add_rms_norm(torch.randn(2, 33), quantize="float8_e4m3fn")
    with pytest.raises(NotImplementedError):
        ops.add_rms_norm(x, quantize="int8")
    with pytest.raises(RuntimeError, match="no backward"):
        ops.add_rms_norm(x.clone().requires_grad_())
    with torch.no_grad():
        ops.add_rms_norm(x.clone().requires_grad_())


def test_oracle_without_residual_and_empty():
    x = torch.randn(2, 3, 64)
    y, s = ops.add_rms_norm(x)
    assert s is x and y.shape == x.shape
    y, s = ops.add_rms_norm(x[:0], x[:0], scale=torch.ones(1, 64))
    assert y.shape == s.shape == (0, 3, 64)


# ----------------------------------------------------------------------------- B200
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,D,batch", [(1, 1, 0), (3, 8, 0), (5, 33, 2), (130, 256, 3), (7, 520, 0), (9, 1023, 2), (64, 1536, 2),
                                       (257, 2048, 0), (33, 5120, 5), (4, 8191, 0), (3, 10240, 1), (2, 16384, 2)])
def test_kernel(native, M, D, batch, dtype):
    _case(M, D, dtype, "cuda", batch, w_dtype=torch.float32 if M % 2 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("M,D,batch,dtype,fmt", [(9601, 1032, 3, torch.bfloat16, None), (2501, 4096, 2, torch.float32, None),
                                                 (2400, 8192, 0, torch.float16, None), (9700, 1024, 1, torch.bfloat16, "float8_e4m3fn"),
                                                 (2431, 5120, 7, torch.bfloat16, "float8_e5m2"), (5000, 2048, 2, torch.float32, "float8_e4m3fn")])
def test_kernel_many_rows(native, M, D, batch, dtype, fmt):
    x, resid, w, scale, shift = _inputs(M, D, dtype, "cuda", M, max(batch, 1))
    m = torch.randint(0, max(batch, 1), (M,), device="cuda", dtype=torch.int32)
    kw = dict(eps=1e-5, scale=scale, shift=shift, row_map=m) if batch else dict(eps=1e-5)
    rs, ry, size = _ref(x, resid, w, 1e-5, scale if batch else None, shift if batch else None, m.long())
    y, s = ops.add_rms_norm(x, resid, w, quantize=fmt, **kw)
    _check(s, rs, x.double().abs() + resid.double().abs(), dtype)
    if fmt is None:
        _check(y, ry, size, dtype)
        _check(ops.add_rms_norm(x, None, w, eps=1e-5)[0], *_ref(x, None, w, 1e-5, None, None, None)[1:], dtype)
        a, b = x.clone(), resid.clone()
        ops.add_rms_norm(a, b, w, out=a, resid_out=b, **kw)
        assert torch.equal(a, y) and torch.equal(b, s)
    else:
        _check_mx(*y, ry, size, *((8, 448.0, 3, -6) if fmt == "float8_e4m3fn" else (15, 57344.0, 2, -14)))
        (qb, sb), _ = ops.add_rms_norm(x, resid, w, quantize=fmt, blocked=True, **kw)
        assert torch.equal(qb.view(torch.uint8), y[0].view(torch.uint8)) and torch.equal(sb, F.block_scales(y[1]))


@pytest.mark.gpu
def test_kernel_refusals(native):
    x = torch.randn(4, 96, device="cuda")
    c = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)  # noqa: E731
    for kw in (dict(resid=c(4, 95)), dict(resid=c(4, 96).half()), dict(resid=torch.zeros(4, 96)), dict(weight=c(95)), dict(weight=c(96).half()),
               dict(scale=c(96)), dict(shift=c(2, 95)), dict(shift=c(2, 96).half()), dict(scale=c(2, 96), rows_per_batch=1),
               dict(scale=c(2, 96), shift=c(1, 96)), dict(resid_out=c(4, 96)), dict(out=c(4, 95)), dict(blocked=True),
               dict(quantize="float8_e4m3fn", blocked=True), dict(quantize="float8_e4m3fn", out=c(4, 96)),
               dict(row_map=c(3, dtype=torch.int32)), dict(row_map=c(4, dtype=torch.int64)), dict(weight=c(192)[::2])):
        with pytest.raises(ValueError):
            ops.add_rms_norm(x, **kw)
    for bad in (c(2, 16385), x.t(), x.double(), x.int()):
        with pytest.raises(ValueError):
            ops.add_rms_norm(bad)
    for bad in (c(2, 33), c(2, 65)[:, 1:]):
        with pytest.raises(ValueError):
            ops.add_rms_norm(bad, quantize="float8_e4m3fn")
    with pytest.raises(NotImplementedError):
        ops.add_rms_norm(x, quantize="int8")
    with pytest.raises(RuntimeError, match="no backward"):
        ops.add_rms_norm(x.clone().requires_grad_())


@pytest.mark.gpu
def test_kernel_strided_aliased_mapped(native):
    big = torch.randn(40, 2, 1032, device="cuda").bfloat16()
    for off in (0, 8, 3):  # aligned and odd starts of strided rows
        x, resid = big[:, 0, off:off + 1024], big[:, 1, off:off + 1024]
        m = torch.randint(0, 3, (40,), device="cuda", dtype=torch.int32)
        mod = torch.randn(3, 2, 1024, device="cuda")
        y, s = ops.add_rms_norm(x, resid, scale=mod[:, 0], shift=mod[:, 1], row_map=m)
        rs, ry, size = _ref(x, resid, None, 1e-6, mod[:, 0], mod[:, 1], m.long())
        _check(y, ry, size, x.dtype)
        _check(s, rs, x.double().abs() + resid.double().abs(), x.dtype)
    x, r = torch.randn(2, 9, 640, device="cuda").half(), torch.randn(2, 9, 640, device="cuda").half()
    want = ops.add_rms_norm(x, r)
    a, b = x.clone(), r.clone()
    y, s = ops.add_rms_norm(a, b, out=a, resid_out=b)  # in place
    assert y is a and s is b and torch.equal(a, want[0]) and torch.equal(b, want[1])
    assert ops.add_rms_norm(x)[1] is x
    y, s = ops.add_rms_norm(x[:0], r[:0], quantize="float8_e4m3fn", blocked=True)
    assert y[0].shape == (0, 9, 640) and y[1].numel() == 0


def _check_mx(q, sf, ry, size, emax, top, mant, low):
    """Elements within half an FP8 step of the (clamped) value at the stored scale, scales floor(log2(amax)) - emax."""
    M, D = ry.shape
    e = sf.view(M, D // 32, 1).double() - 127
    blocks, slack = ry.view(M, D // 32, 32), size.view(M, D // 32, 32) * F32
    amax = blocks.abs().amax(-1, keepdim=True)
    d = slack.amax(-1, keepdim=True)
    lo = (torch.log2((amax - d).clamp_min(2.0 ** -140)).floor() - emax).clamp(-127, 127)
    hi = (torch.log2((amax + d).clamp_min(2.0 ** -140)).floor() - emax).clamp(-127, 127)
    assert bool(((e >= lo) & (e <= hi)).all())
    v = q.double().view(M, D // 32, 32) * torch.exp2(e)
    want = torch.minimum(torch.maximum(blocks, -top * torch.exp2(e)), top * torch.exp2(e))
    tol = want.abs() * 2.0 ** -(mant + 1) + torch.exp2(e + low - mant - 1) + 2 * slack
    assert bool(((v - want).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["float8_e4m3fn", "float8_e5m2"])
@pytest.mark.parametrize("M,D,dtype", [(1, 32, torch.bfloat16), (70, 96, torch.float32), (129, 384, torch.float16), (300, 5120, torch.bfloat16),
                                       (5, 2048, torch.float32)])
def test_kernel_mx(native, M, D, dtype, fmt):
    x, resid, w, scale, shift = _inputs(M, D, dtype, "cuda", 7, 1)
    x[0], resid[0] = 0, 0  # a row of zeros: only the shift is left
    (q, sf), s = ops.add_rms_norm(x, resid, w, scale=scale, shift=shift, quantize=fmt)
    rs, ry, size = _ref(x, resid, w, 1e-6, scale, shift, torch.zeros(M, dtype=torch.long, device="cuda"))
    form = (8, 448.0, 3, -6) if fmt == "float8_e4m3fn" else (15, 57344.0, 2, -14)
    _check_mx(q, sf, ry, size, *form)
    _check(s, rs, x.double().abs() + resid.double().abs(), dtype)
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        got = ops.dequantize_mx(q, sf, dtype=fmt, output_dtype=dt)
        want = (q.double().view(M, -1, 32) * torch.exp2(sf.double() - 127)[..., None]).view(M, D).to(dt)
        assert torch.equal(got, want)
    if D % 128 == 0:
        (qb, sb), _ = ops.add_rms_norm(x, resid, w, scale=scale, shift=shift, quantize=fmt, blocked=True)
        assert torch.equal(qb.view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(sb, F.block_scales(sf))  # the padding rows are zero too


@pytest.mark.gpu
def test_kernel_mx_feeds_the_block_scaled_gemm(native):
    M, D, N = 200, 512, 256
    x, resid, w, _, _ = _inputs(M, D, torch.bfloat16, "cuda", 3)
    wq = F.MXWeight.quantize(torch.randn(N, D, device="cuda") * D ** -0.5)
    (q, sf), _ = ops.add_rms_norm(x, resid, w, quantize="float8_e4m3fn", blocked=True)
    y = F.linear_mx(q, sf, wq.q, wq.sf)
    a = ops.dequantize_mx(q, F.unblock_scales(sf, M, D), output_dtype=torch.float32).double()
    ref = a @ wq.dequantize(torch.float32).double().t()
    # products of 4-bit significands are exact in f32; D f32 additions and the rounding to bf16
    tol = 2.0 ** -8 * ref.abs() + D * 2.0 ** -24 * (a.abs() @ wq.dequantize(torch.float32).double().abs().t())
    assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.gpu
def test_kernel_edges(native):
    x = torch.randn(4, 256, device="cuda")
    x[0] = 0
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    y, _ = ops.add_rms_norm(x, eps=0.5)
    assert bool((y[0] == 0).all()) and bool(y[2].isnan().all()) and bool(y[1, 3].isnan())
    assert bool((y[1, 4:] == 0).all()) and bool(y[3].isfinite().all())
    # a modulation row that does not exist: reported, and the row is normalised without it
    from difflet_b200 import _native

    m = torch.tensor([0, 1, 5, -1], device="cuda", dtype=torch.int32)
    good = ops.add_rms_norm(x)[0]
    y, _ = ops.add_rms_norm(x, scale=torch.ones(2, 256, device="cuda"), row_map=m)
    assert torch.equal(y[3], good[3])
    with pytest.raises(Exception):
        _native.check_device_errors()
    _native.check_device_errors()


@pytest.mark.gpu
def test_kernel_graph_and_stream(native):
    x, resid, w, _, _ = _inputs(64, 1024, torch.bfloat16, "cuda", 5)
    want = ops.add_rms_norm(x, resid, w)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = ops.add_rms_norm(x, resid, w)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cap = ops.add_rms_norm(x, resid, w)
    x.copy_(torch.randn_like(x))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(cap[0], ops.add_rms_norm(x, resid, w)[0])
