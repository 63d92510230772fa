"""``ops.linear_lora`` / ``ops.LoraBank`` against the formula in 64 bits.

Tolerances, u = half a bf16 step: the rank-r intermediate T = s x A^T is rounded once (u of sum |T||B|), the
result once (u of |y|); f32 accumulation in any order adds 2^-24 (K + r) of the sums of magnitudes. An
activation multiplies what comes before it by at most its steepest slope, 1.13; the GELU's tanh is
evaluated to 2^-11.
"""

import pytest
import torch

from difflet_b200 import ops
from difflet_b200.ops import fused as F

BF = torch.bfloat16


def _make(M, N, K, ranks, device, dtype=BF, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, w, b = r(M, K).to(device, dtype), (r(N, K) * K ** -0.5).to(device, dtype), (0.1 * r(N)).to(device, dtype)
    A = [(r(k, K) * K ** -0.5).to(device, dtype) for k in ranks]
    B = [(r(N, k) * k ** -0.5).to(device, dtype) for k in ranks]
    scale = [0.5 + 0.25 * i for i in range(len(ranks))]
    return x, w, b, A, B, scale


def _ref(x, w, b, A, B, scale, rows, u):
    """Sums before the epilogue and their error bound."""
    x, w = x.double(), w.double()
    K = x.shape[1]
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    rounding = torch.zeros_like(y)
    for i, (a, bb, s) in enumerate(zip(A, B, scale)):
        at = rows == i
        if at.any():
            a, bb = a.double(), bb.double()
            t = s * (x[at] @ a.t())
            y[at] += t @ bb.t()
            mag = abs(s) * (x[at].abs() @ a.abs().t()) @ bb.abs().t()
            size[at] += 2 * mag
            rounding[at] += u * t.abs() @ bb.abs().t()
    if b is not None:
        y = y + b.double()
        size = size + b.double().abs()
    return y, rounding + 2.0 ** -24 * (K + 128) * size


def _act(y, act):
    if act == "gelu":
        return torch.nn.functional.gelu(y, approximate="tanh")
    return torch.nn.functional.silu(y) if act == "silu" else y


def _compare(got, y, err, act, u, scale_of_act=1.0):
    want = _act(y, act)
    tol = (1.13 if act else 1.0) * err + u * want.abs() + (2.0 ** -11 * y.abs() if act == "gelu" else 0) + 1e-30
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"worst {(off / tol).max().item():.3g} of the tolerance"


# ----------------------------------------------------------------------------- CPU
def test_oracle_and_layout():
    x, w, b, A, B, scale = _make(7, 24, 32, [3, 16, 5], "cpu", torch.float32)
    bank = ops.LoraBank(A, B, scale)
    assert bank.rank == 16 and bank.A.shape == (3, 16, 32) and bank.B.shape == (3, 24, 16) and bank.ranks == [3, 16, 5]
    ids = torch.tensor([0, 2, -1, 1, 1, 0, 2])
    for kw in ({}, {"act": "gelu"}, {"act": "silu"}):
        y = ops.linear_lora(x, w, b, bank=bank, ids=ids, **kw)
        want, _ = _ref(x, w, b, A, B, scale, ids, 0)
        assert torch.allclose(y.double(), _act(want, kw.get("act")), atol=1e-4)
    y = ops.linear_lora(x.view(1, 7, 32), w, b, bank=bank, ids=torch.tensor([1, -1, 2]), rows_per_batch=3)
    want, _ = _ref(x, w, b, A, B, scale, torch.tensor([1, 1, 1, -1, -1, -1, 2]), 0)
    assert y.shape == (1, 7, 24) and torch.allclose(y[0].double(), want, atol=1e-4)
    gate, resid = torch.randn(3, 24), torch.randn(7, 24)
    y = ops.linear_lora(x, w, b, bank=bank, ids=torch.tensor([1, -1, 2]), rows_per_batch=3, gate=gate, resid=resid)
    assert torch.allclose(y.double(), resid.double() + gate.double().repeat_interleave(3, 0)[:7] * want, atol=1e-4)
    two = ops.LoraBank(bank.A, bank.B, bank.scale)  # already laid out: used as it is
    assert two.A.data_ptr() == bank.A.data_ptr() and two.B.data_ptr() == bank.B.data_ptr()
    assert ops.LoraBank(A, B, scale).to(dtype=torch.float64).A.dtype == torch.float64


def test_refusals():
    x, w, b, A, B, scale = _make(6, 24, 32, [4, 4], "cpu", torch.float32)
    bank = ops.LoraBank(A, B, scale)
    ids = torch.zeros(6, dtype=torch.long)
    for args in (([], []), (A, B[:1]), ([A[0], A[1][:, :16]], B), ([A[0][:3], A[1]], B), ([A[0].double(), A[1]], B),
                 ([torch.zeros(129, 32)], [torch.zeros(24, 129)]), ([A[0].int()], [B[0].int()])):
        with pytest.raises(ValueError):
            ops.LoraBank(*args)
    with pytest.raises(ValueError):
        ops.LoraBank(A, B, [1.0])
    with pytest.raises(ValueError, match="infinities"):
        ops.LoraBank(A, [B[0], B[1] / 0.0])
    for a, kw in (((x[:, :16], w, b), {}), ((x, w[:16], b), {}), ((x, w, b), dict(ids=ids[:5])), ((x, w, b), dict(ids=ids.float())),
                  ((x, w, b), dict(ids=ids[:1], rows_per_batch=4)), ((x, w, b), dict(act="swiglu")),
                  ((x, w, b), dict(gate=torch.ones(1, 24))), ((x, w, b), dict(resid=torch.ones(6, 24))),
                  ((x, w, b), dict(act="gelu", gate=torch.ones(1, 24), resid=torch.ones(6, 24))),
                  ((x, w, b), dict(act="gelu", out_f32=True)), ((x, w, b), dict(out=torch.empty(6, 23))), ((x.double(), w.double(), b.double()), {})):
        with pytest.raises(ValueError):
            ops.linear_lora(*a, bank=bank, **{"ids": ids, **kw})
    with pytest.raises(RuntimeError, match="no backward"):
        ops.linear_lora(x.clone().requires_grad_(), w, b, bank=bank, ids=ids)
    q = F.MXWeight(torch.zeros(24, 32, dtype=torch.float8_e4m3fn), torch.zeros(256, dtype=torch.uint8))
    with pytest.raises(NotImplementedError):
        ops.linear_lora(x, q, b, bank=bank, ids=ids)


# ----------------------------------------------------------------------------- B200
CASES = [  # M, N, K, ranks
    (1, 64, 64, [1]), (4, 4096, 1024, [16] * 4), (130, 520, 200, [8, 3]), (37, 1536, 5120, [64, 16, 40]), (300, 1024, 512, [128] * 5),
    (1100, 1536, 1536, [32] * 3), (2049, 2048, 256, [16] * 40), (700, 1024, 320, [16] * 200), (5000, 1280, 640, [4, 100]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["rows", "batch", "none"])
@pytest.mark.parametrize("M,N,K,ranks", CASES)
def test_kernel(native, M, N, K, ranks, how):
    x, w, b, A, B, scale = _make(M, N, K, ranks, "cuda", seed=M)
    bank = ops.LoraBank(A, B, scale)
    n, rpb = len(ranks), 0
    g = torch.Generator().manual_seed(1)
    if how == "rows":
        ids = rows = torch.randint(-1, n, (M,), generator=g).cuda()
    elif how == "batch":
        rpb = max(1, M // 3 + 1)
        ids = torch.randint(0, n, (-(-M // rpb),), generator=g, dtype=torch.int32).cuda()
        rows = ids.repeat_interleave(rpb)[:M]
    else:
        ids = rows = torch.full((M,), -1, device="cuda", dtype=torch.int32)
    u = 2.0 ** -8
    y, err = _ref(x, w, b, A, B, scale, rows, u)
    for act in (None, "gelu", "silu"):
        _compare(ops.linear_lora(x, w, b, bank=bank, ids=ids, rows_per_batch=rpb, act=act), y, err, act, u)
    if how == "none" and M >= 1024:  # large M never splits K: the plain projection, bit for bit
        assert torch.equal(ops.linear_lora(x, w, b, bank=bank, ids=ids), F.linear(x, w, b))
    y32 = ops.linear_lora(x, w, None, bank=bank, ids=ids, rows_per_batch=rpb, out_f32=True)
    _compare(y32, y - b.double(), err, None, 0.0)
    from difflet_b200 import _native

    _native.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["rows", "batch"])
@pytest.mark.parametrize("M,N,K,ranks", [
    (200, 384, 1280, [128] * 9), (664, 640, 2000, [128, 100] * 6), (90, 3200, 2880, [64] * 11), (1333, 2048, 2048, [8] * 7),  # passes shared out
    (17, 24, 72, [48]), (32, 1000, 2056, [128, 3, 64]), (16, 2056, 520, [128, 80]),  # rows and columns at the ends of a thread's share
])
def test_kernel_passes_and_few_rows(native, M, N, K, ranks, how):
    test_kernel(native, M, N, K, ranks, how)


@pytest.mark.gpu
def test_kernel_gated_residual_layouts(native):
    M, N, K = 600, 1024, 512
    x, w, b, A, B, scale = _make(M, N, K, [16, 32], "cuda")
    bank = ops.LoraBank(A, B, scale)
    ids = torch.tensor([1, 0, -1], device="cuda")
    rows = ids.repeat_interleave(200)
    gate, resid = torch.randn(3, N, device="cuda"), torch.randn(M, N, device="cuda", dtype=BF)
    u = 2.0 ** -8
    y, err = _ref(x, w, b, A, B, scale, rows, u)
    gr = gate.double().repeat_interleave(200, 0)
    want = resid.double() + gr * y
    buf = resid.clone()
    got = ops.linear_lora(x, w, b, bank=bank, ids=ids, rows_per_batch=200, gate=gate, resid=buf, out=buf)
    assert got is buf
    tol = gr.abs() * err + u * want.abs() + 2.0 ** -22 * (resid.double().abs() + (gr * y).abs())
    assert bool(((buf.double() - want).abs() <= tol).all())
    big = torch.full((M, N + 64), 3.0, device="cuda", dtype=BF)
    ops.linear_lora(x, w, b, bank=bank, ids=ids, rows_per_batch=200, out=big[:, 32:32 + N])
    plain = ops.linear_lora(x, w, b, bank=bank, ids=ids, rows_per_batch=200)
    assert torch.equal(big[:, 32:32 + N], plain) and bool((big[:, :32] == 3).all() and (big[:, 32 + N:] == 3).all())
    wide = torch.empty(M, K + 3, device="cuda", dtype=BF)[:, 1:K + 1]
    wide.copy_(x)  # rows no copy engine addresses
    assert torch.equal(ops.linear_lora(wide, w, b, bank=bank, ids=ids, rows_per_batch=200), plain)
    assert ops.linear_lora(x[:0], w, b, bank=bank, ids=rows[:0]).shape == (0, N)
    y3 = ops.linear_lora(x.view(3, 200, K), w, b, bank=bank, ids=ids, rows_per_batch=200)
    assert y3.shape == (3, 200, N) and torch.equal(y3.view(M, N), plain)


@pytest.mark.gpu
def test_kernel_refusals(native):
    x, w, b, A, B, scale = _make(6, 24, 32, [4, 4], "cuda")
    bank = ops.LoraBank(A, B, scale)
    ids = torch.zeros(6, dtype=torch.long, device="cuda")
    c = lambda *s, **kw: torch.ones(*s, device="cuda", **kw)  # noqa: E731
    for a, kw in (((x[:, :16], w, b), {}), ((x, w[:16], b), {}), ((x.float(), w, b), {}), ((x, w.float(), b), {}), ((x, w.cpu(), b), {}),
                  ((x, w, b[:16]), {}), ((x, w, b.float()), {}), ((x, w, b), dict(ids=ids[:5])), ((x, w, b), dict(ids=ids.float())),
                  ((x, w, b), dict(ids=ids.cpu())), ((x, w, b), dict(ids=ids[:1], rows_per_batch=4)), ((x, w, b), dict(act="swiglu")),
                  ((x, w, b), dict(gate=c(1, 24))), ((x, w, b), dict(resid=c(6, 24, dtype=BF))),
                  ((x, w, b), dict(gate=c(1, 24), resid=c(6, 24, dtype=BF), gate_rows_per_batch=2)),
                  ((x, w, b), dict(gate=c(1, 24), resid=c(6, 24))), ((x, w, b), dict(act="gelu", gate=c(1, 24), resid=c(6, 24, dtype=BF))),
                  ((x, w, b), dict(out=c(6, 23, dtype=BF))), ((x, w, b), dict(out=c(6, 24))), ((x, w, b), dict(out=c(6, 25, dtype=BF)[:, 1:]))):
        with pytest.raises(ValueError):
            ops.linear_lora(*a, bank=bank, **{"ids": ids, **kw})
    odd = ops.LoraBank([a[:, :30] for a in A], B, scale)  # rows that are no whole 16-byte pieces
    with pytest.raises(ValueError):
        ops.linear_lora(x[:, :30], w[:, :30], b, bank=odd, ids=ids)


@pytest.mark.gpu
def test_kernel_beside_a_weight_kept_in_eight_bits(native):
    x, w, b, A, B, scale = _make(70, 256, 512, [8, 8], "cuda")
    bank, ids = ops.LoraBank(A, B, scale), torch.randint(-1, 2, (70,), device="cuda")
    q = F.MXWeight.quantize(w, compute="dequant")
    got = ops.linear_lora(x.view(7, 10, 512), q, b, bank=bank, ids=ids, act="gelu")
    assert got.shape == (7, 10, 256)
    assert torch.equal(got.view(70, 256), ops.linear_lora(x, q.dequantize(), b, bank=bank, ids=ids, act="gelu"))
    with pytest.raises(NotImplementedError):
        ops.linear_lora(x, F.MXWeight.quantize(w), b, bank=bank, ids=ids)
    row = ops.linear_lora(x[0], w, b, bank=bank, ids=ids[:1])  # a single row as a vector
    assert row.shape == (256,) and torch.equal(row, ops.linear_lora(x[:1], w, b, bank=bank, ids=ids[:1])[0])


@pytest.mark.gpu
def test_kernel_rows_do_not_see_each_other(native):
    """A row's result does not depend on which adapters its neighbours use."""
    M, N, K = 512, 1024, 256
    x, w, b, A, B, scale = _make(M, N, K, [16] * 6, "cuda")
    bank = ops.LoraBank(A, B, scale)
    ids = torch.randint(-1, 6, (M,), device="cuda")
    whole = ops.linear_lora(x, w, None, bank=bank, ids=ids, out_f32=True)
    bad = x.clone()
    bad[ids == 3] = float("nan")
    part = ops.linear_lora(bad, w, None, bank=bank, ids=ids, out_f32=True)
    assert torch.equal(part[ids != 3], whole[ids != 3]) and bool(part[ids == 3].isnan().all())


@pytest.mark.gpu
def test_kernel_unknown_adapter(native):
    from difflet_b200 import _native

    x, w, b, A, B, scale = _make(40, 256, 128, [8, 8], "cuda")
    bank = ops.LoraBank(A, B, scale)
    ids = torch.tensor([0, 1, -1, 2, 1 << 20, -7] + [0] * 34, device="cuda")
    y = ops.linear_lora(x, w, b, bank=bank, ids=ids)
    none = ops.linear_lora(x, w, b, bank=bank, ids=torch.full_like(ids, -1))
    assert torch.equal(y[2:6], none[2:6])
    with pytest.raises(Exception):
        _native.check_device_errors()
    _native.check_device_errors()


@pytest.mark.gpu
def test_kernel_graph_and_streams(native):
    x, w, b, A, B, scale = _make(64, 2048, 4096, [16] * 4, "cuda")  # few rows: K is split across SMs
    bank = ops.LoraBank(A, B, scale)
    ids = torch.randint(-1, 4, (64,), device="cuda", dtype=torch.int32)
    run = lambda: ops.linear_lora(x, w, b, bank=bank, ids=ids)  # noqa: E731
    want = run()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(6):
        for st in streams:  # calls in flight at once, each with its own workspace
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        c1 = run()
    with torch.cuda.graph(g2):
        c2 = run()
    x.copy_(torch.randn_like(x))
    ids.copy_(torch.randint(-1, 4, (64,), device="cuda", dtype=torch.int32))
    g1.replay()
    g2.replay()
    torch.cuda.synchronize()
    want = run()
    assert torch.equal(c1, want) and torch.equal(c2, want)
