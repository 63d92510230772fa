"""``ops.cross_attention`` (masks, key lengths, shared key heads, head dims 64 / 128) against 64 bits.

Tolerances, with u = half a step of the type: P is rounded once (u of sum p|v| / sum p), the output
once (u of |o|), and the f32 scores (D products summed in any order, one scaling, one 2^x of 2 ulp) move
p by a relative d = 2^-24 (D + 4) max sum|q k| scale + 2^-20, in the products and in their sum (2 d).
fp16 P below 2^-14 is off by at most 2^-25 absolutely (the largest p of a row is at least 1).
"""

import math

import pytest
import torch

from difflet_b200 import ops
from difflet_b200.ops import fused as F


def _ref(q, k, v, scale, mask=None, lens=None):
    """Output, LSE, sum p|v| / sum p and the score bound, in 64 bits; rows without keys are 0."""
    rep = q.shape[1] // k.shape[1]
    k, v = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    B, H, Sq, D = q.shape
    Sk = k.shape[2]
    keep = torch.ones(B, 1, 1, Sk, dtype=torch.bool, device=q.device)
    if lens is not None:
        keep = (torch.arange(Sk, device=q.device) < lens.view(-1, 1))[:, None, None]
    if mask is not None and mask.dtype == torch.bool and mask.dim() == 4 and mask.shape[1] == mask.shape[2] == 1:
        keep = keep & mask
    k = torch.where(keep.transpose(2, 3), k, 0.0)
    v = torch.where(keep.transpose(2, 3), v, 0.0)
    z = q.double() @ k.transpose(2, 3) * scale
    bound = (q.double().abs() @ k.abs().transpose(2, 3)).amax().item() * abs(scale) if Sk else 0.0
    if mask is not None:
        if mask.dtype == torch.bool:
            z = z.masked_fill(~mask, -math.inf)
        else:
            z = (z.float() + mask.float()).double()  # a bias of the type's lowest value absorbs the score in f32
    z = z.masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(z, -1) if Sk else torch.full(z.shape[:-1], -math.inf, device=q.device, dtype=torch.float64)
    # softmax subtracts the maximum (scores at the type's lowest value absorb the log of their sum)
    p = torch.where(torch.isinf(lse)[..., None], 0.0, torch.softmax(z, -1))
    if mask is not None and mask.dtype != torch.bool:
        # f32 rounding of score + bias, here and in the kernel (one that absorbs every score rounds alike)
        big = mask.float().abs()
        big = big[torch.isfinite(big) & (big < 1e30)]
        bound += 2 * (big.max().item() if big.numel() else 0.0) / (D + 4)
    return p @ v, lse, p @ v.abs(), bound


def _check(o, ref, dtype, D, Sk, vmax, lse=None):
    want, lse_ref, size, bound = ref
    u = torch.finfo(dtype).eps / 2
    d = 2.0 ** -24 * (D + 4) * bound + 2.0 ** -20
    tol = (u + 2 * d) * size + u * want.abs() + 1e-30
    if dtype == torch.float16:
        tol = tol + Sk * 2.0 ** -25 * vmax + 2.0 ** -25
    err = (o.double() - want).abs()
    assert bool((err <= tol).all()), f"worst {(err / tol).nan_to_num(1e9).max().item():.3g} of the tolerance"
    if lse is not None:
        fine = torch.isfinite(lse_ref)
        assert torch.equal(fine, torch.isfinite(lse.double()))
        assert bool(((lse.double() - lse_ref).abs()[fine] <= d + 2.0 ** -20 * (1 + lse_ref.abs()[fine])).all())


def _inputs(B, H, Hk, Sq, Sk, D, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(device, dtype)  # noqa: E731
    q = r(B, Sq, H, D).permute(0, 2, 1, 3)
    kv = r(B, Sk, 2, Hk, D)
    return q, kv[:, :, 0].permute(0, 2, 1, 3), kv[:, :, 1].permute(0, 2, 1, 3)


def _mask(kind, B, H, Sq, Sk, device, dtype):
    g = torch.Generator().manual_seed(1)
    keep = torch.rand(B, H if kind == "head" else 1, Sq, Sk, generator=g) < 0.4
    keep[:, :, ::5] = False  # rows without a key
    if kind == "keys":
        keep = keep[:, :, 1 % Sq:1 % Sq + 1].clone()
        keep[..., 0] = True
        keep[-1] = False  # a batch row without a key
        return keep.to(device)
    if kind in ("bool", "head"):
        return keep.to(device)
    if kind == "lowest":
        return torch.where(keep, 0.0, torch.finfo(dtype).min).to(device, dtype)
    bias = torch.where(keep, torch.randn(keep.shape, generator=g), -math.inf)
    return bias.to(device, torch.float32 if kind == "bias32" else dtype)


# ----------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("kind", [None, "keys", "bool", "bias"])
def test_oracle(kind):
    q, k, v = _inputs(2, 4, 2, 6, 9, 16, torch.float32, "cpu")
    mask = kind and _mask(kind, 2, 4, 6, 9, "cpu", torch.float32)
    lens = torch.tensor([9, 4])
    lse = torch.empty(2, 4, 6)
    o = ops.cross_attention(q, k, v, scale=0.25, attention_mask=mask, kv_lens=lens, lse=lse)
    want = _ref(q, k, v, 0.25, mask, lens)
    assert torch.allclose(o.double(), want[0], atol=1e-5) and torch.allclose(lse.double(), want[1], atol=1e-5)


def test_oracle_ignores_what_lies_behind_a_length():
    q, k, v = _inputs(2, 2, 1, 3, 8, 16, torch.float32, "cpu")
    lens = torch.tensor([5, 0])
    clean = ops.cross_attention(q, k, v, scale=0.25, kv_lens=lens)
    k, v = k.clone(), v.clone()
    for b, n in enumerate([5, 0]):
        k[b, :, n:], v[b, :, n:] = math.nan, math.inf
    o = ops.cross_attention(q, k, v, scale=0.25, kv_lens=lens)
    assert torch.equal(o, clean) and bool((o[1] == 0).all())


def test_refusals():
    q, k, v = _inputs(2, 4, 2, 3, 5, 16, torch.float32, "cpu")
    lens = torch.tensor([5, 2])
    for args, kw in (((q, k, v[:, :, :4]), {}), ((q[:, :3], k, v), {}), ((q, k[:1], v[:1]), {}), ((q, k[..., :8], v[..., :8]), {}),
                     ((q, k.double(), v.double()), {}), ((q, k, v), dict(kv_lens=lens.float())),
                     ((q, k, v), dict(kv_lens=lens[:1])), ((q, k, v), dict(kv_lens=lens, bound_min=lens, bound_max=lens)),
                     ((q, k, v), dict(bound_min=lens)), ((q, k, v), dict(attention_mask=torch.ones(2, 4, 3, 4).bool())),
                     ((q, k, v), dict(attention_mask=torch.ones(3, 1, 1, 5).bool())), ((q, k, v), dict(out=q[:1])),
                     ((q, k, v), dict(lse=torch.empty(2, 4, 2))), ((q[0], k[0], v[0]), dict(kv_lens=lens))):
        with pytest.raises(ValueError):
            ops.cross_attention(*args, **kw)


# ----------------------------------------------------------------------------- B200
CASES = [  # B, H, Hk, Sq, Sk, D
    (1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 1, 128), (2, 4, 2, 5, 77, 64), (2, 4, 1, 129, 128, 128), (1, 2, 2, 257, 129, 128),
    (3, 2, 2, 300, 640, 64), (2, 3, 3, 128, 1000, 128), (1, 8, 4, 1, 2048, 128), (3, 24, 8, 600, 200, 128), (3, 24, 8, 1100, 130, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [None, "lens", "keys", "bool", "head", "bias", "bias32", "lowest"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", CASES)
def test_kernel(native, B, H, Hk, Sq, Sk, D, kind, dtype):
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, dtype, "cuda", Sq + Sk)
    lens = mask = None
    if kind == "lens":
        lens = torch.tensor([max(0, Sk - 61 * b * b - (b > 1) * Sk) for b in range(B)], device="cuda", dtype=torch.int32)
    elif kind:
        mask = _mask(kind, B, H, Sq, Sk, "cuda", dtype)
    lse = torch.empty(B, H, Sq, device="cuda")
    o = ops.cross_attention(q, k, v, scale=D ** -0.5, attention_mask=mask, kv_lens=lens, lse=lse)
    assert o.shape == q.shape and o.dtype == dtype
    _check(o, _ref(q, k, v, D ** -0.5, mask, lens), dtype, D, Sk, v.abs().max().item(), lse)
    F._lib()
    from difflet_b200 import _native

    _native.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["lens", "keys"])
def test_kernel_ignores_masked_contents(native, kind, D):
    """NaN and infinities at excluded keys (an unfilled buffer) reach no output, whatever the tile."""
    B, H, Hk, Sq, Sk = 4, 4, 2, 300, 700
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, torch.bfloat16, "cuda")
    n = torch.tensor([700, 130, 1, 0], device="cuda")
    keep = torch.arange(Sk, device="cuda") < n[:, None]
    if kind == "keys":
        keep = keep & (torch.arange(Sk, device="cuda") % 3 != 1)
    kw = dict(kv_lens=n) if kind == "lens" else dict(attention_mask=keep[:, None, None])
    clean = ops.cross_attention(q, k, v, scale=0.1, **kw)
    k, v = (torch.where(keep[:, None, :, None], t, float("nan")) for t in (k, v))
    v = torch.where(v.isnan() & (torch.arange(D, device="cuda") % 2 == 0), float("inf"), v)
    o = ops.cross_attention(q, k, v, scale=0.1, **kw)
    assert torch.equal(o, clean) and bool((o[3] == 0).all())


# Up to 16 rows per key head: every way to share the keys among CTAs (one key to a turn of sixteen CTAs, more heads than
# fit at once), one and two blocks of eight rows.
FEW = [  # B, H, Hk, Sq, Sk, D
    (2, 4, 4, 1, 1, 128), (2, 2, 1, 3, 63, 64), (1, 16, 1, 1, 129, 128), (3, 16, 2, 1, 1023, 64), (2, 8, 2, 2, 2081, 128), (1, 3, 3, 16, 4100, 64),
    (1, 2, 1, 5, 5000, 128), (7, 64, 64, 1, 100, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [None, "lens", "keys", "head", "bias"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", FEW)
def test_few_queries(native, B, H, Hk, Sq, Sk, D, kind, dtype):
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, dtype, "cuda", 7 * Sq + Sk)
    lens = mask = None
    if kind == "lens":
        lens = torch.tensor([(Sk, Sk // 3, 1, 0)[b % 4] for b in range(B)], device="cuda", dtype=torch.int32)
    elif kind:
        mask = _mask(kind, B, H, Sq, Sk, "cuda", dtype)
    lse = torch.empty(B, H, Sq, device="cuda")
    o = ops.cross_attention(q, k, v, scale=D ** -0.5, attention_mask=mask, kv_lens=lens, lse=lse)
    _check(o, _ref(q, k, v, D ** -0.5, mask, lens), dtype, D, Sk, v.abs().max().item(), lse)
    if kind == "lens":  # what lies behind a length is not used, whatever it holds
        behind = (torch.arange(Sk, device="cuda") >= lens[:, None])[:, None, :, None]
        k, v = k.masked_fill(behind, float("nan")), v.masked_fill(behind, float("inf"))
    elif kind == "keys":
        gone = ~mask.expand(B, 1, 1, Sk).transpose(2, 3)
        k, v = k.masked_fill(gone, float("inf")), v.masked_fill(gone, float("nan"))
    else:  # repeatable, and the same from other strides
        k, v = k.contiguous(), v.contiguous()
    assert torch.equal(o, ops.cross_attention(q, k, v, scale=D ** -0.5, attention_mask=mask, kv_lens=lens))
    F._lib()
    from difflet_b200 import _native

    _native.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [None, "lens", "keys", "bool", "bias"])
@pytest.mark.parametrize("B,H,Hk,Sq,Sk,D", [  # a few groups of 16 rows, the last one short; heads that end inside a group
    (1, 16, 16, 78, 2355, 64), (2, 8, 2, 23, 1500, 128), (1, 3, 1, 17, 3001, 128), (1, 2, 1, 150, 2000, 128), (4, 3, 3, 33, 1030, 64),
])
def test_few_tiles(native, B, H, Hk, Sq, Sk, D, kind, dtype):
    test_few_queries(native, B, H, Hk, Sq, Sk, D, kind, dtype)


@pytest.mark.gpu
def test_few_queries_rise(native):
    """Scores that rise along the keys (the running maximum moves at almost every block), and rows that differ."""
    B, H, Hk, Sq, Sk, D = 1, 8, 2, 4, 3000, 128
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, torch.bfloat16, "cuda")
    k[..., 0] = torch.arange(Sk, device="cuda") / 64
    q[..., 0] = torch.arange(H, device="cuda")[:, None] - 2.0
    lse = torch.empty(B, H, Sq, device="cuda")
    o = ops.cross_attention(q, k, v, scale=0.5, lse=lse)
    _check(o, _ref(q, k, v, 0.5), torch.bfloat16, D, Sk, v.abs().max().item(), lse)


@pytest.mark.gpu
def test_kernel_refusals(native):
    q, k, v = _inputs(2, 4, 2, 3, 5, 64, torch.bfloat16, "cuda")
    lens = torch.tensor([5, 2], device="cuda")
    ones = lambda *s: torch.ones(*s, device="cuda", dtype=torch.bool)  # noqa: E731
    for args, kw in (((q, k, v[:, :, :4]), {}), ((q[:, :3], k, v), {}), ((q, k[:1], v[:1]), {}), ((q, k.half(), v.half()), {}),
                     ((q, k.cpu(), v.cpu()), {}), ((q, k, v), dict(kv_lens=lens.float())), ((q, k, v), dict(kv_lens=lens[:1])),
                     ((q, k, v), dict(kv_lens=lens, bound_min=lens, bound_max=lens)), ((q, k, v), dict(bound_min=lens)),
                     ((q, k, v), dict(attention_mask=ones(2, 4, 3, 4))), ((q, k, v), dict(attention_mask=ones(3, 1, 1, 5))),
                     ((q, k, v), dict(attention_mask=ones(1, 2, 4, 3, 5))), ((q, k, v), dict(attention_mask=ones(5).cpu())),
                     ((q, k, v), dict(out=q[:1])), ((q, k, v), dict(out=q.half())),
                     ((q, k, v), dict(lse=torch.empty(2, 4, 2, device="cuda"))), ((q[0], k[0], v[0]), dict(kv_lens=lens))):
        with pytest.raises(ValueError):
            ops.cross_attention(*args, **kw)


@pytest.mark.gpu
def test_kernel_layouts(native):
    B, H, Sq, Sk, D = 2, 6, 200, 300, 64
    q, k, v = _inputs(B, H, H, Sq, Sk, D, torch.bfloat16, "cuda")
    want = ops.cross_attention(q, k, v, scale=0.125)
    assert torch.equal(ops.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), scale=0.125), want)
    odd = torch.empty(B, H, Sq, D + 3, device="cuda", dtype=q.dtype)[..., 1:D + 1]  # rows no copy engine addresses
    odd.copy_(q)
    assert torch.equal(ops.cross_attention(odd, k, v, scale=0.125), want)
    res = torch.full((B, H, Sq, D + 3), 7.0, device="cuda", dtype=q.dtype)
    ops.cross_attention(q, k, v, scale=0.125, out=res[..., 1:D + 1])
    assert torch.equal(res[..., 1:D + 1], want) and bool((res[..., D + 1:] == 7).all() and (res[..., 0] == 7).all())
    one_k, one_v = k[:, :1].expand(B, H, Sk, D), v[:, :1].expand(B, H, Sk, D)  # repeated heads and batch rows
    assert torch.equal(ops.cross_attention(q, one_k, one_v, scale=0.125), ops.cross_attention(q, k[:, :1], v[:, :1], scale=0.125))
    rep_k, rep_v = k[:1].expand(B, H, Sk, D), v[:1].expand(B, H, Sk, D)
    assert torch.equal(ops.cross_attention(q, rep_k, rep_v, scale=0.125)[1], ops.cross_attention(q[1:], k[:1], v[:1], scale=0.125)[0])
    folded = ops.cross_attention(q[0], k[0], v[0], scale=0.125)
    assert torch.equal(folded, want[0])
    m = torch.rand(Sk, Sq, device="cuda").t() < 0.5  # a transposed mask, and one shared by all
    a = ops.cross_attention(q, k, v, scale=0.125, attention_mask=m)
    assert torch.equal(a, ops.cross_attention(q, k, v, scale=0.125, attention_mask=m.contiguous().expand(B, H, Sq, Sk).contiguous()))
    bias = torch.randn(Sk + 1, Sq, device="cuda")[1:].t()
    a = ops.cross_attention(q, k, v, scale=0.125, attention_mask=bias)
    assert torch.equal(a, ops.cross_attention(q, k, v, scale=0.125, attention_mask=bias.contiguous()))
    assert torch.equal(ops.cross_attention(-q, k, v, scale=-0.125), want)
    assert ops.cross_attention(q[:, :, :0], k, v).shape == (B, H, 0, D)
    lse = torch.empty(B, H, Sq, device="cuda")
    assert bool((ops.cross_attention(q, k[:, :, :0], v[:, :, :0], lse=lse) == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.gpu
def test_attention_takes_the_kernel(native):
    """``attention`` with a mask, per-query windows or head dim 64, and the models' head-dim-64 entry."""
    B, H, Sq, Sk, D = 2, 4, 150, 260, 128
    q, k, v = _inputs(B, H, H, Sq, Sk, D, torch.bfloat16, "cuda")
    lo = torch.randint(0, 100, (B, 1, Sq, 1), device="cuda")
    win = (torch.arange(Sk, device="cuda") >= lo) & (torch.arange(Sk, device="cuda") < lo + 90)
    n = F.LAUNCHES[0]
    o = ops.attention(q, k, v, scale=0.1, bound_min=lo, bound_max=lo + 90)
    assert F.LAUNCHES[0] == n + 1
    _check(o, _ref(q, k, v, 0.1, win), q.dtype, D, Sk, v.abs().max().item())
    q, k, v = _inputs(B, H, H, Sq, Sk, 64, torch.bfloat16, "cuda")
    hi = torch.tensor([260, 31], device="cuda", dtype=torch.int32)
    _check(F.attention(q, k, v, 0.1, kv_lo=torch.zeros_like(hi), kv_hi=hi), _ref(q, k, v, 0.1, lens=hi), q.dtype, 64, Sk,
           v.abs().max().item())
    _check(ops.attention(q, k, v, scale=0.1), _ref(q, k, v, 0.1), q.dtype, 64, Sk, v.abs().max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gradients_stay_on_the_torch_path(native, D):
    """Inputs that ask for gradients keep the differentiable path, and get the formula's gradients."""
    q, k, v = (t.detach().requires_grad_() for t in _inputs(2, 2, 2, 20, 33, D, torch.bfloat16, "cuda"))
    m = torch.rand(2, 1, 20, 33, device="cuda") < 0.7
    m[..., 0] = True
    w = torch.randn(2, 2, 20, D, device="cuda")
    ref = [t.detach().double().requires_grad_() for t in (q, k, v)]
    z = (ref[0] @ ref[1].transpose(2, 3) * 0.1).masked_fill(~m, -math.inf)
    want = torch.autograd.grad(((z.softmax(-1) @ ref[2]) * w.double()).sum(), ref)
    for fn in (ops.cross_attention, ops.attention):
        got = torch.autograd.grad((fn(q, k, v, scale=0.1, attention_mask=m) * w).sum(), (q, k, v))
        for a, b in zip(got, want):  # the library's bf16 products: a few roundings (2^-8) of the largest value
            assert (a.double() - b).abs().max() <= 2.0 ** -5 * b.abs().max()
    with torch.no_grad():
        o = ops.cross_attention(q, k, v, scale=0.1, attention_mask=m)
    _check(o, _ref(q.detach(), k.detach(), v.detach(), 0.1, m), q.dtype, D, 33, v.abs().max().item())


@pytest.mark.gpu
def test_kernel_unusual_masks_and_lengths(native):
    B, H, Sq, Sk, D = 2, 2, 40, 50, 64
    q, k, v = _inputs(B, H, H, Sq, Sk, D, torch.bfloat16, "cuda")
    all_keys = ops.cross_attention(q, k, v, scale=0.1)
    for lens in (torch.tensor([1 << 40, 50]), torch.tensor([50, 99], dtype=torch.int16)):  # any integers, any device
        assert torch.equal(ops.cross_attention(q, k, v, scale=0.1, kv_lens=lens), all_keys)
    assert bool((ops.cross_attention(q, k, v, scale=0.1, kv_lens=torch.tensor([-3, 0])) == 0).all())
    m = torch.rand(B, 1, Sq, Sk, device="cuda") < 0.5
    want = ops.cross_attention(q, k, v, scale=0.1, attention_mask=m)
    assert torch.equal(ops.cross_attention(q, k, v, scale=0.1, attention_mask=m.int()), want)
    low = torch.zeros(m.shape, device="cuda", dtype=torch.float64).masked_fill(~m, torch.finfo(torch.float64).min)
    low[:, :, 3] = torch.finfo(torch.float64).min  # a row at the lowest value everywhere: the mean of the values
    o = ops.cross_attention(q, k, v, scale=0.1, attention_mask=low)
    mean = v.double().mean(2)
    assert bool(((o[:, :, 3].double() - mean).abs() <= 2.0 ** -7 * (mean.abs() + v.double().abs().mean(2))).all())
    keep = torch.arange(Sq, device="cuda") != 3
    assert torch.allclose(o[:, :, keep].float(), want[:, :, keep].float(), atol=2.0 ** -6)
    assert torch.equal(ops.cross_attention(q, k, v, scale=0.1, attention_mask=torch.tensor(True, device="cuda")), all_keys)
    big = _inputs(70000, 1, 1, 1, 3, 64, torch.bfloat16, "cuda")  # more batch rows than a grid axis holds
    o = ops.cross_attention(*big, scale=0.1)
    _check(o, _ref(*big, 0.1), q.dtype, 64, 3, big[2].abs().max().item())
    same = q.contiguous()
    got = ops.cross_attention(same, k, v, scale=0.1, out=same)  # in place of the queries
    assert got is same and torch.equal(got, all_keys)


@pytest.mark.gpu
def test_kernel_graph_and_streams(native):
    q, k, v = _inputs(2, 4, 2, 333, 500, 128, torch.bfloat16, "cuda")
    m = torch.rand(2, 1, 333, 500, device="cuda") < 0.5
    run = lambda: ops.cross_attention(q, k, v, scale=0.1, attention_mask=m)  # noqa: E731
    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for st in streams:  # calls in flight at once
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cap = run()
    m.copy_(torch.rand(2, 1, 333, 500, device="cuda") < 0.3)
    q.copy_(torch.randn_like(q))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(cap, run())
