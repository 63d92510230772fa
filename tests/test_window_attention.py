"""``ops.window_attention`` (causal, the last ``window`` and the first ``sinks`` keys) against 64 bits; tolerances as in
test_cross_attention.py."""

import math

import pytest
import torch

from difflet_b200 import ops
from difflet_b200.ops import fused as F
from test_cross_attention import _check, _inputs, _ref

BF, HF = torch.bfloat16, torch.float16


def _mask(B, Sq, Sk, window, sinks, lens, start):
    """[B, 1, Sq, Sk], one comparison at a time."""
    m = torch.zeros(B, 1, Sq, Sk, dtype=torch.bool)
    j = torch.arange(Sk)
    for b in range(B):
        n = min(max(int(lens[b]), 0), Sk)
        for i in range(Sq):
            p = int(start[b]) + i
            m[b, 0, i] = (j < n) & (j <= p) & ((j > p - window) | (j < sinks))
    return m


def _args(B, Sq, Sk, form, seed=0):
    g = torch.Generator().manual_seed(seed)
    if form == "all":  # (the newest keys are the queries' own)
        return [Sk] * B, [Sk - Sq] * B, {}
    if form == "cache":
        lens = torch.randint(min(Sq, Sk), Sk + 1, (B,), generator=g)
        return lens.tolist(), (lens - Sq).tolist(), dict(kv_lens=lens)
    if form == "prompt":
        lens = torch.randint(0, Sk + 1, (B,), generator=g)
        return lens.tolist(), [0] * B, dict(kv_lens=lens, q_start=0)
    start = torch.randint(-Sq, Sk + 40, (B,), generator=g)  # anywhere
    lens = torch.randint(0, Sk + 1, (B,), generator=g)
    return lens.tolist(), start.tolist(), dict(kv_lens=lens, q_start=start)


def _on(kw, device):
    return {k: v.to(device) if torch.is_tensor(v) else v for k, v in kw.items()}


# ----------------------------------------------------------------------------- CPU
@pytest.mark.parametrize("form", ["all", "cache", "prompt", "any"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (100, 0), (5, 100)])
def test_oracle(form, window, sinks):
    B, H, Hk, Sq, Sk, D = 3, 4, 2, 6, 17, 8
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, torch.float64, "cpu")
    lens, start, kw = _args(B, Sq, Sk, form)
    m = _mask(B, Sq, Sk, window, sinks, lens, start)
    lse = torch.empty(B, H, Sq, dtype=torch.float64)
    want, lse_ref, _, _ = _ref(q, k, v, 0.3, m)
    k, v = k.clone(), v.clone()
    unseen = ~m.any(2)[:, 0]  # [B, Sk]
    for t in (k, v):
        t.transpose(1, 2)[unseen] = float("nan")
    o = ops.window_attention(q, k, v, window=window, sinks=sinks, scale=0.3, lse=lse, **kw)
    assert torch.allclose(o, want, atol=1e-12) and torch.allclose(lse, lse_ref, atol=1e-12)
    assert bool((o.transpose(1, 2)[~m.any(-1)[:, 0]] == 0).all())


def test_plain_causal_and_gradients_on_cpu():
    q, k, v = (t.contiguous().requires_grad_() for t in _inputs(2, 2, 1, 5, 5, 4, torch.float64, "cpu"))
    o = ops.window_attention(q, k, v, window=5, scale=0.5)
    want = torch.nn.functional.scaled_dot_product_attention(q, k.expand(2, 2, 5, 4), v.expand(2, 2, 5, 4), is_causal=True, scale=0.5)
    assert torch.allclose(o, want)
    assert torch.autograd.gradcheck(lambda *t: ops.window_attention(*t, window=2, sinks=1, scale=0.5), (q, k, v))


def test_refusals():
    q, k, v = _inputs(2, 4, 2, 3, 9, 16, torch.float32, "cpu")
    for kw in (dict(window=0), dict(window=2, sinks=-1), dict(window=2, kv_lens=torch.ones(2)), dict(window=2, kv_lens=torch.tensor([1])),
               dict(window=2, q_start=torch.tensor([0, 1, 2])), dict(window=2, out=torch.empty(2, 4, 3, 8)),
               dict(window=2, lse=torch.empty(3))):
        with pytest.raises(ValueError):
            ops.window_attention(q, k, v, **kw)
    for bad in ((q, k, v[:, :, :-1]), (q[0], k, v), (q, k.double(), v), (q[:, :3], k, v), (q[:1], k, v)):
        with pytest.raises(ValueError):
            ops.window_attention(*bad, window=2)


# ----------------------------------------------------------------------------- kernels
CASES = [  # B, H, Hk, Sq, Sk, window, sinks
    (1, 1, 1, 1, 1, 1, 0), (2, 4, 2, 1, 300, 64, 4), (3, 8, 2, 1, 2000, 700, 0), (2, 6, 6, 2, 90, 33, 40), (1, 16, 1, 1, 513, 512, 1),
    (2, 8, 2, 5, 700, 130, 3), (1, 12, 12, 17, 1300, 1000, 100), (2, 2, 1, 40, 40, 7, 0), (2, 3, 3, 128, 128, 128, 0), (1, 4, 4, 129, 385, 1, 1),
    (3, 4, 1, 300, 300, 50, 3), (1, 2, 2, 700, 1500, 300, 200), (1, 40, 40, 513, 700, 129, 128), (2, 16, 4, 1021, 1021, 255, 1),
    (1, 24, 24, 900, 900, 10 ** 6, 0), (1, 3, 1, 257, 260, 128, 255), (5, 7, 7, 33, 64, 20, 70),
    (1, 4, 4, 300, 6000, 4000, 200), (1, 6, 2, 200, 3000, 2500, 0), (2, 2, 1, 384, 2100, 2000, 1), (1, 1, 1, 1025, 1300, 700, 129),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", CASES)
def test_kernels(native, case, D, dtype):
    B, H, Hk, Sq, Sk, window, sinks = case
    q, k, v = _inputs(B, H, Hk, Sq, Sk, D, dtype, "cuda")
    for form in ("all", "cache", "prompt", "any"):
        lens, start, kw = _args(B, Sq, Sk, form)
        m = _mask(B, Sq, Sk, window, sinks, lens, start).cuda()
        ref = _ref(q, k, v, D ** -0.5, m)
        lse = torch.empty(B, H, Sq, device="cuda")
        kn, vn = k.clone(), v.clone()
        for t in (kn, vn):  # what no query sees may be anything
            t.transpose(1, 2)[~m.any(2)[:, 0]] = float("nan")
        o = ops.window_attention(q, kn, vn, window=window, sinks=sinks, scale=D ** -0.5, lse=lse, **_on(kw, "cuda"))
        _check(o, ref, dtype, D, Sk, v.abs().max().item(), lse)
        assert bool((o.transpose(1, 2)[~m.any(-1)[:, 0]] == 0).all())


@pytest.mark.gpu
def test_long_offsets(native):
    """A cache whose offsets pass 32 bits: 2 x 8 heads x 1,200,000 keys x 128."""
    Sk, window, sinks = 1_200_000, 300, 5
    g = torch.Generator(device="cuda").manual_seed(0)
    k = torch.empty(2, 8, Sk, 128, device="cuda", dtype=BF)
    k.view(torch.int16).fill_(0x7fff)  # NaN but for what is seen
    v = k.clone()
    lens = torch.tensor([Sk, 700_001], device="cuda")
    for Sq in (1, 200):
        q = torch.randn(2, 8, Sq, 128, device="cuda", generator=g).to(BF)
        want, kk, vv = [], [], []
        for b, n in enumerate(lens.tolist()):
            near = slice(n - Sq - window + 1, n)
            for t in (k, v):
                t[b, :, near] = torch.randn(8, Sq + window - 1, 128, device="cuda", generator=g).to(BF)
                t[b, :, :sinks] = torch.randn(8, sinks, 128, device="cuda", generator=g).to(BF)
            kk.append(torch.cat([k[b, :, :sinks], k[b, :, near]], 1))
            vv.append(torch.cat([v[b, :, :sinks], v[b, :, near]], 1))
        n = Sq + window - 1
        i, j = torch.arange(Sq, device="cuda")[:, None], torch.arange(sinks + n, device="cuda") - sinks
        m = ((j < 0) | ((j >= i) & (j < i + window)))[None, None]
        ref = _ref(q, torch.stack(kk), torch.stack(vv), 0.09, m)
        o = ops.window_attention(q, k, v, window=window, sinks=sinks, scale=0.09, kv_lens=lens)
        _check(o, ref, BF, 128, sinks + n, 6.0)
        k.view(torch.int16).fill_(0x7fff)
        v.view(torch.int16).fill_(0x7fff)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [2, 300])
def test_lengths_and_starts_of_any_kind(native, Sq):
    q, k, v = _inputs(2, 4, 4, Sq, 400, 64, BF, "cuda")
    call = lambda **kw: ops.window_attention(q, k, v, window=90, sinks=3, scale=0.1, **kw)  # noqa: E731
    want = call(kv_lens=torch.tensor([400, 350], device="cuda"))
    for t in (torch.int32, torch.int64, torch.int16):
        for dev in ("cuda", "cpu"):
            assert torch.equal(call(kv_lens=torch.tensor([400, 350], dtype=t, device=dev)), want)
    assert torch.equal(call(kv_lens=torch.tensor([2 ** 40, 350], device="cuda")), want)
    assert torch.equal(call(kv_lens=torch.tensor([400, 350]), q_start=torch.tensor([400 - Sq, 350 - Sq])), want)
    zero = torch.zeros_like(want)
    assert torch.equal(call(kv_lens=torch.tensor([0, -5])), zero)
    for far in (-(2 ** 31), -(2 ** 62), -Sq):  # no query has reached a key
        assert torch.equal(call(q_start=torch.tensor([far, far])), zero)
    only_sinks = ops.window_attention(q, k[:, :, :3], v[:, :, :3], window=3, scale=0.1, q_start=2 ** 20)  # none: the window has passed
    assert not bool(only_sinks.any())
    for far in (1000, 2 ** 31 - 1, 2 ** 62):  # the window has passed every key but the sinks
        got = call(q_start=torch.tensor([far, far]))
        ref = _ref(q, k[:, :, :3], v[:, :, :3], 0.1)
        _check(got, ref, BF, 64, 3, 6.0)
    assert torch.equal(ops.window_attention(q, k, v, window=2 ** 62, sinks=2 ** 62, scale=0.1), ops.window_attention(q, k, v, window=400, scale=0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 150])
def test_layouts(native, Sq):
    q, k, v = _inputs(2, 4, 2, Sq, 260, 64, BF, "cuda")
    kw = dict(window=100, sinks=2, scale=0.2, kv_lens=torch.tensor([260, 200], device="cuda"))
    want = ops.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), **kw)
    assert torch.equal(ops.window_attention(q, k, v, **kw), want)
    wide = torch.zeros(2, 2, 260, 80, device="cuda", dtype=BF)
    for off in (0, 8, 3):
        wide[..., off:off + 64] = k
        assert torch.equal(ops.window_attention(q, wide[..., off:off + 64], v, **kw), want)
    out = torch.full((2, Sq, 4, 64), 7.0, device="cuda", dtype=BF)
    o = ops.window_attention(q, k, v, out=out.transpose(1, 2), **kw)
    assert o.data_ptr() == out.data_ptr() and torch.equal(out.transpose(1, 2), want)
    odd = torch.zeros(2, 4, Sq, 65, device="cuda", dtype=BF)[..., :64]
    assert torch.equal(ops.window_attention(q, k, v, out=odd, **kw), want)
    lse = torch.empty(2, 4, Sq, device="cuda")
    ops.window_attention(q, k, v, lse=lse, **kw)
    for other in (torch.empty(2, 4, Sq, device="cuda", dtype=torch.float64), torch.empty(2, 4, 2 * Sq, device="cuda")[..., ::2]):
        ops.window_attention(q, k, v, lse=other, **kw)
        assert torch.equal(other.float(), lse)
    one = ops.window_attention(q, k[:, :1].expand(2, 2, 260, 64), v[:, :1].expand(2, 2, 260, 64), **kw)
    assert torch.equal(one, ops.window_attention(q, k[:, :1], v[:, :1], **kw))
    for s in (-0.2, 0.0):
        neg = ops.window_attention(q, k, v, **{**kw, "scale": s})
        if s:
            assert torch.equal(neg, ops.window_attention(-q, k, v, **kw))
        else:
            assert bool(neg.isfinite().all())


@pytest.mark.gpu
def test_off_the_kernel(native):
    """Other head dims and types, and inputs that ask for gradients: the same mask on the torch path (values below 4 and
    gradients through at most eight roundings of 2^-8)."""
    for D, dtype in ((32, BF), (96, HF), (64, torch.float32)):
        q, k, v = _inputs(2, 4, 2, 9, 30, D, dtype, "cuda")
        lens, start, kw = _args(2, 9, 30, "cache")
        m = _mask(2, 9, 30, 8, 2, lens, start).cuda()
        ref = _ref(q, k, v, 0.1, m)[0]
        got = ops.window_attention(q, k, v, window=8, sinks=2, scale=0.1, **_on(kw, "cuda"))
        assert got.dtype == dtype and bool(((got.double() - ref).abs() <= 8 * 2.0 ** -8 * 4).all())
    q, k, v = (t.contiguous().requires_grad_() for t in _inputs(1, 2, 2, 20, 20, 64, BF, "cuda"))
    o = ops.window_attention(q, k, v, window=8, scale=0.1)
    grads = torch.autograd.grad(o.float().square().sum(), (q, k, v))
    d = [t.detach().double().requires_grad_() for t in (q, k, v)]
    m = _mask(1, 20, 20, 8, 0, [20], [0]).cuda()
    z = (d[0] @ d[1].transpose(2, 3) * 0.1).masked_fill(~m, -math.inf)
    want = torch.autograd.grad((torch.softmax(z, -1) @ d[2]).square().sum(), d)
    for a, b in zip(grads, want):
        assert (a.double() - b).norm() <= 2 ** -5 * b.norm()
    assert ops.window_attention(q.detach()[:, :, :0], k.detach(), v.detach(), window=3).shape == (1, 2, 0, 64)
    none = ops.window_attention(q.detach(), k.detach()[:, :, :0], v.detach()[:, :, :0], window=3)
    assert none.shape == (1, 2, 20, 64) and not bool(none.any())


@pytest.mark.gpu
@pytest.mark.parametrize("Sq", [1, 4, 200])
def test_captured(native, Sq):
    q, k, v = _inputs(2, 8, 2, Sq, 900, 128, BF, "cuda")
    lens = torch.tensor([900, 500], device="cuda", dtype=torch.int32)
    call = lambda: ops.window_attention(q, k, v, window=333, sinks=4, scale=0.1, kv_lens=lens)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    lens.copy_(torch.tensor([610, 899]))
    q.copy_(q.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, call())


def test_window_of_everything_is_the_masked_attention_on_cpu():
    q, k, v = _inputs(2, 4, 4, 6, 6, 16, torch.float32, "cpu")
    m = torch.ones(6, 6, dtype=torch.bool).tril()
    assert torch.allclose(ops.window_attention(q, k, v, window=6, scale=0.2), F.cross_attention(q, k, v, 0.2, mask=m[None, None]), atol=1e-6)
