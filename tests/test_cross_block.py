"""The operators together, as a cross-attention sub-layer of a batch of requests uses them:
residual norm -> q projection with each request's adapter -> attention to its encoder states ->
output projection with adapter, gated onto the residual; beside it the MXFP8 projection fed by the norm."""

import pytest
import torch

from difflet_b200 import ops
from difflet_b200.ops import fused as F


def _setup(device, dtype, B=3, S=70, D=256, H=4, L=40, Dk=96):
    g = torch.Generator().manual_seed(0)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(device, dtype)  # noqa: E731
    p = dict(x=r(B, S, D), h=r(B, S, D), nw=1 + r(D, std=0.1), text=r(B, L, Dk), wq=r(D, D, std=D ** -0.5), bq=r(D, std=0.1),
             wkv=r(2 * D, Dk, std=Dk ** -0.5), wo=r(D, D, std=D ** -0.5), bo=r(D, std=0.1))
    p["scale"], p["shift"], p["gate"] = (0.2 * torch.randn(3, B, D, generator=g)).to(device)
    p["Aq"], p["Bq"] = [r(k, D, std=D ** -0.5) for k in (4, 16)], [r(D, k, std=0.5) for k in (4, 16)]
    p["Ao"], p["Bo"] = [r(k, D, std=D ** -0.5) for k in (4, 16)], [r(D, k, std=0.5) for k in (4, 16)]
    return p, torch.tensor([1, -1, 0], device=device), torch.tensor([40, 7, 0], device=device)


def _layer(p, ids, lens, H=4):
    B, S, D = p["x"].shape
    dh = D // H
    bq, bo = ops.LoraBank(p["Aq"], p["Bq"], [0.5, 2.0]), ops.LoraBank(p["Ao"], p["Bo"])
    n, h = ops.add_rms_norm(p["x"], p["h"], p["nw"], scale=p["scale"], shift=p["shift"], rows_per_batch=S)
    q = ops.linear_lora(n, p["wq"], p["bq"], bank=bq, ids=ids, rows_per_batch=S).view(B, S, H, dh).permute(0, 2, 1, 3)
    kv = F.linear(p["text"].reshape(-1, p["text"].shape[-1]), p["wkv"]).view(B, -1, 2, H, dh)
    o = torch.empty(B, S, D, device=q.device, dtype=q.dtype)
    ops.cross_attention(q, kv[:, :, 0].permute(0, 2, 1, 3), kv[:, :, 1].permute(0, 2, 1, 3), scale=dh ** -0.5, kv_lens=lens,
                        out=o.view(B, S, H, dh).permute(0, 2, 1, 3))
    return ops.linear_lora(o, p["wo"], p["bo"], bank=bo, ids=ids, rows_per_batch=S, gate=p["gate"], resid=h, out=h)


def _formula(p, ids, lens, H=4):
    B, S, D = p["x"].shape
    p = {k: [t.double() for t in v] if isinstance(v, list) else v.double() for k, v in p.items()}
    h = p["x"] + p["h"]
    n = h / (h.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * p["nw"] * (1 + p["scale"][:, None]) + p["shift"][:, None]

    def proj(v, w, b, A, Bm, s):
        y = v @ w.t() + b
        for i, a in enumerate(ids.tolist()):
            if a >= 0:
                y[i] += s[a] * (v[i] @ A[a].t() @ Bm[a].t())
        return y

    q = proj(n, p["wq"], p["bq"], p["Aq"], p["Bq"], [0.5, 2.0]).view(B, S, H, -1).transpose(1, 2)
    kv = (p["text"] @ p["wkv"].t()).view(B, -1, 2, H, D // H)
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    o = torch.zeros_like(q)
    for i, L in enumerate(lens.tolist()):
        if L:
            o[i] = torch.softmax(q[i] @ k[i, :, :L].transpose(1, 2) * (D // H) ** -0.5, -1) @ v[i, :, :L]
    o = o.transpose(1, 2).reshape(B, S, D)
    return h + p["gate"][:, None] * proj(o, p["wo"], p["bo"], p["Ao"], p["Bo"], [1.0, 1.0])


def test_layer_oracle():
    p, ids, lens = _setup("cpu", torch.float32)
    want = _formula(p, ids, lens)
    assert torch.allclose(_layer(p, ids, lens).double(), want, atol=1e-4)


@pytest.mark.gpu
def test_layer_kernels_and_graph(native):
    p, ids, lens = _setup("cuda", torch.bfloat16)
    # ~8 roundings to bf16 (2^-8 each) stand between the inputs and the residual sum, whose values are of order 3
    want = _formula(p, ids, lens)
    tol = 8 * 2.0 ** -8 * want.abs().max()
    got = _layer(p, ids, lens)
    assert bool(((got.double() - want).abs() <= tol).all())
    bq, bo = ops.LoraBank(p["Aq"], p["Bq"], [0.5, 2.0]), ops.LoraBank(p["Ao"], p["Bo"])
    B, S, D = p["x"].shape

    def step():
        n, h = ops.add_rms_norm(p["x"], p["h"], p["nw"], scale=p["scale"], shift=p["shift"], rows_per_batch=S)
        q = ops.linear_lora(n, p["wq"], p["bq"], bank=bq, ids=ids, rows_per_batch=S).view(B, S, 4, 64).permute(0, 2, 1, 3)
        kv = F.linear(p["text"].reshape(-1, 96), p["wkv"]).view(B, -1, 2, 4, 64)
        o = ops.cross_attention(q, kv[:, :, 0].permute(0, 2, 1, 3), kv[:, :, 1].permute(0, 2, 1, 3), scale=0.125, kv_lens=lens)
        return ops.linear_lora(o.permute(0, 2, 1, 3).reshape(B, S, D), p["wo"], p["bo"], bank=bo, ids=ids, rows_per_batch=S,
                               gate=p["gate"], resid=h)

    assert torch.equal(step(), got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cap = step()
    p["x"].copy_(torch.randn_like(p["x"]))
    lens.copy_(torch.tensor([3, 40, 11]))
    ids.copy_(torch.tensor([0, 0, 1]))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(cap, step())


def test_dispatcher_ops():
    from difflet_b200.ops import library  # noqa: F401  (registers the ops)

    g = torch.Generator().manual_seed(0)
    x, r, w = torch.randn(5, 32, generator=g), torch.randn(5, 32, generator=g), torch.randn(32, generator=g)
    y, s = torch.ops.difflet.add_rms_norm(x, r, w)
    want = ops.add_rms_norm(x, r, w)
    assert torch.equal(y, want[0]) and torch.equal(s, want[1])
    q, k = torch.randn(2, 4, 3, 16, generator=g), torch.randn(2, 2, 7, 16, generator=g)
    lens = torch.tensor([7, 2])
    assert torch.equal(torch.ops.difflet.cross_attention(q, k, k, 0.25, None, lens), ops.cross_attention(q, k, k, scale=0.25, kv_lens=lens))
    for op, args in ((torch.ops.difflet.add_rms_norm, (x, r, w)), (torch.ops.difflet.cross_attention, (q, k, k, 0.25, None, lens))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_norm_feeds_both_projections(native):
    """One residual norm in bf16 for the adapters and one in MXFP8 for the block-scaled projection agree."""
    p, ids, _ = _setup("cuda", torch.bfloat16)
    w = F.MXWeight.quantize(p["wq"])
    n, h = ops.add_rms_norm(p["x"], p["h"], p["nw"])
    (q, sf), h8 = ops.add_rms_norm(p["x"], p["h"], p["nw"], quantize="float8_e4m3fn", blocked=True)
    assert torch.equal(h, h8)
    y8 = F.linear_mx(q.view(-1, 256), sf, w.q, w.sf, p["bq"]).double()
    y = n.view(-1, 256).double() @ p["wq"].double().t() + p["bq"].double()
    # E4M3 on both sides (2^-4 each, 2^-3 where a block's largest value saturates)
    size = n.view(-1, 256).double().abs() @ p["wq"].double().abs().t()
    assert bool(((y8 - y).abs() <= 2.0 ** -2 * size).all())
    assert (y8 - y).norm() <= 2.0 ** -4 * y.norm()
