"""The lookup, the windowed attention and the gated projection as a decoder layer of a prompt encoder uses them, beside the residual
norm: prompts read at once, then continued token by token over a cache; learned embeddings and feed-forward weights.  Calls in
flight on several streams and graphs replayed at once keep apart."""

import pytest
import torch

from difflet_b200 import ops
from difflet_b200.ops import fused as F

BF, HF = torch.bfloat16, torch.float16
H, HK, DH, D, FF, V = 4, 2, 64, 256, 520, 300
WINDOW, SINKS = 20, 3


def _weights(device, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(device, dtype)  # noqa: E731
    return dict(emb=r(V, D, std=D ** -0.5), n1=1 + r(D, std=0.1), n2=1 + r(D, std=0.1), qkv=r((H + 2 * HK) * DH, D, std=D ** -0.5),
                o=r(D, H * DH, std=(H * DH) ** -0.5), gate=r(FF, D, std=D ** -0.5), up=r(FF, D, std=D ** -0.5), down=r(D, FF, std=FF ** -0.5))


def _linear(x, w):
    return F.linear(x.reshape(-1, x.shape[-1]), w).view(*x.shape[:-1], w.shape[0])


def _layer(p, ids, cache, pos, lens):
    """One layer over ids [B, S] at positions pos .. pos + S; keys and values go to cache [2, B, HK, Smax, DH]."""
    B, S = ids.shape
    x = ops.embedding(ids, p["emb"], scale=D ** 0.5)
    n, _ = ops.add_rms_norm(x, None, p["n1"])
    q, k, v = _linear(n, p["qkv"]).view(B, S, H + 2 * HK, DH).permute(0, 2, 1, 3).split([H, HK, HK], 1)
    cache[0, :, :, pos:pos + S], cache[1, :, :, pos:pos + S] = k, v
    o = ops.window_attention(q, cache[0], cache[1], window=WINDOW, sinks=SINKS, scale=DH ** -0.5, kv_lens=lens, q_start=pos)
    n, x = ops.add_rms_norm(_linear(o.permute(0, 2, 1, 3).reshape(B, S, H * DH), p["o"]), x, p["n2"])
    return x + _linear(ops.gated_linear(n, p["gate"], p["up"]), p["down"])


def _formula(p, ids, lens):
    p = {n: t.double() for n, t in p.items()}
    norm = lambda t, w: t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w  # noqa: E731
    B, S = ids.shape
    x = p["emb"][ids] * D ** 0.5
    q, k, v = (norm(x, p["n1"]) @ p["qkv"].t()).view(B, S, H + 2 * HK, DH).transpose(1, 2).split([H, HK, HK], 1)
    k, v = k.repeat_interleave(H // HK, 1), v.repeat_interleave(H // HK, 1)
    i, j = torch.arange(S, device=ids.device)[:, None], torch.arange(S, device=ids.device)
    seen = ((j <= i) & ((j > i - WINDOW) | (j < SINKS)))[None] & (j < lens[:, None, None])
    z = (q @ k.transpose(2, 3) * DH ** -0.5).masked_fill(~seen[:, None], -1e30)
    x = x + (torch.softmax(z, -1) @ v).transpose(1, 2).reshape(B, S, H * DH) @ p["o"].t()
    n = norm(x, p["n2"])
    return x + (torch.nn.functional.silu(n @ p["gate"].t()) * (n @ p["up"].t())) @ p["down"].t()


def _setup(device, dtype):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (2, 90), generator=g).to(device)
    return _weights(device, dtype), ids, torch.zeros(2, 2, HK, 96, DH, device=device, dtype=dtype)


def test_layer_oracle():
    p, ids, cache = _setup("cpu", torch.float32)
    lens = torch.tensor([90, 90])
    want = _formula(p, ids, lens)
    assert torch.allclose(_layer(p, ids, cache, 0, lens).double(), want, atol=1e-4)
    steps = torch.cat([_layer(p, ids[:, i:i + 1], cache.zero_() if i == 0 else cache, i, torch.full((2,), i + 1)) for i in range(90)], 1)
    assert torch.allclose(steps.double(), want, atol=1e-4)


@pytest.mark.gpu
def test_layer_kernels_and_graph(native):
    p, ids, cache = _setup("cuda", BF)
    lens = torch.tensor([90, 90], device="cuda")
    want = _formula(p, ids, lens)
    # ~10 roundings to bf16 (2^-8 each) stand between the embeddings and the sum, whose values are of order 3
    tol = 10 * 2.0 ** -8 * want.abs().max()
    got = _layer(p, ids, cache, 0, lens)
    assert bool(((got.double() - want).abs() <= tol).all())
    first = cache.clone()
    cache.fill_(float("nan"))  # (what lies behind a row's length is not used)
    for i in range(0, 90, 9):  # continued token by token, or in chunks of a few
        n = 1 if i % 2 else 9
        for c in range(i, i + 9, n):
            step = _layer(p, ids[:, c:c + n], cache, c, torch.full((2,), c + n, device="cuda"))
            assert bool(((step.double() - want[:, c:c + n]).abs() <= tol).all())
    assert torch.allclose(cache[:, :, :, :90], first[:, :, :, :90], atol=2.0 ** -6)
    graph = torch.cuda.CUDAGraph()
    call = lambda: _layer(p, ids, cache, 0, lens)  # noqa: E731
    call()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call()
    ids.copy_(ids.flip(1))
    lens.copy_(torch.tensor([90, 41]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call())


@pytest.mark.gpu
def test_learned_prompt(native):
    """Gradients of the table and of the feed-forward weights through the two operators that record them."""
    p, ids, _ = _setup("cuda", BF)
    dy = torch.randn(2, 90, D, device="cuda").to(BF)
    leaves = [p[n].clone().requires_grad_() for n in ("emb", "gate", "up")]

    def step(emb, gate, up):
        x = ops.embedding(ids, emb, scale=D ** 0.5, padding_idx=0)
        return torch.nn.functional.linear(ops.gated_linear(x, gate, up, act="gelu"), p["down"])

    got = torch.autograd.grad(step(*leaves), leaves, dy)
    d = [t.detach().double().requires_grad_() for t in leaves]
    x = torch.nn.functional.embedding(ids, d[0], padding_idx=0) * D ** 0.5
    h = torch.nn.functional.gelu(x @ d[1].t(), approximate="tanh") * (x @ d[2].t())
    want = torch.autograd.grad(h @ p["down"].double().t(), d, dy.double())
    for a, b in zip(got, want):  # eight roundings of 2^-8 between dy and a gradient, in the norm
        assert a.dtype == BF and (a.double() - b).norm() <= 8 * 2.0 ** -8 * b.norm()
    assert not bool(got[0][0].any())


# ----------------------------------------------------------------------------- several calls at once
STREAMS = 3


def _gated_calls(M, K, N, grad):
    calls = []
    for i in range(STREAMS):
        g = torch.Generator().manual_seed(i)
        x, wg, wu, dh = (torch.randn(*s, generator=g).to("cuda", BF) * 0.1 for s in ((M, K), (N, K), (N, K), (M, N)))
        if grad:
            t = [v.requires_grad_() for v in (x, wg, wu)]
            calls.append(lambda t=t, dh=dh: torch.cat([v.flatten() for v in torch.autograd.grad(ops.gated_linear(*t), t, dh)]))
        else:
            calls.append(lambda x=x, wg=wg, wu=wu: ops.gated_linear(x, wg, wu))
    return calls


def _embed_calls(n, rows, dim, dtype):
    calls = []
    for i in range(STREAMS):
        g = torch.Generator().manual_seed(i)
        ids = (torch.rand(n, generator=g).pow(4) * rows).long().clamp(max=rows - 1).cuda()
        dy = torch.randn(n, dim, generator=g).to("cuda", dtype)
        calls.append(lambda ids=ids, dy=dy: F.embedding_grad(dy, ids, rows, 2.0, 1))
    return calls


def _window_calls(B, Hq, Hk, Sq, Sk, dim, **kw):
    calls = []
    for i in range(STREAMS):
        g = torch.Generator().manual_seed(i)
        q, k, v = (torch.randn(B, h, s, dim, generator=g).to("cuda", BF) for h, s in ((Hq, Sq), (Hk, Sk), (Hk, Sk)))
        lens = torch.randint(Sk // 2, Sk + 1, (B,), generator=g).cuda()
        calls.append(lambda q=q, k=k, v=v, lens=lens: ops.window_attention(q, k, v, scale=0.1, kv_lens=lens, **kw))
    return calls


CASES = {
    "gated few rows": lambda: _gated_calls(5, 512, 800, False),
    "gated": lambda: _gated_calls(300, 512, 800, False),
    "gated parts": lambda: _gated_calls(64, 4096, 512, False),
    "gated gradients in parts": lambda: _gated_calls(200, 256, 4096, True),
    "embedding gradient": lambda: _embed_calls(5000, 700, 200, torch.float32),
    "window": lambda: _window_calls(2, 8, 2, 600, 700, 64, window=130, sinks=3),
    "window parts": lambda: _window_calls(1, 4, 4, 300, 6000, 128, window=4000, sinks=200),
    "window few queries": lambda: _window_calls(3, 8, 2, 1, 3000, 128, window=900, sinks=4),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(CASES))
def test_calls_in_flight_keep_apart(native, case):
    calls = CASES[case]()
    want = [c() for c in calls]  # one after another
    torch.cuda.synchronize()
    assert not any(torch.equal(want[0], w) for w in want[1:])
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        got = [[] for _ in calls]
        for _ in range(5):
            for st, call, outs in zip(streams, calls, got):
                with torch.cuda.stream(st):
                    outs.append(call())
        torch.cuda.synchronize()
        for outs, w in zip(got, want):
            assert all(torch.equal(o, w) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(CASES))
def test_graphs_replayed_at_once_keep_apart(native, case):
    calls = CASES[case]()
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        want = [c() for c in calls]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in calls], []
    for g, call in zip(graphs, calls):
        with torch.cuda.graph(g):
            outs.append([call() for _ in range(2)])
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for own, w in zip(outs, want):
        assert all(torch.equal(o, w) for o in own)


# ----------------------------------------------------------------------------- other ways to call them
def test_dispatcher_ops():
    from difflet_b200.ops import library  # noqa: F401  (registers the ops)

    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, lens = r(2, 4, 3, 16), r(2, 2, 7, 16), r(2, 2, 7, 16), torch.tensor([7, 4])
    x, wg, wu = r(5, 32), r(24, 32), r(24, 32)
    ids, w = torch.tensor([[1, 2], [0, 1]]), r(3, 8)
    ops_ = torch.ops.difflet
    assert torch.equal(ops_.window_attention(q, k, v, 0.25, 3, 1, lens), ops.window_attention(q, k, v, scale=0.25, window=3, sinks=1, kv_lens=lens))
    assert torch.equal(ops_.gated_linear(x, wg, wu, "gelu"), ops.gated_linear(x, wg, wu, act="gelu"))
    assert torch.equal(ops_.embedding(ids, w, 2.0), ops.embedding(ids, w, scale=2.0))
    for op, args in ((ops_.window_attention, (q, k, v, 0.25, 3, 1, lens)), (ops_.gated_linear, (x, wg, wu)), (ops_.embedding, (ids, w, 2.0))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.gpu
def test_dispatcher_ops_on_the_kernels(native):
    from difflet_b200.ops import library  # noqa: F401

    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to("cuda", BF)  # noqa: E731
    q, k, v = r(2, 4, 30, 64), r(2, 2, 70, 64), r(2, 2, 70, 64)
    x, wg, wu, ids, w = r(50, 32), r(24, 32), r(24, 32), torch.tensor([[1, 2], [0, 1]], device="cuda"), r(3, 8)
    ops_ = torch.ops.difflet
    assert torch.equal(ops_.window_attention(q, k, v, 0.25, 30, 1), ops.window_attention(q, k, v, scale=0.25, window=30, sinks=1))
    assert torch.equal(ops_.gated_linear(x, wg, wu, "gelu"), ops.gated_linear(x, wg, wu, act="gelu"))
    assert torch.equal(ops_.embedding(ids, w, 2.0), ops.embedding(ids, w, scale=2.0))
    with pytest.raises(RuntimeError):  # (no gradient through the dispatcher's form)
        torch.autograd.grad(ops_.gated_linear(x.requires_grad_(), wg, wu).sum(), x)


def test_block_scaled_weights_are_refused():
    w = F.MXWeight.quantize(torch.randn(128, 128))
    with pytest.raises(NotImplementedError):
        ops.gated_linear(torch.randn(2, 128), w, w)


@pytest.mark.gpu
def test_compiled(native):
    """Under tracing the operators are torch operations."""
    p, ids, _ = _setup("cuda", torch.float32)

    @torch.compile(backend="eager")
    def f(ids):
        x = ops.embedding(ids, p["emb"], scale=2.0)
        q = x.view(2, 90, H, DH).transpose(1, 2)
        return ops.gated_linear(ops.window_attention(q, q, q, window=7, scale=0.1).transpose(1, 2).reshape(2, 90, D), p["gate"], p["up"])

    x = p["emb"][ids] * 2.0
    q = x.view(2, 90, H, DH).transpose(1, 2)
    want = F.gated_linear(ops.window_attention(q, q, q, window=7, scale=0.1).transpose(1, 2).reshape(2, 90, D), p["gate"], p["up"])
    assert torch.allclose(f(ids), want, atol=1e-4, rtol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["gated_linear", "embedding"])
def test_capture_beside_a_living_eager_graph(native, name):
    """Gradients cannot be captured while an eager graph of the default stream holds the same leaves: refused before anything is
    recorded, and both passes work afterwards."""
    g = torch.Generator().manual_seed(0)
    if name == "embedding":
        leaves, ids = [torch.randn(50, 64, generator=g).to("cuda", BF)], torch.randint(0, 50, (70,), generator=g).cuda()
        run = lambda: ops.embedding(ids, leaves[0], scale=2.0)  # noqa: E731
    else:
        leaves = [torch.randn(*s, generator=g).to("cuda", BF) for s in ((70, 64), (40, 64), (40, 64))]
        run = lambda: ops.gated_linear(*leaves)  # noqa: E731
    for t in leaves:
        t.requires_grad_()
    y = run()
    dy = torch.ones_like(y)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            run()
    with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
        run()  # (nothing is recorded for gradients)
    want = torch.autograd.grad(y, leaves, dy)
    del y

    def captured():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(run(), leaves, dy)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))

    captured()


@pytest.mark.gpu
def test_rows_that_overlap(native):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1024, generator=g).to("cuda", BF).as_strided((90, 64), (8, 1))  # windows of a signal
    w = torch.randn(700, generator=g).to("cuda", BF).as_strided((40, 64), (16, 1))
    assert torch.equal(ops.gated_linear(x, w, w), ops.gated_linear(x.contiguous(), w.contiguous(), w.contiguous()))
    ids = torch.arange(40, device="cuda").flip(0)
    assert torch.equal(ops.embedding(ids, w), w[ids])
