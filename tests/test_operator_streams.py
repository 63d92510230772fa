"""Calls in flight at once on several streams, and captured graphs replayed at once, each with inputs of its own: a workspace
that two calls shared would mix their tile lists, partial tiles, laid-out masks or windows."""

import pytest
import torch

from difflet_b200 import ops
from test_cross_attention import _inputs, _mask
from test_linear_lora import _make

BF = torch.bfloat16
STREAMS = 3


def _lora_calls(M, N, K, ranks, **kw):
    """One call per stream: other rows, ids and factors, one weight."""
    calls = []
    _, w, b, A, B, _ = _make(M, N, K, ranks, "cuda")
    for i in range(STREAMS):
        g = torch.Generator().manual_seed(10 + i)
        x = torch.randn(M, K, generator=g).to("cuda", BF)
        ids = torch.randint(-1, len(ranks), (M,), generator=g).cuda().int()
        bank = ops.LoraBank(A, B, [float(i + j + 1) for j in range(len(ranks))])
        calls.append(lambda x=x, ids=ids, bank=bank: ops.linear_lora(x, w, b, bank=bank, ids=ids, **kw))
    return calls


def _cross_calls(B, H, Hk, Sq, Sk, D, kind, dtype=BF):
    calls = []
    for i in range(STREAMS):
        q, k, v = _inputs(B, H, Hk, Sq, Sk, D, dtype, "cuda", 20 + i)
        kw = {}
        if kind == "lens":
            kw = dict(kv_lens=torch.randint(1, Sk + 1, (B,), generator=torch.Generator().manual_seed(i)).cuda())
        elif kind:
            m = _mask(kind, B, H, Sq, Sk, "cuda", dtype)
            kw = dict(attention_mask=m.roll(5 * i + 1, -1).contiguous())
        calls.append(lambda q=q, k=k, v=v, kw=kw: ops.cross_attention(q, k, v, scale=0.1, **kw))
    return calls


def _norm_calls(M, D):
    calls = []
    for i in range(STREAMS):
        g = torch.Generator().manual_seed(i)
        x, r = (torch.randn(M, D, generator=g).to("cuda", BF) for _ in range(2))
        calls.append(lambda x=x, r=r: ops.add_rms_norm(x, r, quantize="float8_e4m3fn", blocked=True)[0][0].view(torch.uint8))
    return calls


CASES = {
    "lora split K": lambda: _lora_calls(64, 2048, 4096, [16] * 4),
    "lora mixed adapters": lambda: _lora_calls(1333, 2048, 2048, [8] * 7),
    "lora many passes": lambda: _lora_calls(200, 384, 1280, [128] * 9, act="gelu"),
    "lora few rows": lambda: _lora_calls(7, 1024, 2048, [16, 8, 4]),
    "attention key mask": lambda: _cross_calls(2, 8, 8, 501, 1024, 64, "keys", torch.float16),
    "attention bool mask": lambda: _cross_calls(2, 4, 2, 333, 500, 128, "bool"),
    "attention additive mask": lambda: _cross_calls(2, 4, 4, 333, 500, 128, "bias"),
    "attention f32 mask": lambda: _cross_calls(2, 4, 4, 200, 300, 64, "bias32"),
    "attention lengths": lambda: _cross_calls(3, 6, 6, 700, 600, 128, "lens"),
    "few queries": lambda: _cross_calls(4, 8, 2, 1, 3000, 128, "lens"),
    "few queries, mask": lambda: _cross_calls(2, 8, 4, 2, 2081, 64, "keys"),
    "norm": lambda: _norm_calls(2000, 1024),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(CASES))
def test_calls_in_flight_keep_apart(native, case):
    calls = CASES[case]()
    want = [c() for c in calls]  # one after another
    torch.cuda.synchronize()
    assert not any(torch.equal(want[0], w) for w in want[1:])
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(4):
        got = [[] for _ in calls]
        for _ in range(6):
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
    want = [c() for c in calls]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in calls], []
    for g, call in zip(graphs, calls):
        with torch.cuda.graph(g):
            outs.append([call() for _ in range(3)])
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(4):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for own, w in zip(outs, want):
        assert all(torch.equal(o, w) for o in own)
