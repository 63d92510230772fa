"""Measured cases of the residual RMSNorm, the adapter projection and the cross attention.

``listed()`` / ``draw(rng)`` give the cases, ``prepare(case, seed)`` the tensors of one case,
``run(state)`` one pass (the plain torch form, or the framework's operators when ``own`` is set),
``work(case)`` what a pass has to move and compute, ``exact(case, seed)`` the result in 64 bits.

Operators (``op`` of a case):

* ``norm``  s = x + resid; y = s / sqrt(mean(s^2) + eps) * w * (1 + scale[b]) + shift[b]; s and y are
  returned, y in the input type or through MXFP8 (32 values share a power-of-two scale).
* ``lora``  y = act(x W^T + b + a_i (x A_i^T) B_i^T), i = the adapter of the row's request (-1: none).
* ``cross`` softmax(scale q k^T + mask) v with keys of another length than the queries.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
FP8 = {"e4m3": (8, 448.0, torch.float8_e4m3fn), "e5m2": (15, 57344.0, torch.float8_e5m2)}


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of each of four requests, two streams of width 4096 (refiner / decoder LM step)
        dict(name="norm_tokens", op="norm", batch=4, rows=1, dim=4096, dtype="bf16", mod=False, out="same"),
        # an audio clip's tokens, width 2048, half precision
        dict(name="norm_audio_fp16", op="norm", batch=2, rows=501, dim=2048, dtype="fp16", mod=True, out="same"),
        # an odd width that no vector load divides, single precision
        dict(name="norm_odd_fp32", op="norm", batch=3, rows=777, dim=1023, dtype="fp32", mod=False, out="same"),
        # every token of a 480p, 81-frame clip at width 5120, adaLN-modulated, into the MXFP8 projection
        dict(name="norm_video_mx", op="norm", batch=1, rows=32760, dim=5120, dtype="bf16", mod=True, out="e4m3"),
        # one row of each of four requests, every one with its own adapter (a modulation / time projection)
        dict(name="lora_tokens", op="lora", batch=4, rows=1, k=4096, n=4096, rank=16, adapters=4, mixed=False, act="none"),
        # tokens of many requests packed without order, some without an adapter
        dict(name="lora_mixed", op="lora", batch=1, rows=1333, k=2048, n=2048, rank=8, adapters=7, mixed=True, act="none"),
        # four requests' feed-forward projection at width 4096 with GELU
        dict(name="lora_ffn", op="lora", batch=4, rows=1280, k=4096, n=16384, rank=32, adapters=4, mixed=False, act="gelu"),
        # both guidance branches of a 480p clip, attention output projection at width 5120
        dict(name="lora_video", op="lora", batch=2, rows=16380, k=5120, n=5120, rank=64, adapters=3, mixed=False, act="none"),
        # one query per request (attention pooling) over long encoder states with shared key heads
        dict(name="cross_pool", op="cross", batch=8, heads=32, kv_heads=8, sq=1, sk=4096, dim=128, dtype="bf16", mask="lens", fill=0.8),
        # audio tokens over padded text, head dim 64
        dict(name="cross_audio", op="cross", batch=2, heads=32, kv_heads=32, sq=501, sk=1024, dim=64, dtype="fp16", mask="keys", fill=0.3),
        # regional prompts: every query has keys of its own, additive mask
        dict(name="cross_regions", op="cross", batch=2, heads=16, kv_heads=16, sq=2040, sk=777, dim=128, dtype="bf16", mask="add", fill=0.5),
        # every token of a 480p, 81-frame clip over the text, 40 heads
        dict(name="cross_video", op="cross", batch=1, heads=40, kv_heads=40, sq=32760, sk=512, dim=128, dtype="bf16", mask="lens", fill=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "lora", "cross"])
    if op == "norm":
        out = rng.choice(["same", "same", "e4m3", "e5m2"])
        dim = _log(rng, 64, 8192)
        dim = max(64, dim // 128 * 128) if out != "same" or rng.random() < 0.5 else dim
        batch = rng.choice([1, 2, 3, 4])
        rows = _log(rng, 1, max(2, min(32760, 150_000_000 // dim) // batch))
        return dict(op=op, batch=batch, rows=rows, dim=dim, dtype=rng.choice(["bf16", "fp16", "fp32"] if out == "same" else ["bf16", "bf16", "fp16"]),
                    mod=rng.random() < 0.5, out=out)
    if op == "lora":
        k, n = 64 * _log(rng, 8, 96), 64 * _log(rng, 8, 128)
        batch = rng.choice([1, 2, 3, 4, 8])
        rows = _log(rng, 1, max(2, int(min(32760, 5e11 / (k * n))) // batch))
        return dict(op=op, batch=batch, rows=rows, k=k, n=n, rank=rng.choice([4, 8, 13, 16, 32, 64, 128]), adapters=rng.randint(1, 12),
                    mixed=rng.random() < 0.3, act=rng.choice(["none", "none", "gelu", "silu"]))
    dim, kv_heads = rng.choice([64, 128]), rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    batch, sk = rng.choice([1, 2, 3, 5]), _log(rng, 1, 4096)
    mask = rng.choice(["none", "lens", "keys", "bool", "add"])
    sq = _log(rng, 1, max(2, min(32760, int(6e8 / (batch * heads * sk)))))
    return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, sq=sq, sk=sk, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]), mask=mask,
                fill=round(rng.uniform(0.1, 1.0), 2))


def _lens(c):
    """Valid keys of each batch row: ``fill`` of the keys in the first, fewer in the later ones."""
    return [max(1, int(c["sk"] * c["fill"] * (1 - 0.5 * b / c["batch"]))) for b in range(c["batch"])]


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    c = case
    s = {"case": dict(case)}
    if c["op"] == "norm":
        M, D, dt = c["batch"] * c["rows"], c["dim"], DTYPES[c["dtype"]]
        s.update(x=rnd(M, D, dtype=dt), resid=rnd(M, D, dtype=dt, std=3.0), w=1 + rnd(D, dtype=dt, std=0.1))
        s["scale"] = rnd(c["batch"], D, std=0.2) if c["mod"] else None
        s["shift"] = rnd(c["batch"], D, std=0.2) if c["mod"] else None
    elif c["op"] == "lora":
        M, K, N, R, n = c["batch"] * c["rows"], c["k"], c["n"], c["rank"], c["adapters"]
        dt = torch.bfloat16
        s.update(x=rnd(M, K, dtype=dt), w=rnd(N, K, dtype=dt, std=K ** -0.5), b=rnd(N, dtype=dt, std=0.1),
                 A=rnd(n, R, K, dtype=dt, std=K ** -0.5), B=rnd(n, N, R, dtype=dt, std=0.5 * R ** -0.5),
                 alpha=torch.linspace(0.5, 1.5, n, device="cuda"))
        if c["mixed"]:  # one adapter per row, -1 (none) among them
            s["ids"] = torch.randint(-1, n, (M,), generator=g, device="cuda", dtype=torch.int32)
        else:  # one adapter per request
            s["ids"] = torch.randint(0, n, (c["batch"],), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from difflet_b200 import ops

            s["bank"] = ops.LoraBank(s["A"], s["B"], s["alpha"])
    else:
        B, H, Hk, Sq, Sk, D, dt = c["batch"], c["heads"], c["kv_heads"], c["sq"], c["sk"], c["dim"], DTYPES[c["dtype"]]
        # token-major projections viewed by head, as the q and k / v projections leave them
        s["q"] = rnd(B, Sq, H, D, dtype=dt).permute(0, 2, 1, 3)
        kv = rnd(B, Sk, 2, Hk, D, dtype=dt)
        s["k"], s["v"] = kv[:, :, 0].permute(0, 2, 1, 3), kv[:, :, 1].permute(0, 2, 1, 3)
        s["mask"] = s["lens"] = None
        lens = torch.tensor(_lens(c), device="cuda", dtype=torch.int32)
        if c["mask"] == "lens":
            s["lens"] = lens
        elif c["mask"] == "keys":
            s["mask"] = (torch.arange(Sk, device="cuda")[None] < lens[:, None])[:, None, None, :]
        elif c["mask"] in ("bool", "add"):
            keep = torch.rand(B, 1, Sq, Sk, generator=g, device="cuda") < c["fill"]
            keep[:, :, ::7] = False  # some queries have no key at all
            keep[:, :, ::7, :1] = c["mask"] == "add"
            if c["mask"] == "bool":
                s["mask"] = keep
            else:
                bias = rnd(B, 1, Sq, Sk)
                s["mask"] = torch.where(keep, bias, torch.full_like(bias, float("-inf"))).to(dt)
    return s


# ----------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "lora": _plain_lora, "cross": _plain_cross}[state["case"]["op"]](state)


def _run_own(s):
    from difflet_b200 import ops

    c = s["case"]
    if c["op"] == "norm":
        quant = None if c["out"] == "same" else {"e4m3": "float8_e4m3fn", "e5m2": "float8_e5m2"}[c["out"]]
        y, r = ops.add_rms_norm(s["x"], s["resid"], s["w"], eps=1e-6, scale=s["scale"], shift=s["shift"], rows_per_batch=c["rows"], quantize=quant)
        if quant is not None:
            y = ops.dequantize_mx(y[0], y[1], dtype=quant, output_dtype=s["x"].dtype)
        return {"y": y, "resid": r}
    if c["op"] == "lora":
        return ops.linear_lora(s["x"], s["w"], s["b"], bank=s["bank"], ids=s["ids"], rows_per_batch=0 if c["mixed"] else c["rows"],
                               act=None if c["act"] == "none" else c["act"])
    return ops.cross_attention(s["q"], s["k"], s["v"], scale=c["dim"] ** -0.5, attention_mask=s["mask"], kv_lens=s["lens"])


def _plain_norm(s):
    c = s["case"]
    t = s["x"].float() + s["resid"].float()
    y = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * s["w"].float()
    if c["mod"]:
        y = y.view(c["batch"], c["rows"], c["dim"])
        y = (y * (1 + s["scale"][:, None]) + s["shift"][:, None]).view(t.shape)
    if c["out"] != "same":
        emax, top, fp8 = FP8[c["out"]]
        blocks = y.view(y.shape[0], -1, 32)
        e = (torch.frexp(blocks.abs().amax(-1, keepdim=True)).exponent - 1 - emax).clamp(-127, 127)
        q = torch.ldexp(blocks, -e).clamp(-top, top).to(fp8)
        y = torch.ldexp(q.float(), e).view(t.shape)
    return {"y": y.to(s["x"].dtype), "resid": t.to(s["x"].dtype)}


def _plain_lora(s):
    c = s["case"]
    n, R, K = s["A"].shape
    x = s["x"].float()
    ids = s["ids"].long() if c["mixed"] else s["ids"].long().repeat_interleave(c["rows"])
    pick = (ids[:, None] == torch.arange(n, device=ids.device)[None]).float() * s["alpha"][None]
    t = (x @ s["A"].float().view(n * R, K).t()).view(-1, n, R) * pick[..., None]
    y = x @ s["w"].float().t() + s["b"].float() + t.view(-1, n * R) @ s["B"].float().permute(0, 2, 1).reshape(n * R, -1)
    if c["act"] == "gelu":  # tanh form
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif c["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(s["x"].dtype)


def _plain_cross(s):
    c = s["case"]
    rep = c["heads"] // c["kv_heads"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if rep > 1:
        k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    z = (q * c["dim"] ** -0.5) @ k.transpose(-1, -2)
    if s["lens"] is not None:
        z.masked_fill_((torch.arange(c["sk"], device=z.device)[None] >= s["lens"][:, None])[:, None, None], float("-inf"))
    elif s["mask"] is not None and s["mask"].dtype == torch.bool:
        z.masked_fill_(~s["mask"], float("-inf"))
    elif s["mask"] is not None:
        z += s["mask"].float()
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)  # 0 where the mask leaves nothing: such a row is 0
    return ((p @ v) / torch.where(total > 0, total, torch.ones_like(total))).to(s["q"].dtype)


# ----------------------------------------------------------------------------- floors
def work(case):
    c = case
    if c["op"] == "norm":
        M, D, e = c["batch"] * c["rows"], c["dim"], SIZE[c["dtype"]]
        return {"bytes": 4 * M * D * e + D * e + (2 * c["batch"] * D * 4 if c["mod"] else 0), "flops": 8 * M * D}
    if c["op"] == "lora":
        M, K, N, R = c["batch"] * c["rows"], c["k"], c["n"], c["rank"]
        used = min(c["adapters"], M if c["mixed"] else c["batch"])
        return {"bytes": 2 * (M * K + N * K + M * N + N) + 2 * used * R * (K + N), "flops": 2 * M * N * K + 2 * M * R * (K + N)}
    B, H, Hk, Sq, Sk, D = c["batch"], c["heads"], c["kv_heads"], c["sq"], c["sk"], c["dim"]
    keys = sum(_lens(c)) if c["mask"] in ("lens", "keys") else B * Sk
    mask = {"bool": 1, "add": 2}.get(c["mask"], 0) * B * Sq * Sk
    return {"bytes": 2 * (2 * B * H * Sq * D + 2 * Hk * keys * D) + mask, "flops": 4 * H * Sq * keys * D}


# ----------------------------------------------------------------------------- 64 bits
def _exact_norm(s):
    c = s["case"]
    D = c["dim"]
    a = s["x"].double() + s["resid"].double()
    norm = torch.sqrt((a * a).sum(1) / D + 1e-6)
    y = a / norm[:, None] * s["w"].double()[None]
    if c["mod"]:
        batch_of = torch.arange(y.shape[0], device=y.device) // c["rows"]
        y = y + y * s["scale"].double()[batch_of] + s["shift"].double()[batch_of]
    if c["out"] != "same":  # the value of the nearest 8-bit element times the block's power of two
        emax, top, fp8 = FP8[c["out"]]
        bits, low = (3, -6) if c["out"] == "e4m3" else (2, -14)
        b = y.unflatten(1, (D // 32, 32))
        unit = torch.exp2(torch.frexp(b.abs().max(-1, keepdim=True).values).exponent.double() - 1 - emax)
        v = (b / unit).clamp(-top, top)
        step = torch.exp2((torch.frexp(v.abs()).exponent.double() - 1).clamp(min=low) - bits)
        y = (torch.round(v / step) * step * unit).flatten(1)
    return {"y": y, "resid": a}


def _exact_lora(s):
    c = s["case"]
    ids = s["ids"].long() if c["mixed"] else s["ids"].long().repeat_interleave(c["rows"])
    x = s["x"].double()
    y = torch.addmm(s["b"].double()[None], x, s["w"].double().t())
    for i in range(c["adapters"]):
        at = (ids == i).nonzero()[:, 0]
        y[at] += float(s["alpha"][i]) * (x[at] @ s["A"][i].double().t() @ s["B"][i].double().t())
    if c["act"] == "gelu":
        return 0.5 * y * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    return y * torch.sigmoid(y) if c["act"] == "silu" else y


def _exact_cross(s):
    c = s["case"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    rep = c["heads"] // c["kv_heads"]
    for b in range(c["batch"]):
        n = int(s["lens"][b]) if s["lens"] is not None else c["sk"]
        m = None if s["mask"] is None else s["mask"][b, 0]
        for h in range(c["heads"]):
            k, v = s["k"][b, h // rep, :n].double(), s["v"][b, h // rep, :n].double()
            z = s["q"][b, h].double() @ k.t() / math.sqrt(c["dim"])
            if m is not None:
                z = torch.where(m, z, -math.inf) if m.dtype == torch.bool else z + m.double()
            out[b, h] = torch.nan_to_num(torch.softmax(z, -1), nan=0.0) @ v
    return out


def exact(case, seed):
    return {"norm": _exact_norm, "lora": _exact_lora, "cross": _exact_cross}[case["op"]](prepare(case, seed))
