"""Public attention ops for model code (the reference's ``difflet.ops`` attention surface).

Contract (difflet/ops/attention.py:4-128, difflet/backends/cuda/ops_impl/attention.py:1-17):

* ``q, k, v``: ``[B, H, S, D]`` or ``[B*H, S, D]``; the result has ``q``'s shape.
* ``scale=None`` means 1.0 (not ``1/sqrt(D)``).
* ``attention_mask``: bool (True = attend) or additive (integers too); ``bound_min`` / ``bound_max``
  (both or neither, exclusive with a mask) select the keys ``[bound_min, bound_max)``.
* ``tp_q`` / ``tp_k`` / ``tp_out`` are layout hints of other hardware: accepted, ignored.

Dispatch (the kernels record no backward pass: inputs that ask for gradients take the library
path on CUDA): CUDA tensors with head dim 128, bf16, no mask, non-causal and bounds that are
per batch row (shape ``[B]`` or ``[B, 1, ...]``, the padded-text key windows every
model here uses) run the tcgen05 kernel of ``csrc/attention.cu``.  Masks (boolean or
additive), per-query windows, head dim 64 and fp16 run the tcgen05 kernel of
``csrc/cross_attn.cuh``, which ``cross_attention`` always takes.  Anything else on CUDA
(causal, other head dims, values of another width, fp32, tracing and function transforms) is the library path:
``torch.nn.functional.scaled_dot_product_attention``.  CPU tensors run the fp32 / fp64
oracle of ``ops.fused``.

Context-parallel ops (``ring_attention``, ``joint_ring_attention``,
``ulysses_attention``, ``joint_ulysses_attention``) run over the cp group of the
mesh (``parallel.groups``) with ``torch.distributed`` transfers; the built-in models
use the fused peer-memory transports of ``parallel.ulysses`` / ``parallel.ring``
instead.  Semantics: difflet/backends/neuron/ops_impl/attention.py:435-713.
"""

from __future__ import annotations

import operator

import torch
import torch.nn.functional as TF

from difflet_b200.ops import fused as F


def _bounds_to_mask(k, bound_min, bound_max, attention_mask):
    if bound_min is None and bound_max is None:
        return attention_mask
    if bound_min is None or bound_max is None:
        raise ValueError("bound_min and bound_max must both be provided")
    if attention_mask is not None:
        raise ValueError("attention_mask and bounds are mutually exclusive")
    idx = torch.arange(k.shape[-2], device=k.device)
    return (idx >= bound_min.to(k.device)) & (idx < bound_max.to(k.device))


def _per_batch(bound, B):
    """A [B] int32 window edge when ``bound`` does not vary over queries, else None."""
    if bound is None:
        return None
    b = torch.as_tensor(bound)
    if b.dim() == 0:
        b = b.expand(B)
    elif b.shape[0] == B and all(s == 1 for s in b.shape[1:]):
        b = b.reshape(B)
    else:
        return None
    return b


def _edge(t, n, device):
    """A window edge as int32 for keys [0, n): what lies past either end is that end, fractions count as in ``key < edge``."""
    if t.is_floating_point():
        t = t.ceil().clamp(0, n)
    elif t.dtype == torch.int64:  # (the kernels clamp what fits 32 bits)
        t = t.clamp(0, n)
    return t.to(device, torch.int32).contiguous()


def attention(q, k, v, *, scale=None, causal=False, attention_mask=None, bound_min=None, bound_max=None,
              tp_q=False, tp_k=False, tp_out=False, lse=None, **kwargs):
    del tp_q, tp_k, tp_out, kwargs
    scale = 1.0 if scale is None else float(scale)
    folded = q.dim() == 3
    q4, k4, v4 = (t.unsqueeze(0) for t in (q, k, v)) if folded else (q, k, v)
    B = q4.shape[0]
    if (bound_min is None) != (bound_max is None):
        raise ValueError("bound_min and bound_max must both be provided")
    if attention_mask is not None and bound_min is not None:
        raise ValueError("attention_mask and bounds are mutually exclusive")
    lo, hi = _per_batch(bound_min, B), _per_batch(bound_max, B)
    simple = attention_mask is None and not causal and (bound_min is None or (lo is not None and hi is not None))
    kernel = (q.is_cuda and simple and q.shape[-1] == v.shape[-1] == 128 and q.dtype == torch.bfloat16
              and not F.wants_grad(q, k, v))
    if kernel or (simple and not q.is_cuda):
        if lo is not None:
            lo = lo.to(q.device, torch.int32 if q.is_cuda else torch.int64).contiguous()
            hi = hi.to(q.device, torch.int32 if q.is_cuda else torch.int64).contiguous()
        out = F.attention(q4, k4, v4, scale, lse=lse, kv_lo=lo, kv_hi=hi)
    elif (F.cross_kernel_ok(q, k, v, attention_mask) and not causal and k4.dtype == v4.dtype == q4.dtype
          and k4.shape == v4.shape and k4.shape[:2] == q4.shape[:2] and (lse is None or simple)):
        mask = attention_mask if simple or bound_min is None else _bounds_to_mask(k4, bound_min, bound_max, None)
        if lo is not None and simple:
            lo, hi = (_edge(t, k4.shape[2], q.device) for t in (lo, hi))
        else:
            lo = hi = None
        out = F.cross_attention(q4, k4, v4, scale, mask=_mask_on(mask, q), kv_lo=lo, kv_hi=hi, lse=lse,
                                precise_p=lse is not None)  # (partials that are merged by their LSE: f32 up to the result)
    else:
        if simple and lo is not None:  # (one edge per batch row, whatever shape it came in)
            bound_min, bound_max = (t.view(B, 1, 1, 1) for t in (lo, hi))
        mask = _bounds_to_mask(k4, bound_min, bound_max, attention_mask)
        if lse is not None or not q.is_cuda:  # math path (oracle, or LSE requested off the kernel)
            out = _oracle_masked(q4, k4, v4, scale, causal, mask, lse)
        else:
            out = _sdpa(q4, k4, v4, scale, causal, mask)
    return out.squeeze(0) if folded else out


def _sdpa(q, k, v, scale, causal, mask):
    if mask is None:
        return TF.scaled_dot_product_attention(q, k, v, is_causal=causal, scale=scale)
    Lq, Lk = q.shape[-2], k.shape[-2]
    if mask.dtype == torch.bool:
        m = mask.to(q.device)
        if causal:
            m = m & torch.ones(Lq, Lk, dtype=torch.bool, device=q.device).tril()
        return TF.scaled_dot_product_attention(q, k, v, attn_mask=m, scale=scale)
    add = mask.to(device=q.device, dtype=q.dtype)
    if causal:
        tri = torch.ones(Lq, Lk, dtype=torch.bool, device=q.device).tril()
        add = add.masked_fill(~tri, torch.finfo(q.dtype).min)
    return TF.scaled_dot_product_attention(q, k, v, attn_mask=add, scale=scale)


def _oracle_masked(q, k, v, scale, causal, mask, lse=None):
    ct = torch.float64 if q.dtype == torch.float64 else torch.float32
    s = torch.einsum("bhqd,bhkd->bhqk", q.to(ct), k.to(ct)) * scale
    if mask is not None:
        if mask.dtype == torch.bool:
            s = s.masked_fill(~mask.to(s.device), float("-inf"))
        else:
            s = s + mask.to(device=s.device, dtype=ct)
    if causal:
        tri = torch.ones(s.shape[-2], s.shape[-1], dtype=torch.bool, device=s.device).tril()
        s = s.masked_fill(~tri, float("-inf"))
    if lse is not None:
        lse.copy_(torch.logsumexp(s, -1).to(lse.dtype).reshape(lse.shape))
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
    return torch.einsum("bhqk,bhkd->bhqd", p, v.to(ct)).to(q.dtype)


_MASK_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _mask_on(mask, q):
    """A mask on q's device whose type the kernel reads; what is not boolean is added to the scores, integers too."""
    if mask is None or mask.dtype == torch.bool:
        return mask if mask is None else mask.to(q.device)
    if not mask.is_floating_point():
        mask = mask.float()
    elif mask.dtype not in _MASK_DTYPES and q.is_cuda:  # finite values stay finite (the type's lowest masks softly)
        low = torch.finfo(torch.float32)
        mask = torch.where(mask.isfinite(), mask.clamp(low.min, low.max), mask).float()
    return mask.to(q.device)


def _is_key_mask(mask) -> bool:
    """Whether a mask broadcastable to [B, H, Sq, Sk] is the same for every head and query."""
    return all(n == 1 for n in mask.shape[-3:-1])


def cross_attention(q, k, v, *, scale=None, attention_mask=None, kv_lens=None, lse=None, out=None, bound_min=None,
                    bound_max=None, **kwargs):
    """Attention of ``q [B, H, Sq, D]`` to encoder states ``k [B, Hk, Sk, D]``, ``v [B, Hk, Sk, Dv]`` of another length.

    ``Hk`` divides ``H`` (query head h reads key head ``h // (H // Hk)``); where the heads are equal, or one, so may be the batch
    rows: one of q, or of k and v, then serves all of the other side.  ``attention_mask``: bool (True =
    attend) or additive (integers too), broadcastable to ``[B, H, Sq, Sk]``; moved to q's device as in ``attention``
    (refused there with shared key heads on CUDA).  ``kv_lens`` (integers ``[B]``): the valid keys of
    each batch row; what k and v hold behind them is not used.  ``bound_min`` / ``bound_max`` as in
    ``attention``.  A query that no key is left for gives 0.  ``out`` (``[B, H, Sq, Dv]``) and ``lse`` (``[B, H, Sq]``,
    natural log) are filled when given (an LSE that is not contiguous f32 on q's device by a copy).  CUDA: bf16 and fp16
    with D = Dv = 64 or 128; anything else, and what asks for gradients, runs as ``attention``."""
    if (q.is_cuda and type(q) is torch.Tensor and q.dtype in F.CROSS_DTYPES and q.shape[-1] in (64, 128)
            and bound_min is None and bound_max is None and not torch.compiler.is_compiling()):
        try:  # the binding checks everything; what it refuses is looked at again below
            return F.cross_attention(q, k, v, 1.0 if scale is None else float(scale), mask=attention_mask, kv_hi=kv_lens,
                                     out=out, lse=lse)
        except ValueError:
            pass
    for key in ("tp_q", "tp_k", "tp_out", "causal"):
        kwargs.pop(key, None)
    if q.dim() == 3:
        if kv_lens is not None or out is not None:
            raise ValueError("kv_lens and out need q [B, H, S, D]")
        o = cross_attention(q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0), scale=scale, attention_mask=attention_mask,
                            lse=lse, bound_min=bound_min, bound_max=bound_max)
        return o.squeeze(0)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3]:
        raise ValueError(f"q [B, H, Sq, D], k [B, Hk, Sk, D], v [B, Hk, Sk, Dv]; got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    B, H, Sq, D = q.shape
    Bk, Hk = k.shape[:2]
    if (k.shape[3] != D or Hk < 1 or (H != 1 and H % Hk)
            or (Bk != B and (1 not in (B, Bk) or (H != 1 and Hk not in (1, H))))):
        raise ValueError(f"k / v {tuple(k.shape)} do not match q {tuple(q.shape)} (H must be a multiple of Hk)")
    if Bk != B or Hk > H:  # one batch row (one query head) for all
        B, H = Bk if B == 1 else B, max(H, Hk)
        q, k, v = q.expand(B, H, Sq, D), *(t.expand(B, *t.shape[1:]) for t in (k, v))
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must share type and device")
    if out is not None and (out.shape != (B, H, Sq, v.shape[3]) or out.dtype != q.dtype or out.device != q.device):
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} is not {(B, H, Sq, v.shape[3])} {q.dtype}")
    if lse is not None and lse.numel() != B * H * Sq:
        raise ValueError(f"lse must hold [{B}, {H}, {Sq}]")
    lo = hi = None
    if kv_lens is not None:
        if bound_min is not None or bound_max is not None:
            raise ValueError("kv_lens and bounds are mutually exclusive")
        if kv_lens.shape != (B,) or kv_lens.is_floating_point() or kv_lens.dtype == torch.bool:
            raise ValueError(f"kv_lens must be integers [{B}]")
        hi = _edge(kv_lens, k.shape[2], q.device)
    elif bound_min is not None or bound_max is not None:
        if bound_min is None or bound_max is None:
            raise ValueError("bound_min and bound_max must both be provided")
        if attention_mask is not None:
            raise ValueError("attention_mask and bounds are mutually exclusive")
        lo, hi = _per_batch(bound_min, B), _per_batch(bound_max, B)
        if lo is None or hi is None:
            attention_mask, lo, hi = _bounds_to_mask(k, bound_min, bound_max, None), None, None
        else:
            lo, hi = (_edge(t, k.shape[2], q.device) for t in (lo, hi))
    mask = attention_mask
    kernel = k.shape == v.shape and F.cross_kernel_ok(q, k, v, mask)
    if mask is not None:
        if kernel and mask.device != q.device and k.shape[1] != q.shape[1]:
            raise ValueError("the mask must be on q's device where heads share keys")
        mask = _mask_on(mask, q)
        want = (B, H, Sq, k.shape[2])
        if mask.dim() > 4 or any(m not in (1, w) for m, w in zip(mask.shape[::-1], want[::-1])):
            raise ValueError(f"attention_mask {tuple(mask.shape)} does not broadcast to {want}")
        mask = mask.reshape((1,) * (4 - mask.dim()) + mask.shape)
    scale = 1.0 if scale is None else float(scale)
    if not q.is_cuda or kernel:
        return F.cross_attention(q, k, v, scale, mask=mask, kv_lo=lo, kv_hi=hi, out=out, lse=lse)
    # off the kernel: the window and a key mask as one mask; what lies at their excluded keys may be anything, and 0 * NaN
    # would reach the sums
    keys = None
    if hi is not None:
        idx = torch.arange(k.shape[2], device=q.device)
        keys = ((idx < hi[:, None]) if lo is None else (idx < hi[:, None]) & (idx >= lo[:, None]))[:, None, None]
    if mask is not None and mask.dtype == torch.bool:
        if _is_key_mask(mask):
            keys, mask = mask if keys is None else keys & mask, None
        elif keys is not None:
            mask = mask & keys
    elif mask is not None and keys is not None:
        mask = mask.masked_fill(~keys, float("-inf"))
    if keys is not None:
        keys = keys.expand(*keys.shape[:-1], k.shape[2])
        k, v = (t.masked_fill(~keys.transpose(2, 3), 0.0) for t in (k, v))
        mask = keys if mask is None else mask
    rep = H // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    if mask is None:
        o = attention(q, k, v, scale=scale, lse=lse)
        return o if out is None else out.copy_(o)
    # a row without a key attends to all of them and is cleared afterwards (softmax of nothing has no value and no gradient)
    if mask.dtype == torch.bool:
        empty = ~mask.any(-1, keepdim=True)
        mask = mask | empty
    else:
        empty = (mask == float("-inf")).all(-1, keepdim=True)
        mask = mask.masked_fill(empty, 0.0)
    o = attention(q, k, v, scale=scale, attention_mask=mask, lse=lse).masked_fill(empty, 0.0)
    if lse is not None:
        lse.masked_fill_(empty.expand(B, H, Sq, 1).reshape(lse.shape), float("-inf"))
    return o if out is None else out.copy_(o)


def _positions(q, k, kv_lens, q_start):
    """Valid keys and the first query's position of each batch row, int64 [B]."""
    B, Sk = q.shape[0], k.shape[2]
    lens = torch.full((B,), Sk, device=q.device) if kv_lens is None else kv_lens.to(q.device, torch.int64).clamp(0, Sk)
    return lens, lens - q.shape[2] if q_start is None else q_start.to(q.device, torch.int64)


def window_attention(q, k, v, *, window, sinks=0, scale=None, kv_lens=None, q_start=None, lse=None, out=None):
    """Causal attention to the last ``window`` keys and to the first ``sinks`` ones, which stay visible.

    q [B, H, Sq, D]; k, v [B, Hk, Sk, D] (the cache), ``Hk`` divides ``H`` (query head h reads key head ``h // (H // Hk)``); any
    strides.  Query i of batch row b stands at position ``p = q_start[b] + i`` and sees the keys ``j <= p`` with ``j > p - window``
    or ``j < sinks``, among the row's ``kv_lens[b]`` valid ones (integers ``[B]``; None: all).  ``q_start`` (an integer or integers
    ``[B]``; None: ``kv_lens - Sq``, the queries are the newest keys' own): 0 for prompts that are padded behind their ends.  A
    window of ``Sk`` or more is plain causal attention.  ``scale=None`` means 1.0 as in ``attention``.

    A query without a visible key gives 0 (LSE -inf).  What k and v hold at keys that no query of the call sees is not used; a
    value that only some queries see must be finite (it meets the others with weight 0).  ``out`` (``[B, H, Sq, D]``) and ``lse``
    (``[B, H, Sq]``, natural log) are filled when given.  CUDA: bf16 and fp16 with D 64 or 128, whose P is rounded to
    the type for its product with v; only the tiles that some query sees are read, and few queries share the keys among many
    CTAs.  Anything else, and what asks for gradients, runs as ``cross_attention`` under the same mask."""
    if (q.is_cuda and type(q) is torch.Tensor and q.dtype in F.CROSS_DTYPES and (q_start is None or type(q_start) is torch.Tensor)
            and not torch.compiler.is_compiling()):
        try:  # the binding checks everything; what it refuses is looked at again below
            return F.window_attention(q, k, v, 1.0 if scale is None else float(scale), window, sinks, kv_lens=kv_lens,
                                      q_start=q_start, out=out, lse=lse)
        except (ValueError, TypeError):
            pass
    window, sinks = (min(operator.index(n), 2 ** 62) for n in (window, sinks))
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0, got {window} and {sinks}")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q [B, H, Sq, D], k and v [B, Hk, Sk, D]; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, H, Sq, _ = q.shape
    if k.shape[1] < 1 or H % k.shape[1]:
        raise ValueError(f"the query heads ({H}) must be a multiple of the key heads ({k.shape[1]})")
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must share type and device")
    if q_start is not None and not torch.is_tensor(q_start):
        q_start = torch.full((B,), int(q_start), device=q.device)
    for name, t in (("kv_lens", kv_lens), ("q_start", q_start)):
        if t is not None and (t.shape != (B,) or t.is_floating_point() or t.is_complex() or t.dtype == torch.bool):
            raise ValueError(f"{name} must be integers [{B}]")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device):
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} does not match q {tuple(q.shape)} {q.dtype}")
    if lse is not None and lse.numel() != B * H * Sq:
        raise ValueError(f"lse must hold [{B}, {H}, {Sq}]")
    scale = 1.0 if scale is None else float(scale)
    if F.cross_kernel_ok(q, k, v) and F.kernel_tensors(kv_lens, q_start):
        own = lse
        if lse is not None and (lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != q.device):
            own = torch.empty(B, H, Sq, device=q.device, dtype=torch.float32)
        o = F.window_attention(q, k, v, scale, window, sinks, kv_lens=kv_lens, q_start=q_start, out=out, lse=own)
        if own is not lse:
            lse.copy_(own.reshape(lse.shape))
        return o
    lens, first = _positions(q, k, kv_lens, q_start)
    j = torch.arange(k.shape[2], device=q.device)
    p = (first[:, None] + torch.arange(Sq, device=q.device))[:, :, None]
    seen = (j <= p) & ((j > p - window) | (j < sinks)) & (j < lens[:, None, None])
    keys = seen.any(1)[:, None, :, None]  # (what no query sees may be anything, and 0 * NaN would reach the sums)
    k, v = (t.masked_fill(~keys, 0.0) for t in (k, v))
    return cross_attention(q, k, v, scale=scale, attention_mask=seen[:, None], lse=lse, out=out)


def attention_with_lse(q, k, v, *, scale, bound_min=None, bound_max=None):
    """(out, lse) of one key block: lse fp32 [B, H, Sq] (natural log)."""
    lse = torch.empty(q.shape[:-1], device=q.device, dtype=torch.float64 if q.dtype == torch.float64
                      else torch.float32)
    out = attention(q, k, v, scale=scale, bound_min=bound_min, bound_max=bound_max, lse=lse)
    return out, lse


def merge_partials(out, lse, o_r, l_r):
    """Log-sum-exp merge of two partial attentions (max-subtracted; empty partials weigh 0)."""
    m = torch.maximum(lse, l_r)
    safe = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    w, w_r = torch.exp(lse - safe), torch.exp(l_r - safe)
    tot = w + w_r
    den = torch.where(tot > 0, tot, torch.ones_like(tot))
    merged = (out * w.unsqueeze(-1) + o_r * w_r.unsqueeze(-1)) / den.unsqueeze(-1)
    return merged, torch.where(tot > 0, safe + torch.log(den), torch.full_like(tot, float("-inf")))


# ----------------------------------------------------------------------------- context parallel
def _cp():
    import torch.distributed as dist

    from difflet_b200.parallel import groups

    ranks = groups.get_group_ranks("cp")
    if not dist.is_initialized() or len(ranks) == 1:
        return None, 1, 0
    return groups.get_group("cp"), len(ranks), ranks.index(dist.get_rank())


def _ring_partials(q, k, v, scale, group, cp, rank, out=None, lse=None):
    import torch.distributed as dist

    from difflet_b200.parallel import groups

    ranks = groups.get_group_ranks("cp")
    kv = torch.stack([k, v]).contiguous()
    nxt = torch.empty_like(kv)
    for step in range(cp):
        reqs = []
        if step < cp - 1:
            ops = [dist.P2POp(dist.isend, kv, ranks[(rank + 1) % cp], group=group),
                   dist.P2POp(dist.irecv, nxt, ranks[(rank - 1) % cp], group=group)]
            reqs = dist.batch_isend_irecv(ops)
        o_r, l_r = attention_with_lse(q, kv[0], kv[1], scale=scale)
        o_r = o_r.to(l_r.dtype)
        out, lse = (o_r, l_r) if out is None else merge_partials(out, lse, o_r, l_r)
        for r in reqs:
            r.wait()
        kv, nxt = nxt, kv
    return out, lse


def ring_attention(q, k, v, *, scale, causal=False):
    """q, k, v ``[B, H, S/cp, D]`` sequence-sharded over cp -> ``[B, H, S/cp, D]``."""
    if causal:
        raise NotImplementedError("ring_attention supports non-causal attention only")
    group, cp, rank = _cp()
    if cp == 1:
        return attention(q, k, v, scale=scale)
    out, _ = _ring_partials(q, k, v, scale, group, cp, rank)
    return out.to(q.dtype)


def joint_ring_attention(q, image_k, image_v, text_k, text_v, *, scale, causal=False, text_valid_len=None):
    """Image K/V sharded over cp, text K/V replicated: the text partial (masked past
    ``text_valid_len``) seeds the ring over the image blocks."""
    if causal:
        raise NotImplementedError("joint_ring_attention supports non-causal attention only")
    B = q.shape[0]
    lo = hi = None
    if text_valid_len is not None:
        lo = torch.zeros(B, dtype=torch.int32, device=q.device)
        hi = torch.as_tensor(text_valid_len).to(device=q.device, dtype=torch.int32)
    o_t, l_t = attention_with_lse(q, text_k, text_v, scale=scale, bound_min=lo, bound_max=hi)
    o_t = o_t.to(l_t.dtype)
    group, cp, rank = _cp()
    if cp == 1:
        o_i, l_i = attention_with_lse(q, image_k, image_v, scale=scale)
        out, _ = merge_partials(o_t, l_t, o_i.to(l_i.dtype), l_i)
        return out.to(q.dtype)
    out, _ = _ring_partials(q, image_k, image_v, scale, group, cp, rank, out=o_t, lse=l_t)
    return out.to(q.dtype)


def _a2a_heads_to_seq(x, group, cp):
    """[B, H, S/cp, D] sharded by sequence -> [B, H/cp, S, D] (full sequence, fewer heads)."""
    from difflet_b200.parallel.ulysses import all_to_all

    B, H, s, D = x.shape
    send = x.reshape(B, cp, H // cp, s, D).transpose(0, 1).contiguous()  # [cp, B, H/cp, s, D]
    recv = torch.empty_like(send)
    all_to_all(list(recv.unbind(0)), list(send.unbind(0)), group)
    return recv.permute(1, 2, 0, 3, 4).reshape(B, H // cp, cp * s, D)


def _a2a_seq_to_heads(x, group, cp):
    """[B, H/cp, S, D] -> [B, H, S/cp, D]."""
    from difflet_b200.parallel.ulysses import all_to_all

    B, h, S, D = x.shape
    s = S // cp
    send = x.reshape(B, h, cp, s, D).permute(2, 0, 1, 3, 4).contiguous()  # [cp, B, h, s, D]
    recv = torch.empty_like(send)
    all_to_all(list(recv.unbind(0)), list(send.unbind(0)), group)
    return recv.transpose(0, 1).reshape(B, cp * h, s, D)


def ulysses_attention(q, k, v, *, scale, causal=False):
    """q, k, v ``[B, H_local, S/cp, D]``; needs ``H_local % cp == 0``."""
    group, cp, _ = _cp()
    if cp == 1:
        return attention(q, k, v, scale=scale, causal=causal)
    if q.shape[1] % cp:
        raise ValueError(f"ulysses_attention needs heads % cp == 0, got {q.shape[1]} heads, cp={cp}")
    qf, kf, vf = (_a2a_heads_to_seq(t, group, cp) for t in (q, k, v))
    return _a2a_seq_to_heads(attention(qf, kf, vf, scale=scale, causal=causal), group, cp)


def joint_ulysses_attention(q_img, q_txt, image_k, image_v, text_k, text_v, *, scale, causal=False,
                            key_valid_len=None):
    """Image sharded over cp, text replicated; keys in ``[image_full ; text]`` order with an
    optional per-batch valid count.  Returns ``(img_out [B, H, S_img/cp, D], txt_out [B, H, S_txt, D])``."""
    import torch.distributed as dist

    if causal:
        raise NotImplementedError("joint_ulysses_attention supports non-causal attention only")
    group, cp, rank = _cp()
    B, H = q_img.shape[:2]
    if cp > 1 and H % cp:
        raise ValueError(f"joint_ulysses_attention needs heads % cp == 0, got {H} heads, cp={cp}")
    h = H // cp
    hs = slice(rank * h, (rank + 1) * h)
    if cp > 1:
        qi, ki, vi = (_a2a_heads_to_seq(t, group, cp) for t in (q_img, image_k, image_v))
    else:
        qi, ki, vi = q_img, image_k, image_v
    S_img = qi.shape[2]
    qj = torch.cat([qi, q_txt[:, hs]], 2)
    kj = torch.cat([ki, text_k[:, hs]], 2)
    vj = torch.cat([vi, text_v[:, hs]], 2)
    lo = hi = None
    if key_valid_len is not None:
        hi = torch.as_tensor(key_valid_len).to(device=q_img.device, dtype=torch.int32)
        lo = torch.zeros_like(hi)
    oj = attention(qj, kj, vj, scale=scale, bound_min=lo, bound_max=hi)
    o_img, o_txt = oj[:, :, :S_img], oj[:, :, S_img:]
    if cp == 1:
        return o_img.contiguous(), o_txt.contiguous()
    img_out = _a2a_seq_to_heads(o_img.contiguous(), group, cp)
    parts = [torch.empty_like(o_txt.contiguous()) for _ in range(cp)]
    dist.all_gather(parts, o_txt.contiguous(), group=group)
    return img_out, torch.cat(parts, 1)


__all__ = ["attention", "cross_attention", "window_attention", "ring_attention", "joint_ring_attention", "ulysses_attention",
           "joint_ulysses_attention", "attention_with_lse", "merge_partials"]
