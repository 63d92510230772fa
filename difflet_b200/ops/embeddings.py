"""Embedding lookup and rotary embeddings.

``embedding``: rows of a table, scaled, with a gradient for the table (``csrc/embed.cu``).

Rotary embeddings of the public op surface (difflet/ops/embeddings.py; laws of
difflet/backends/_torch_megatron/embeddings.py:13-37).  Tables are full head-dim
``cos`` / ``sin`` with each frequency repeated for its (even, odd) pair.  The built-in
models rotate q/k inside the fused norm + RoPE + scatter kernel instead."""

from __future__ import annotations

import torch

from difflet_b200.ops import fused as F


_PLAIN = (torch.Tensor, torch.nn.Parameter)


def embedding(ids, weight, *, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: ids of any shape and integer type, weight [V, D] -> [..., D].

    The product is formed in f32 and rounded once.  Differentiable in ``weight`` (once): the gradient is a dense [V, D] of its
    type, every row summed in f32 in the order of the ids; the row ``padding_idx`` (negative: from the end) gets none.
    CUDA: bf16, fp16 and fp32; an id outside the table gives a row of zeros and no gradient, and sets the device error word
    (``_native.check_device_errors`` raises it); on the CPU it raises IndexError.  Other types, tracing, function transforms and
    forward-mode tangents run as torch operations."""
    if weight.is_cuda and type(weight) in _PLAIN and not torch.compiler.is_compiling():
        try:  # the binding checks everything; what it refuses is looked at again below
            y = (F._nat or F._lib()).embedding(ids, weight, scale, padding_idx)
            F.LAUNCHES[0] += 1
            return y
        except ValueError:
            pass
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"weight must be floating-point [V, D], got {tuple(weight.shape)} {weight.dtype}")
    if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
        raise ValueError(f"ids must be integers, got {ids.dtype}")
    if ids.device != weight.device:
        raise ValueError(f"ids on {ids.device}, weight on {weight.device}")
    V, pad = weight.shape[0], None
    if padding_idx is not None:
        pad = int(padding_idx) + (V if padding_idx < 0 else 0)
        if not 0 <= pad < V:
            raise ValueError(f"padding_idx {padding_idx} is not a row of {V}")
    return F.embedding(ids, weight, float(scale), pad)


def apply_rotary_emb(hidden_states, freqs_cos, freqs_sin):
    """Interleaved pairs (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos), in the input dtype."""
    dt = hidden_states.dtype
    x1, x2 = hidden_states.unflatten(-1, (-1, 2)).unbind(-1)
    cos = freqs_cos[..., 0::2]
    sin = freqs_sin[..., 1::2]
    out = torch.empty_like(hidden_states)
    out[..., 0::2] = x1 * cos - x2 * sin
    out[..., 1::2] = x1 * sin + x2 * cos
    return out.to(dt)


def apply_rotary_emb_fp32(hidden_states, freqs_cos, freqs_sin):
    """The same rotation evaluated in fp32 (x cos + rot(x) sin), cast back."""
    x = hidden_states
    re, im = x.reshape(*x.shape[:-1], -1, 2).unbind(-1)
    rot = torch.stack([-im, re], dim=-1).flatten(-2)
    return (x.float() * freqs_cos + rot.float() * freqs_sin).to(x.dtype)


def apply_rotary_emb_slices(hidden_states, freqs_cos, freqs_sin):
    """The interleaved law computed with stride-2 slices (identical to ``apply_rotary_emb``)."""
    return apply_rotary_emb(hidden_states, freqs_cos, freqs_sin)


__all__ = ["embedding", "apply_rotary_emb", "apply_rotary_emb_fp32", "apply_rotary_emb_slices"]
