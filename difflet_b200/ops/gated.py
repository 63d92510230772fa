"""The gated projection of a feed-forward block, and its gradients.

``gated_linear`` evaluates ``act(x W_gate^T) * (x W_up^T)`` (the first half of the SwiGLU / gated-GELU blocks of the
prompt encoders) as one kernel: both products, the activation and the multiplication (``csrc/glu.cu``).  The down projection
is an ordinary ``linear``.  The weights stay as checkpoints hold them, two [F, K] tensors or the halves of one.
"""

from __future__ import annotations

import torch

from difflet_b200.ops import fused as F


_PLAIN = (torch.Tensor, torch.nn.Parameter)


def gated_linear(x, w_gate, w_up, *, act="silu"):
    """``act(x w_gate^T) * (x w_up^T)``: x [..., K]; w_gate, w_up [F, K] -> [..., F].

    ``act``: "silu", "gelu" / "gelu_tanh" (tanh form) or "gelu_erf".  Products are accumulated and the activation is
    evaluated in f32; the result is rounded to x's type once.  Differentiable in all three (once): the two projections are
    kept in f32 for it (8 bytes a value of the result), their gradients are
    rounded to x's type.  CUDA: bf16 and fp16 with K a multiple of 8; other types and sizes, tracing,
    function transforms and forward-mode tangents run as torch operations."""
    if x.is_cuda and act in F.GATED_ACTS and type(x) in _PLAIN and not torch.compiler.is_compiling():
        try:  # the binding checks everything; what it refuses is looked at again below
            h = (F._nat or F._lib()).gated_linear(x, w_gate, w_up, F.GATED_ACTS[act])
            F.LAUNCHES[0] += 1
            return h
        except (ValueError, TypeError):
            pass
    if isinstance(w_gate, F.MXWeight) or isinstance(w_up, F.MXWeight):
        raise NotImplementedError("gated_linear with block-scaled weights: dequantize() them first")
    if act not in F.GATED_ACTS:
        raise ValueError(f"act {act!r}: one of {sorted(F.GATED_ACTS)}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_gate.shape[1] != x.shape[-1]:
        raise ValueError(f"x [..., K] and two weights [F, K] expected, got {tuple(x.shape)}, {tuple(w_gate.shape)}, {tuple(w_up.shape)}")
    for name, t in (("w_gate", w_gate), ("w_up", w_up)):
        if t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f"{name} {t.dtype} on {t.device} does not match x {x.dtype} on {x.device}")
    if not x.is_floating_point():
        raise ValueError(f"gated_linear needs floating-point tensors, got {x.dtype}")
    return F.gated_linear(x, w_gate, w_up, act)


__all__ = ["gated_linear"]
