"""Low-rank adapters of many requests beside one shared projection.

``LoraBank`` holds the adapters of one Linear (``A_i [r_i, K]``, ``B_i [N, r_i]`` and a factor, alpha / r in
LoRA's terms) laid out once; ``linear_lora`` evaluates

    y = act(x W^T + b + s_i (x A_i^T) B_i^T)

where every row (or every request's rows) names its adapter ``i``, -1 for none.  On CUDA the adapters' terms
are accumulated inside the base projection's tcgen05 GEMM (``csrc/lora.cu``): the rows of a batch may
mix adapters freely, without sorting, and the ids stay on the device.
"""

from __future__ import annotations

import torch

from difflet_b200.ops import fused as F


def _padded_rank(r: int) -> int:
    return -(-r // 16) * 16 if r <= 64 else 128


class LoraBank:
    """Adapters of one projection: ``A`` [n, r, K] or a list of [r_i, K]; ``B`` [n, N, r] or a list of
    [N, r_i]; ``scale``: one factor per adapter (numbers or a tensor; default 1).  Ranks up to 128 (shorter ones
    are padded with zeros to the longest, in steps of 16), at most 1024 adapters.

    The weights must be finite (checked here; also after later changes in place).  Kept in A's type on A's device; tensors
    that already have the padded layout are used as they are.  No gradient is recorded: tensors that ask for one are refused
    outside ``torch.no_grad()``."""

    MAX_ADAPTERS, MAX_RANK = 1024, 128

    def __init__(self, A, B, scale=None):
        a, b = list(A), list(B)
        n = len(a)
        if not 1 <= n <= self.MAX_ADAPTERS or len(b) != n:
            raise ValueError(f"1 to {self.MAX_ADAPTERS} adapters with one A and one B each, got {n} and {len(b)}")
        K, N = a[0].shape[-1], b[0].shape[0]
        for i, (x, y) in enumerate(zip(a, b)):
            if x.dim() != 2 or y.dim() != 2 or x.shape[1] != K or y.shape[0] != N or x.shape[0] != y.shape[1]:
                raise ValueError(f"adapter {i}: A [r, {K}] and B [{N}, r] expected, got {tuple(x.shape)}, {tuple(y.shape)}")
            if not 1 <= x.shape[0] <= self.MAX_RANK:
                raise ValueError(f"adapter {i}: rank {x.shape[0]} is not in 1..{self.MAX_RANK}")
            if x.dtype != a[0].dtype or y.dtype != a[0].dtype or x.device != a[0].device or y.device != a[0].device:
                raise ValueError(f"adapter {i} differs from the first one in type or device")
        F._no_grad("LoraBank", *a, *b, scale if torch.is_tensor(scale) else None)
        if not a[0].is_floating_point():
            raise ValueError(f"adapters are floating-point tensors, got {a[0].dtype}")
        self.n, self.in_features, self.out_features = n, K, N
        self.ranks = [x.shape[0] for x in a]
        self.rank = R = _padded_rank(max(self.ranks))
        dev, dt = a[0].device, a[0].dtype
        self.A = self._laid_out(A, a, (n, R, K))
        self.B = self._laid_out(B, b, (n, N, R))
        if scale is None:
            scale = [1.0] * n
        if not bool(torch.isfinite(self.A).all() & torch.isfinite(self.B).all()):
            # a tile of rows multiplies the adapters of its neighbours by zero: 0 * inf would reach them
            raise ValueError("the adapters hold infinities or NaN")
        s = scale.detach() if torch.is_tensor(scale) else torch.tensor([float(v) for v in scale])
        if s.shape != (n,):
            raise ValueError(f"scale holds one factor for each of the {n} adapters")
        self.scale = s.to(device=dev, dtype=torch.float64 if dt == torch.float64 else torch.float32).contiguous()

    @staticmethod
    def _laid_out(given, parts, shape):
        if torch.is_tensor(given) and given.shape == shape and given.is_contiguous() and given.data_ptr() % 16 == 0:
            return given.detach()
        out = torch.zeros(shape, dtype=parts[0].dtype, device=parts[0].device)
        for o, x in zip(out, parts):
            o[:x.shape[0], :x.shape[1]] = x.detach()
        return out

    @property
    def device(self):
        return self.A.device

    @property
    def dtype(self):
        return self.A.dtype

    def to(self, device=None, dtype=None) -> "LoraBank":
        ranks = self.ranks
        bank = LoraBank([x[:r].to(device=device, dtype=dtype) for x, r in zip(self.A, ranks)],
                        [x[:, :r].to(device=device, dtype=dtype) for x, r in zip(self.B, ranks)], self.scale)
        return bank


def linear_lora(x, w, b=None, *, bank: LoraBank, ids, rows_per_batch: int = 0, act=None, act_lo=0, act_hi=None, gate=None,
                resid=None, gate_rows_per_batch: int = 0, out=None, out_f32: bool = False):
    """``act(x W^T + b + s_i (x A_i^T) B_i^T)``, or ``resid + gate * (...)``: ``ops.fused.linear`` with adapters.

    x [..., K]; w [N, K] (or an ``MXWeight`` with ``compute="dequant"``); ``ids`` (int32 / int64, on x's device):
    the adapter of each row, or with ``rows_per_batch`` of each run of that many rows; -1 (or any
    number outside the bank, which also sets the device error word) means none.  ``gate`` f32 [B, N] with
    ``gate_rows_per_batch`` rows each (0: ``rows_per_batch``, else all).  The rank-r
    intermediate is rounded to x's type once; everything is accumulated in f32 and rounded at the end."""
    F._no_grad("linear_lora", x, b, gate, resid, None if isinstance(w, F.MXWeight) else w)
    if act not in (None, "none", "gelu", "gelu_tanh", "silu"):
        raise ValueError(f"act {act!r}: linear_lora has none, gelu and silu")
    if gate is not None and act not in (None, "none"):
        raise ValueError("act and gate are mutually exclusive")
    if out_f32 and (gate is not None or act not in (None, "none")):
        raise ValueError("out_f32 comes without act and gate")
    rpb = gate_rows_per_batch or rows_per_batch
    if x.is_cuda and not isinstance(w, F.MXWeight):  # the binding checks shapes, types and devices (ValueError)
        return F.linear_lora(x, w, b, bank, ids, rows_per_batch, act=act, act_lo=act_lo, act_hi=act_hi, gate=gate,
                             resid=resid, gate_rows_per_batch=rpb, out=out, out_f32=out_f32)
    if x.dim() < 1 or x.shape[-1] != bank.in_features:
        raise ValueError(f"x {tuple(x.shape)} does not end in the bank's {bank.in_features} inputs")
    if tuple(w.shape) != (bank.out_features, bank.in_features):
        raise ValueError(f"weight {tuple(w.shape)} is not [{bank.out_features}, {bank.in_features}]")
    if bank.device != x.device or w.device != x.device or ids.device != x.device:
        raise ValueError("x, weight, bank and ids must be on one device")
    if (gate is None) != (resid is None):
        raise ValueError("gate and resid come together")
    x2 = F._rows2d(x)
    M, N = x2.shape[0], bank.out_features
    if ids.is_floating_point() or ids.dim() != 1:
        raise ValueError("ids must be a vector of integers")
    want = M if rows_per_batch <= 0 else -(-M // rows_per_batch)
    if ids.shape[0] != want:
        raise ValueError(f"{want} ids expected for {M} rows" + (f" of {rows_per_batch} a batch" if rows_per_batch > 0 else "")
                         + f", got {ids.shape[0]}")
    if b is not None and tuple(b.shape) != (N,):
        raise ValueError(f"bias must be [{N}], got {tuple(b.shape)}")
    if gate is not None and (gate.dim() != 2 or gate.shape[1] < N or gate.shape[0] * (rpb if rpb > 0 else M) < M):
        raise ValueError(f"gate must be [B, {N}] with a row for every {rpb if rpb > 0 else M} rows, got {tuple(gate.shape)}")
    if resid is not None and tuple(resid.shape) != (*x.shape[:-1], N):
        raise ValueError(f"resid must be {(*x.shape[:-1], N)}, got {tuple(resid.shape)}")
    if isinstance(w, F.MXWeight):
        if w.compute == "mx":
            raise NotImplementedError("linear_lora beside a block-scaled weight: use MXWeight(compute='dequant')")
        w = w.dequantize(x.dtype)
    if w.dtype != x.dtype or bank.dtype != x.dtype:
        raise ValueError(f"x {x.dtype}, weight {w.dtype} and bank {bank.dtype} differ in type")
    res2 = None if resid is None else F._rows2d(resid)
    out2 = None
    if out is not None:
        if out.shape != (*x.shape[:-1], N):
            raise ValueError(f"out must be {(*x.shape[:-1], N)}, got {tuple(out.shape)}")
        out2 = out if out.dim() == 2 else out.view(M, N)
    y = F.linear_lora(x2, w, b, bank, ids, rows_per_batch, act=act, act_lo=act_lo, act_hi=act_hi, gate=gate, resid=res2,
                      gate_rows_per_batch=rpb, out=out2, out_f32=out_f32)
    return out if out is not None else (y if x.dim() == 2 else y.view(*x.shape[:-1], N))


__all__ = ["LoraBank", "linear_lora"]
