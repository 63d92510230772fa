"""What ``ops.add_rms_norm`` accepts beside ``test_add_rms_norm``'s cases."""

import pytest
import torch

from difflet_b200 import ops

BF = torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("pad", [3, 4, 8])
def test_one_row_of_any_pitch(native, pad, dtype):
    """A single aligned row cut from a matrix of an odd width: a row has no stride to speak of, the MX output takes it."""
    D = 512
    g = torch.Generator().manual_seed(0)
    big = [torch.randn(3, D + pad, generator=g).to("cuda", dtype) for _ in range(4)]
    x, resid, s_out, y_out = (t[:1, :D] for t in big)
    mods = [torch.randn(2, D + pad, generator=g).cuda()[:1, :D] for _ in range(2)]
    plain = [t.clone(memory_format=torch.contiguous_format).reshape(-1).clone().view(1, D) for t in (x, resid, *mods)]
    kw = dict(scale=mods[0], shift=mods[1])
    own = dict(scale=plain[2], shift=plain[3])
    for q in (None, "float8_e4m3fn", "float8_e5m2"):
        for blocked in (False, True) if q else (False,):
            y, s = ops.add_rms_norm(x, resid, quantize=q, blocked=blocked, **kw)
            want, s_want = ops.add_rms_norm(plain[0], plain[1], quantize=q, blocked=blocked, **own)
            assert torch.equal(s, s_want)
            for a, b in zip(y, want) if q else ((y, want),):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    rest = [t.clone() for t in big]
    y, s = ops.add_rms_norm(x, resid, out=y_out, resid_out=s_out, **kw)
    want, s_want = ops.add_rms_norm(plain[0], plain[1], **own)
    assert torch.equal(y, want) and torch.equal(s, s_want) and y is y_out and s is s_out
    for t, was in zip(big, rest):
        assert torch.equal(t[1:], was[1:]) and torch.equal(t[:, D:], was[:, D:])


def test_a_row_map_entry_that_does_not_exist():
    """An error (on CUDA in the device error word); -1 is not the last row."""
    x, mod = torch.randn(3, 8), torch.randn(2, 8)
    for kw in (dict(scale=mod), dict(shift=mod), dict(scale=mod, shift=mod)):
        ops.add_rms_norm(x, row_map=torch.tensor([0, 1, 1], dtype=torch.int32), **kw)
        for bad in (-1, 2):
            with pytest.raises(IndexError):
                ops.add_rms_norm(x, row_map=torch.tensor([0, bad, 1], dtype=torch.int32), **kw)


@pytest.mark.gpu
def test_results_whose_rows_overlap_are_refused(native):
    """One row of memory for all rows (expand), or rows that run into one another."""
    x = torch.randn(5, 64, device="cuda")
    one, close = torch.empty(1, 64, device="cuda").expand(5, 64), torch.empty(400, device="cuda").as_strided((5, 64), (32, 1))
    for bad in (one, close):
        with pytest.raises(ValueError, match="overlap"):
            ops.add_rms_norm(x, out=bad)
        with pytest.raises(ValueError, match="overlap"):
            ops.add_rms_norm(x, x, resid_out=bad)
    y, s = ops.add_rms_norm(one, one)  # (inputs may)
    assert torch.equal(s, one + one)
