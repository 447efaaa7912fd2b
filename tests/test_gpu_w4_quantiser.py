"""What the quantiser of 4-bit weights makes of values that are not finite, or near the end of their type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zeros", [False, True])
def test_not_finite(group, zeros):
    """A group with such a value is NaN as a whole, every other one is what it is without."""
    from roc_shmem_b200.ops.gemm_w4 import linear_w4, quantize_w4, widen_w4
    clean = (torch.randn(12, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(group)) * 0.05).to(BF)
    w = clean.clone()
    spots = ((0, 0, "nan"), (2, 511, "nan"), (3, group - 1, "inf"), (5, group, "-inf"), (7, 31, "-nan"), (8, 17, "inf"), (8, 18, "-inf"))
    hit = torch.zeros(12, 512 // group, dtype=torch.bool, device="cuda")
    for row, col, what in spots:
        w[row, col] = -float("nan") if what == "-nan" else float(what)
        hit[row, col // group] = True
    t, ref = quantize_w4(w, group, zeros=zeros), quantize_w4(clean, group, zeros=zeros)
    whole = hit.repeat_interleave(group, 1)
    assert torch.equal(torch.isnan(t.scales), hit)
    for got, expect in ((t.dequantize(), ref.dequantize()), (widen_w4(t), widen_w4(ref))):
        assert torch.isnan(got[whole]).all() and torch.equal(got[~whole], expect[~whole])
    assert torch.equal(t.scales[~hit], ref.scales[~hit]) and (not zeros or torch.equal(t.zeros[~hit], ref.zeros[~hit]))
    x = torch.randn(3, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF)
    got, rows = linear_w4(x, t), hit.any(1)
    assert torch.isnan(got[:, rows]).all() and torch.equal(got[:, ~rows], linear_w4(x, ref)[:, ~rows])


def test_range_beyond_fp32():
    """Weights of both signs near the end of their type: the range is twice what fp32 holds, the scale a fifteenth of it.  The scale's own
    error is half a step of bf16 (2^-8) and three fp32 roundings; a weight is off by half a step, half a step more for the zero point, and
    by what up to 15 steps lack of the scale."""
    from roc_shmem_b200.ops.gemm_w4 import quantize_w4
    w = torch.zeros(4, 64, dtype=BF, device="cuda")
    for row, (lo, hi) in enumerate(((-3e38, 3e38), (-2e38, 1.9e38), (-1e38, 3.3e38), (-1.6e38, 1.6e38))):
        w[row] = torch.linspace(lo / 1e38, hi / 1e38, 64, device="cuda", dtype=torch.float64).mul(1e38).to(BF)
    t = quantize_w4(w, 64, zeros=True)
    d = w.double()
    s = (d.amax(1) - d.amin(1)) / 15
    assert ((t.scales.double()[:, 0] - s).abs() <= s * (2.0 ** -8 + 2.0 ** -22)).all()
    back = (torch.stack((t.q & 15, t.q >> 4), 2).flatten(1).double() - t.zeros.double()) * t.scales.double()
    assert ((back - d).abs() <= t.scales.double() * (1 + 15 * 2.0 ** -8)).all()
