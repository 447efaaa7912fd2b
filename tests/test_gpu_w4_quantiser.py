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
