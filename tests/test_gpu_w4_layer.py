"""A layer with 4-bit weights after its products: what it reports of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def test_check_after_products_of_both_kernels():
    from roc_shmem_b200.ops.gemm_w4 import LinearW4, quantize_w4
    layer = LinearW4(quantize_w4((torch.randn(264, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 0.05).to(BF)))
    for tokens in (1, 40, 300):
        layer(torch.ones(tokens, 512, device="cuda", dtype=BF))
    layer.check()
