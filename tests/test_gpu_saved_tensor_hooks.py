"""Hooks on saved tensors that bring them back at another place: on the host and back, off any boundary, with other strides."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _off(t):
    """The same values behind one more element of the type."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    return flat[1:].view(t.shape)


def _apart(t):
    """The same values with a gap behind each."""
    wide = torch.empty((*t.shape, 2), dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


@pytest.mark.parametrize("unpack", [_off, _apart, lambda t: t.cpu().cuda()], ids=["off", "apart", "host"])
@pytest.mark.parametrize("rows,n,checkpoint", [(7, 200, True), (1500, 1024, True), (9, 257, True), (1500, 1024, False), (9, 264, False)])
def test_norms(unpack, rows, n, checkpoint):
    from roc_shmem_b200.ops.norms import post_pre_norm

    def rand(*shape, seed):
        return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(BF)
    leaves = [rand(rows, n, seed=1), rand(rows, n, seed=2), rand(n, seed=3), rand(n, seed=4), rand(rows, n, seed=5)]
    for t in leaves:
        t.requires_grad_(True)
    y, x, w, w2, g = leaves
    dys = [rand(rows, n, seed=6), rand(rows, n, seed=7)]

    def step():
        return torch.autograd.grad(post_pre_norm(y, x, w, w2, gate=g, scale=0.5, checkpoint=checkpoint), leaves, dys)
    expect = step()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: unpack(t.detach())):
        got = step()
    # Weights off their boundary turn the call into one value by value, whose sums are taken in another order.  Either result is within half a step
    # of bf16 (2^-8) of the exact one, and fp32 sums add 64 roundings of the terms, far less than 2^-12 of the norm.
    for a, b in zip(got, expect):
        assert (a.double() - b.double()).norm() <= (2.0 ** -7 + 2.0 ** -12) * b.double().norm()
