"""Bytes of kept activations that hold no value are zeros, whatever lay there before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _soil(size, byte):
    """Leaves `byte` in the memory that the allocator hands out next."""
    torch.full((size,), byte, dtype=torch.uint8, device="cuda")


def _rand(rows, n, dtype):
    return torch.randn(rows, n, device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n", [(3, 1), (5, 8), (7, 120), (9, 129), (200, 1000), (3, 264)])
def test_store(rows, n, dtype):
    from roc_shmem_b200.ops.checkpoint8 import kept_bytes, store
    x = _rand(rows, n, dtype)
    found = []
    for byte in (255, 90):
        _soil(kept_bytes(rows, n), byte)
        found.append(store(x))
    assert not found[0].q[:, n:].any() and torch.equal(found[0].data, found[1].data)


@pytest.mark.parametrize("rows,n", [(3, 1), (5, 8), (7, 120), (9, 129), (201, 1000), (3, 264), (5001, 232), (701, 8200), (1001, 257)])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_norms(rows, n, mode):
    from roc_shmem_b200.ops import norms
    x = _rand(rows, n, torch.bfloat16)
    count = 2 if mode == norms.POST_PRE else 1
    size, width = norms.kept_size(count, rows, n), (n + 15) // 16 * 16
    found = []
    for byte in (255, 90):
        c = norms._Call("norm", mode, x if mode != norms.PRE else None, x, None, None, None, None, 1e-6, True)
        _soil(size, byte)
        found.append(norms._forward(c, mode, True)[3])
    q, rest = found[0][:count * rows * width].view(-1, width), found[0][count * rows * (width + (n + 127) // 128):]
    assert not q[:, n:].any() and not rest.any() and torch.equal(found[0], found[1])
