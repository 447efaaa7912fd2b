"""Norms whose rows are no whole eights, or lie off 16-byte boundaries, with rows enough for blocks that walk over several of them and end
on a part of a block: values, gradients of every operand and the sums over rows, with and without 8 bits."""
import pytest
import torch

from test_gpu_norms import BF, F32, HF, _call, _case, _check_backward, _check_forward, _train

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", [(1000, 4100), (5001, 233), (3001, 7), (1999, 1030), (450, 12001), (20011, 129)])
@pytest.mark.parametrize("mode,dtype,w,gate,scale", [
    ("pre", F32, F32, None, None), ("pre", BF, F32, None, None), ("post", BF, BF, "column", "tensor"), ("post", HF, HF, "row", "tensor"),
    ("post", F32, F32, "element", 0.5), ("post_pre", BF, BF, "row", "tensor"), ("post_pre", HF, F32, "element", "tensor"),
    ("post_pre", F32, F32, "column", "tensor"), ("post_pre", BF, BF, None, None)])
@pytest.mark.parametrize("kept8", [False, True])
def test_many_odd_rows(rows, n, mode, dtype, w, gate, scale, kept8):
    c = _case(rows, n, dtype, gate, w, scale, seed=n + rows)
    got, grads = _train(mode, c, kept8)
    _check_forward(mode, c, got)
    _check_backward(mode, c, got[0] if mode == "post_pre" else got, grads, kept8, rows)


@pytest.mark.parametrize("rows,n", [(2501, 520), (601, 4096), (301, 8208)])
@pytest.mark.parametrize("mode,gate", [("pre", None), ("post", "element"), ("post_pre", "column")])
@pytest.mark.parametrize("kept8", [False, True])
def test_many_rows_off_their_boundary(rows, n, mode, gate, kept8):
    """Whole eights, three elements behind a boundary and apart."""
    c = _case(rows, n, BF, gate, BF, "tensor", seed=n)
    for name in ("x", "y"):
        wide = torch.zeros(rows, n + 5, dtype=BF, device="cuda")
        wide[:, 3:n + 3] = c[name]
        c[name] = wide[:, 3:n + 3]
    got, grads = _train(mode, c, kept8)
    _check_forward(mode, c, got)
    _check_backward(mode, c, got[0] if mode == "post_pre" else got, grads, kept8, rows)


@pytest.mark.parametrize("rows,n", [(1000, 4100), (450, 12001)])
def test_the_same_bits_again(rows, n):
    c = _case(rows, n, BF, "row", BF, "tensor", seed=1)
    first, second = (_train("post_pre", dict(c), True) for _ in range(2))
    assert all(torch.equal(a, b) for a, b in zip((*first[0], *first[1].values()), (*second[0], *second[1].values())))
    assert all(torch.equal(a, b) for a, b in zip(_call("post_pre", c), first[0]))
