"""Activations in 8 bits: there and back, and the gated activation that keeps its input so."""
import pytest
import torch

from block_reference import close, round8

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _x(rows, cols, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(2 * torch.randn(rows, 1, device="cuda", generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 127), (2, 128), (5, 129), (17, 1000), (300, 4096), (2, 20001), (70001, 16)])
def test_round_trip(rows, cols, dtype):
    from roc_shmem_b200.ops.checkpoint8 import restore, store
    x = _x(rows, cols, dtype, rows + cols)
    kept = store(x)
    ref = round8(x)
    assert torch.equal(restore(kept, torch.float32).double(), ref)          # a power of two loses nothing on the way back
    assert torch.equal(restore(kept), ref.to(dtype)) and kept.restore().shape == x.shape
    # a block's largest value is over 224 steps' worth, 224 * 2^-13 > 2^-6, and e4m3 has all its bits from 2^-6 on (2^-14 would be 2^-6.2)
    big = x.double().abs() >= 2.0 ** -13 * torch.nn.functional.pad(x.double().abs(), (0, -cols % 128)).view(rows, -1, 128).amax(2).repeat_interleave(128, 1)[:, :cols]
    assert ((ref - x.double()).abs()[big] <= 2.0 ** -4 * x.double().abs()[big]).all()
    assert kept.nbytes <= rows * ((cols + 15) // 16 * 16 + (cols + 127) // 128)


def test_borders_and_what_is_not_finite():
    from roc_shmem_b200.ops.checkpoint8 import restore, store
    x = torch.zeros(8, 256, device="cuda")
    x[0, :3] = torch.tensor([448.0, 447.9, 1.0])
    x[1, 0], x[1, 5] = 448.0001, 2.0 ** -9                   # the next power of two
    x[2, 7] = 3.4e38
    x[3, :2] = torch.tensor([1e-38, -1e-38])
    x[4, 1], x[4, 2] = float("inf"), 5.0
    x[5, 3], x[5, 130] = float("nan"), 7.0
    x[6, 200] = -float("inf")
    x[7, 4] = 1e-45                                           # below the smallest exponent byte: zero or a multiple of 2^-135
    ref = round8(x)
    got = restore(store(x))
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.isnan(got[4, 1]) and torch.isnan(got[6, 200])
    keep = torch.ones(8, dtype=torch.bool, device="cuda")
    keep[7] = False
    assert torch.equal(torch.nan_to_num(got[keep]).double(), torch.nan_to_num(ref[keep])) and got[4, 2] == 5.0 and got[5, 130] == 7.0
    assert (got[7].abs() <= 2.0 ** -135).all()
    for dtype in (BF, torch.float16, torch.float32):          # the type's own limits do not become infinities
        big = torch.finfo(dtype).max
        y = torch.tensor([[big, -big, big / 2, 1.0]], dtype=dtype, device="cuda")
        assert torch.equal(restore(store(y)).double(), round8(y)) and torch.isfinite(restore(store(y))).all()
    assert not restore(store(torch.zeros(3, 200, dtype=BF, device="cuda"))).any()


def test_layouts_and_outputs():
    from roc_shmem_b200.ops.checkpoint8 import restore, store
    x = _x(24, 264, BF)
    ref = restore(store(x))
    wide = torch.zeros(24, 600, dtype=BF, device="cuda")
    for at in (8, 5):
        wide[:, at:at + 264] = x
        assert torch.equal(restore(store(wide[:, at:at + 264])), ref)
        out = torch.full((24, 600), 3.0, dtype=BF, device="cuda")
        restore(store(x), out=out[:, at:at + 264])
        assert torch.equal(out[:, at:at + 264], ref) and (out[:, :at] == 3).all() and (out[:, at + 264:] == 3).all()
    assert torch.equal(restore(store(x.t().contiguous().t())), ref)
    assert torch.equal(restore(store(x.view(2, 3, 4, 264))), ref.view(2, 3, 4, 264))
    assert torch.equal(restore(store(x[0])), ref[0])
    e = store(x[:0])
    assert restore(e).shape == (0, 264)


def _gu(rows, F, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, 2 * F, device="cuda", generator=g) * 2).to(BF), torch.randn(rows, F, device="cuda", generator=g).to(BF)


def _parts(gu):
    b = gu.unflatten(1, (-1, 2, 32))
    return b[:, :, 0].flatten(1), b[:, :, 1].flatten(1)


@pytest.mark.parametrize("rows,F", [(1, 32), (3, 64), (5, 96), (130, 3584), (3000, 32)])
def test_swiglu(rows, F):
    from roc_shmem_b200.ops.checkpoint8 import restore, swiglu, swiglu_backward, swiglu_store
    gu, d = _gu(rows, F, rows + F)
    act, kept = swiglu_store(gu)
    # the fast exponential and division are within a few steps of fp32, so 32 roundings of the terms cover each
    g, u = _parts(gu.double())
    ref = g * torch.sigmoid(g) * u
    close(act, ref, ref.abs() * (1 + g.abs()))
    k = round8(gu)
    assert torch.equal(restore(kept, torch.float32).double(), k)
    dgu, again = swiglu_backward(kept, d, act=True)
    g, u = _parts(k)
    s, dd = torch.sigmoid(g), d.double()
    close(again, g * s * u, (g * s * u).abs() * (1 + g.abs()))
    dg, du = dd * u * s * (1 + g * (1 - s)), dd * g * s
    got_g, got_u = _parts(dgu)
    close(got_g.contiguous(), dg, (dd * u).abs() * s * (1 + g.abs()) ** 2)
    close(got_u.contiguous(), du, du.abs() * (1 + g.abs()))
    leaf = gu.clone().requires_grad_(True)
    out = swiglu(leaf)
    grad, = torch.autograd.grad(out, leaf, d)
    assert torch.equal(out, act) and torch.equal(grad, dgu) and torch.equal(swiglu(gu), act)
    assert torch.equal(swiglu_backward(kept, d), dgu)


def test_swiglu_layouts_and_extremes():
    from roc_shmem_b200.ops.checkpoint8 import swiglu_backward, swiglu_store
    gu, d = _gu(12, 64)
    act, kept = swiglu_store(gu)
    off = torch.zeros(12 * 128 + 1, dtype=BF, device="cuda")
    off[1:] = gu.flatten()
    a2, k2 = swiglu_store(off[1:].view(12, 128))              # off its 16-byte boundary
    assert torch.equal(a2, act) and torch.equal(k2.q, kept.q)
    a3, k3 = swiglu_store(gu.view(3, 4, 128))
    assert a3.shape == (3, 4, 64) and torch.equal(swiglu_backward(k3, d.view(3, 4, 64)).view(12, 128), swiglu_backward(kept, d))
    wide = torch.zeros(12, 100, dtype=BF, device="cuda")
    wide[:, 3:67] = d
    assert torch.equal(swiglu_backward(kept, wide[:, 3:67]), swiglu_backward(kept, d))
    big = torch.zeros(2, 64, dtype=BF, device="cuda")
    big[0, 0], big[0, 32], big[1, 0], big[1, 32] = 1e4, 2.0, -1e4, 2.0      # gates beyond the exponential's range
    act, kept = swiglu_store(big)
    assert act[0, 0] == big[0, 0] * 2 and act[1, 0] == 0 and torch.isfinite(swiglu_backward(kept, torch.ones_like(act)).float()).all()
    act, kept = swiglu_store(gu[:0])
    assert act.shape == (0, 64) and swiglu_backward(kept, d[:0]).shape == (0, 128)


def test_refusals():
    from roc_shmem_b200.ops.checkpoint8 import restore, store, swiglu_backward, swiglu_store
    x, (gu, d) = _x(4, 64, BF), _gu(4, 64)
    _, kept = swiglu_store(gu)
    for bad in (lambda: store(x.cpu()), lambda: store(x.double()), lambda: store(x[:, :0]), lambda: store(torch.tensor(1.0, device="cuda")),
                lambda: restore(store(x), torch.float64), lambda: restore(store(x), out=x[:, :60]), lambda: restore(store(x), torch.float32, out=x),
                lambda: swiglu_store(gu[:, :96]), lambda: swiglu_store(gu.half()), lambda: swiglu_store(gu.cpu()),
                lambda: swiglu_backward(kept, d[:, :32]), lambda: swiglu_backward(kept, d.float()), lambda: swiglu_backward(kept, d[:3]),
                lambda: swiglu_backward(kept, d, dgu_out=gu[:, ::2]), lambda: swiglu_backward(kept, d, act_out=d.float())):
        with pytest.raises(ValueError):
            bad()


def test_graph_capture():
    from roc_shmem_b200.ops.checkpoint8 import restore, store, swiglu_backward, swiglu_store
    gu, d = _gu(64, 128)
    swiglu_backward(swiglu_store(gu)[1], d, act=True), restore(store(d))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        act, kept = swiglu_store(gu)
        got = (act, *swiglu_backward(kept, d, act=True), restore(store(d)))
    n, m = _gu(64, 128, 5)
    gu.copy_(n), d.copy_(m)
    g.replay()
    act, kept = swiglu_store(gu)
    assert all(torch.equal(a, b) for a, b in zip(got, (act, *swiglu_backward(kept, d, act=True), restore(store(d)))))
