"""Products with 4-bit weights and their quantiser against formulas in 64 bits."""
import pytest
import torch

from block_reference import close

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _weight(N, K, group, zeros, seed=0):
    from roc_shmem_b200.ops.gemm_w4 import W4Tensor
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    s = (torch.rand(N, K // group, device="cuda", generator=g) + 0.01).to(BF)
    z = torch.randint(0, 16, (N, K // group), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    return W4Tensor(q, s, z)


def _x(T, K, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, K, device="cuda", generator=g).to(BF)


def _exact(w):
    lo, hi = (w.q & 15).double(), (w.q >> 4).double()
    q = torch.stack((lo, hi), -1).flatten(1)
    z = 8.0 if w.zeros is None else w.zeros.double().repeat_interleave(w.group, 1)
    return (q - z) * w.scales.double().repeat_interleave(w.group, 1)


def _check(x, w, got):
    """Few tokens: the products are exact, sums of K terms in fp32.  The tensor core may cut where fp32 rounds (a whole step), so each
    term counts twice.  Many: each weight is rounded to bf16 as well, half a step of it."""
    from roc_shmem_b200.ops.gemm_w4 import few_tokens
    m = _exact(w)
    size = x.double().abs() @ m.abs().t()
    steps = 2 * (x.shape[1] // 16 + 16)
    if x.shape[0] > few_tokens(w.group) and m.shape[0] % 8 == 0:
        steps += 2.0 ** -8 / 2.0 ** -24
    close(got, x.double() @ m.t(), size, steps)


@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, True), (128, False), (128, True), (256, False)])
@pytest.mark.parametrize("N,K", [(1, 256), (17, 512), (40, 768), (264, 1280), (2048, 2048)])
def test_tokens(N, K, group, zeros):
    from roc_shmem_b200.ops.gemm_w4 import linear_w4
    w = _weight(N, K, group, zeros, N + K + group)
    for T in (1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 65, 200):
        x = _x(T, K, T)
        _check(x, w, linear_w4(x, w))


@pytest.mark.parametrize("K,group", [(32, 32), (64, 64), (96, 32), (160, 32), (192, 64), (128, 128), (384, 384), (4128, 32)])
def test_columns_that_end_inside_a_step(K, group):
    from roc_shmem_b200.ops.gemm_w4 import linear_w4
    w = _weight(100, K, group, True, K)
    for T in (1, 5, 12, 30):
        x = _x(T, K, T)
        _check(x, w, linear_w4(x, w))


@pytest.mark.parametrize("T,N,K", [(1, 16, 16384), (3, 48, 8192), (16, 7168, 8192), (24, 300, 4096), (1, 8192, 3584)])
def test_split_columns(T, N, K):
    """Few rows: clusters of blocks share a tile's columns."""
    from roc_shmem_b200.ops.gemm_w4 import linear_w4
    w, x = _weight(N, K, 128, True), _x(T, K)
    first = linear_w4(x, w)
    _check(x, w, first)
    assert torch.equal(first, linear_w4(x, w))


def test_layouts():
    from roc_shmem_b200.ops.gemm_w4 import linear_w4
    w, x = _weight(64, 512, 128, False), _x(6, 512)
    ref = linear_w4(x, w)
    wide = torch.zeros(6, 900, dtype=BF, device="cuda")
    for at in (8, 3):
        wide[:, at:at + 512] = x
        assert torch.equal(linear_w4(wide[:, at:at + 512], w), ref)
    assert torch.equal(linear_w4(x.t().contiguous().t(), w), ref) and torch.equal(linear_w4(x.view(2, 3, 512), w), ref.view(2, 3, 64))
    assert torch.equal(linear_w4(x[2], w), ref[2]) and torch.equal(linear_w4(x[:1].expand(6, 512), w), ref[:1].expand(6, 64))
    assert linear_w4(x[:0], w).shape == (0, 64)
    x[3, 7] = float("nan")                                    # stays in its token
    got = linear_w4(x, w)
    assert torch.isnan(got[3]).all() and torch.equal(got[[0, 1, 2, 4, 5]], ref[[0, 1, 2, 4, 5]])


@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False), (128, True), (256, True)])
def test_quantiser(group, zeros):
    from roc_shmem_b200.ops.gemm_w4 import quantize_w4, widen_w4
    g = torch.Generator(device="cuda").manual_seed(group)
    w = (torch.randn(37, 768, device="cuda", generator=g) * 0.05 + 0.01 * zeros).to(BF)
    w[3] = 0
    w[4, :group] = 0.25                                       # one sign only
    w[5] = w[5].abs()
    t = quantize_w4(w, group, zeros=zeros)
    b = w.double().view(37, -1, group)
    lo, hi = b.amin(2).clamp(max=0), b.amax(2).clamp(min=0)
    s = ((hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7)
    # bf16 has 7 bits behind the first one: half a step is up to 2^-8 of the scale (at 1.0 the step is 2^-7); the range's
    # difference and quotient are two fp32 roundings more
    assert ((t.scales.double() - s).abs() <= s * (2.0 ** -8 + 2.0 ** -22)).all()
    # nearest of sixteen: half a step, and what a scale that rounded down leaves out at the ends: 8 steps at most lack 2^-8 of
    # themselves; a zero point rounds the range by half a step more
    err = (t.dequantize().double() - w.double()).abs().view(37, -1, group)
    step = t.scales.double().unsqueeze(2)
    assert (err <= step * (0.5 + 16 * 2.0 ** -8 + (0.5 if zeros else 0))).all()
    assert torch.equal(widen_w4(t), t.dequantize().to(BF))
    wide = torch.zeros(37, 1000, dtype=BF, device="cuda")
    wide[:, 5:773] = w
    again = quantize_w4(wide[:, 5:773], group, zeros=zeros)
    assert torch.equal(again.q, t.q) and torch.equal(again.scales, t.scales)


def test_layer():
    from roc_shmem_b200.ops.gemm_w4 import LinearW4, linear_w4, quantize_w4
    from roc_shmem_b200.ops.torch_ops import Linear
    layer = Linear(512, 264, device="cuda")
    served = LinearW4.from_linear(layer, 64, zeros=True)
    x = _x(3, 512)
    w = quantize_w4(layer.weight.detach(), 64, zeros=True)
    assert torch.equal(served(x), linear_w4(x, w)) and served.out_features == 264
    other = LinearW4(_weight(264, 512, 64, True))
    other.load_state_dict(served.state_dict())
    assert torch.equal(other(x), served(x))


def test_graph_capture_and_streams():
    from roc_shmem_b200.ops.gemm_w4 import linear_w4
    w = _weight(512, 4096, 128, False)
    for T in (1, 40):
        x = _x(T, 4096)
        ref = linear_w4(x, w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = linear_w4(x, w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, ref)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear_w4(x, w)
        x.copy_(_x(T, 4096, 9))
        graph.replay()
        assert torch.equal(out, linear_w4(x, w))


def test_refusals():
    from roc_shmem_b200.ops.gemm_w4 import LinearW4, W4Tensor, linear_w4, quantize_w4
    w, x = _weight(64, 512, 128, True), _x(4, 512)
    m = _x(64, 512)
    for bad in (lambda: linear_w4(x[:, :256], w), lambda: linear_w4(x.float(), w), lambda: linear_w4(x.cpu(), w), lambda: linear_w4(x.clone().requires_grad_(True), w),
                lambda: linear_w4(x, W4Tensor(w.q, w.scales[:, :3], None)), lambda: linear_w4(x, W4Tensor(w.q, w.scales.float(), None)),
                lambda: linear_w4(x, W4Tensor(w.q, w.scales, w.zeros[:, :2])), lambda: linear_w4(x, W4Tensor(w.q.int(), w.scales, None)),
                lambda: linear_w4(x, W4Tensor(w.q.t().contiguous().t(), w.scales, None)), lambda: linear_w4(x, W4Tensor(w.q.cpu(), w.scales, None)),
                lambda: linear_w4(x, W4Tensor(w.q, w.scales[:32], None)), lambda: quantize_w4(m, 48), lambda: quantize_w4(m, 96), lambda: quantize_w4(m[:, :500]),
                lambda: quantize_w4(m.float()), lambda: quantize_w4(m.t()), lambda: quantize_w4(m, 0), lambda: quantize_w4(m.cpu()),
                lambda: LinearW4.from_linear(torch.nn.Linear(512, 64, device="cuda", dtype=BF))):
        with pytest.raises(ValueError):
            bad()
