"""Norms, 8-bit activations and 4-bit weights together, as a block's training and serving use them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture
def rt():
    import roc_shmem_b200 as shmem
    r = shmem.init("device", rank=0, world_size=1, heap_bytes=256 << 20)
    yield r
    shmem.finalize()


def _rand(*shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(BF)


def _reference(x, pre, post, scale, wg, wu, wd, eps):
    n = lambda v: v / (v.pow(2).mean(-1, keepdim=True) + eps).sqrt()  # noqa: E731
    h = n(x) * pre
    y = (torch.nn.functional.silu(h @ wg.t()) * (h @ wu.t())) @ wd.t()
    return x + scale * n(y) * post


def _near(got, ref, limit):
    assert (got.double() - ref).norm() <= limit * ref.norm(), float((got.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("M,F", [(512, 768), (2560, 1024)])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_residual_block_trains(rt, M, F, checkpoint):
    """Relative errors in the 2-norm.  A rounding to bf16 is within 2^-8 and uniform in its step, so below 2^-8 / sqrt(3) in the norm; a pass
    goes through about ten: under 2^-8 * 6.  One to 8 bits is within 2^-4, below 2^-4 / sqrt(3) = 0.036 in the norm; of what a gradient
    is made of, at most the norm's input, the norm's output and the pre-activations (which count twice, as factor and derivative) are kept
    so: under 0.036 * 4.  The scale's gradient is one sum of M * H terms of either sign, so it may be far smaller than they: with errors of
    the terms that are independent and below the limit in the norm, the sum is off by a normal number whose deviation is below the
    limit times the terms' 2-norm; four of those are exceeded once in 16000."""
    from roc_shmem_b200.models.llama import LlamaMLPModule
    from roc_shmem_b200.ops.moe import interleave_gate_up
    H = 512
    mod = LlamaMLPModule(rt, H, F, M, norms=True, checkpoint=checkpoint)
    wg, wu, wd = _rand(F, H, seed=1, scale=0.05), _rand(F, H, seed=2, scale=0.05), _rand(H, F, seed=3, scale=0.05)
    mod.block.load(wg, wu, wd)
    with torch.no_grad():
        mod.pre.copy_(1 + _rand(H, seed=4, scale=0.1))
        mod.post.copy_(1 + _rand(H, seed=5, scale=0.1))
        mod.scale.fill_(0.7)
    x, dy = _rand(M, H, seed=6), _rand(M, H, seed=7)
    other = _rand(M, H, seed=8)
    leaf = x.clone().requires_grad_(True)
    out = mod(leaf)
    if checkpoint:
        mod(other)                                            # another forward before the first one's backward
    params = (leaf, mod.pre, mod.post, mod.scale, mod.w13, mod.w2)
    got = torch.autograd.grad(out, params, dy)
    mod.block.check()
    ref = [t.detach().double().requires_grad_(True) for t in (x, mod.pre, mod.post, mod.scale, wg, wu, wd)]
    r = _reference(*ref, mod.eps)
    grads = torch.autograd.grad(r, ref, dy.double())
    expect = [*grads[:4], interleave_gate_up(grads[4], grads[5]), grads[6]]
    _near(out, r.detach(), 2.0 ** -8 * 6)
    limit = 2.0 ** -8 * 6 + (0.036 * 4 if checkpoint else 0)
    for g, e in zip(got[:3] + got[4:], expect[:3] + expect[4:]):
        _near(g, e, limit)
    terms = dy.double() * (r.detach() - x.double()) / 0.7
    assert (terms.sum() - expect[3]).abs() <= 1e-6 * terms.norm() and (got[3].double() - expect[3]).abs() <= 4 * limit * terms.norm()


def test_checkpointed_block_equals_its_own_recomputation(rt):
    """The backward from 8 bits is the unfused backward at exactly the kept values."""
    from roc_shmem_b200.models.llama import LlamaMLP
    M, H, F = 512, 512, 768
    block = LlamaMLP(rt, H, F, M)
    block.load(_rand(F, H, seed=1, scale=0.05), _rand(F, H, seed=2, scale=0.05), _rand(H, F, seed=3, scale=0.05))
    x, dy = _rand(M, H, seed=6), _rand(M, H, seed=7)
    block.forward(x)
    kept = block.keep()
    assert kept[0].nbytes + kept[1].nbytes < 0.52 * 2 * M * (H + 2 * F)
    block.forward(_rand(M, H, seed=9))
    dx, dw13, dw2 = block.backward(dy, kept).clone(), block.dw13.clone(), block.dw2.clone()
    block.check()
    xk, gu = kept[0].restore().double(), kept[1].restore().double().unflatten(1, (-1, 2, 32))
    g, u = gu[:, :, 0].flatten(1), gu[:, :, 1].flatten(1)
    dh = dy.double() @ block.w2.double()
    s = torch.sigmoid(g)
    dgu = torch.stack(((dh * u * s * (1 + g * (1 - s))).unflatten(1, (-1, 32)), (dh * g * s).unflatten(1, (-1, 32))), dim=2).flatten(1)
    for got, ref in ((dw2, dy.double().t() @ (g * s * u)), (dw13, dgu.t() @ xk), (dx, dgu @ block.w13.double())):
        _near(got, ref, 2.0 ** -8 * 3)                        # dh, dgu or the activations, and the result are rounded to bf16


@pytest.mark.parametrize("M,F", [(512, 768), (2560, 1024)])
def test_kept_backward_leaves_the_last_forward_alone(rt, M, F):
    """A (kept), B (not kept), A's backward, B's backward: B's gradients are those without A in between."""
    from roc_shmem_b200.models.llama import LlamaMLP
    H = 512
    block = LlamaMLP(rt, H, F, M)
    block.load(_rand(F, H, seed=1, scale=0.05), _rand(F, H, seed=2, scale=0.05), _rand(H, F, seed=3, scale=0.05))
    a, b, dy = (_rand(M, H, seed=s) for s in (4, 5, 6))
    block.forward(b)
    expect = [t.clone() for t in (block.backward(dy), block.dw13, block.dw2)]
    block.forward(a)
    kept = block.keep()
    block.forward(b)
    block.backward(dy, kept)
    got = (block.backward(dy), block.dw13, block.dw2)
    assert all(torch.equal(x, y) for x, y in zip(got, expect))
    block.check()


_FIRST_CALLS = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from roc_shmem_b200.ops.checkpoint8 import restore, store, swiglu_backward, swiglu_store
from roc_shmem_b200.ops.gemm_w4 import W4Tensor, linear_w4
from roc_shmem_b200.ops.norms import post_pre_norm
bf = torch.bfloat16
x = torch.randn(600, 1024, device="cuda").to(bf)
w = torch.ones(1024, device="cuda", dtype=bf)
leaves = [t.clone().requires_grad_(True) for t in (x, x, w, w)]
q = W4Tensor(torch.randint(0, 256, (512, 512), device="cuda", dtype=torch.uint8), torch.ones(512, 8, device="cuda", dtype=bf))
few = x[:3].clone()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, h = post_pre_norm(*leaves, checkpoint=True)
    grads = torch.autograd.grad((out, h), leaves, (x, x))
    y = linear_w4(few, q)
    act, kept = swiglu_store(x)
    dgu = swiglu_backward(kept, act)
    back = restore(store(x))
graph.replay()
torch.cuda.synchronize()
out2, h2 = post_pre_norm(*leaves, checkpoint=True)
grads2 = torch.autograd.grad((out2, h2), leaves, (x, x))
same = [torch.equal(a, b) for a, b in zip((out, h, *grads, y, dgu, back), (out2, h2, *grads2, linear_w4(few, q), swiglu_backward(swiglu_store(x)[1], act), restore(store(x))))]
print("same", all(same))
"""


def test_first_calls_inside_a_capture():
    """A program whose first use of each operator is recorded into a graph."""
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parent.parent)
    done = subprocess.run([sys.executable, "-c", _FIRST_CALLS, root], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same True" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("rows", [8, 1000])
def test_linear_with_kept_input(rows):
    from roc_shmem_b200.ops.checkpoint8 import restore, store
    from roc_shmem_b200.ops.torch_ops import Linear
    plain, kept = Linear(512, 264, device="cuda"), Linear(512, 264, device="cuda", checkpoint=True)
    kept.load_state_dict(plain.state_dict())
    x, dy = _rand(rows, 512, seed=1), _rand(rows, 264, seed=2)
    grads = []
    for layer in (plain, kept):
        leaf = x.clone().requires_grad_(True)
        y = layer(leaf)
        grads.append((y, *torch.autograd.grad(y, (leaf, layer.weight), dy)))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])
    assert torch.equal(grads[1][2], torch.ops.bshmem.linear_wgrad(dy, restore(store(x))))
    leaf = x.view(2, -1, 512).clone().requires_grad_(True)   # a frozen weight, more dimensions
    kept.weight.requires_grad_(False)
    g, = torch.autograd.grad(kept(leaf), leaf, dy.view(2, -1, 264))
    assert torch.equal(g.view(rows, 512), grads[0][1])
    with torch.no_grad():
        assert torch.equal(kept(x), plain(x))


def test_decode_step_in_a_graph():
    """norm, gate + up in 4 bits, SwiGLU, down in 4 bits, norm with residual and the next block's norm: captured once, replayed on new tokens."""
    from roc_shmem_b200.ops.checkpoint8 import swiglu
    from roc_shmem_b200.ops.gemm_w4 import linear_w4, quantize_w4, w4_error_site
    from roc_shmem_b200.ops.moe import interleave_gate_up
    from roc_shmem_b200.ops.norms import post_pre_norm, rms_norm
    H, F, T = 1024, 2048, 5
    wg, wu, wd = _rand(F, H, seed=1, scale=0.03), _rand(F, H, seed=2, scale=0.03), _rand(H, F, seed=3, scale=0.03)
    up, down = quantize_w4(interleave_gate_up(wg, wu), 64, zeros=True), quantize_w4(wd, 128)
    w = [1 + _rand(H, seed=s, scale=0.1) for s in (4, 5, 6)]
    x = _rand(T, H, seed=7)

    def step():
        h = rms_norm(x, w[0])
        y = linear_w4(swiglu(linear_w4(h, up)), down)
        return post_pre_norm(y, x, w[1], w[2], scale=0.5)
    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, h = step()
        for seed in (8, 9):
            x.copy_(_rand(T, H, seed=seed))
            graph.replay()
            eager = step()
            assert torch.equal(out, eager[0]) and torch.equal(h, eager[1])
    assert w4_error_site() == 0
    g = up.dequantize().double().unflatten(0, (-1, 2, 32))
    wg, wu = g[:, 0].flatten(0, 1), g[:, 1].flatten(0, 1)
    ref = _reference(x.double(), w[0].double(), w[1].double(), 0.5, wg, wu, down.dequantize().double(), 1e-6)
    _near(out, ref, 2.0 ** -8 * 6)
    _near(h, ref / (ref.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w[2].double(), 2.0 ** -8 * 7)


def test_modules():
    from roc_shmem_b200.ops.norms import RMSNorm, rms_norm
    norm = RMSNorm(264, device="cuda", checkpoint=True)
    x = _rand(7, 264, seed=1)
    assert torch.equal(norm(x), rms_norm(x, norm.weight))
    norm(x.requires_grad_(True)).float().sum().backward()
    assert norm.weight.grad.shape == (264,) and x.grad.shape == x.shape


def test_long_offsets():
    """Rows whose bytes lie beyond 2^32 of the tensor's beginning."""
    from roc_shmem_b200.ops.checkpoint8 import restore, store
    from roc_shmem_b200.ops.norms import rms_norm
    rows, n = 140000, 16384                                   # 4.6 GB
    x = torch.zeros(rows, n, dtype=BF, device="cuda")
    last = _rand(3, n, seed=1)
    x[-3:] = last
    w = 1 + _rand(n, seed=2, scale=0.1)
    h = rms_norm(x, w)
    assert torch.equal(h[-3:], rms_norm(last, w)) and not h[:-3].any()
    del h
    assert torch.equal(restore(store(x))[-3:], restore(store(last)))


def test_two_streams_at_once():
    """4-bit products, the bf16 GEMM and norms of two streams in each other's way: what takes whole multiprocessors waits, nothing else changes."""
    from roc_shmem_b200.ops.gemm import gemm_bf16, gemm_error_site
    from roc_shmem_b200.ops.gemm_w4 import linear_w4, quantize_w4, w4_error_site
    from roc_shmem_b200.ops.norms import post_pre_norm
    a, b = quantize_w4(_rand(2048, 4096, seed=1), 128), quantize_w4(_rand(4104, 2048, seed=2), 32, zeros=True)
    x, y, w = _rand(3, 4096, seed=3), _rand(40, 2048, seed=4), _rand(512, 2048, seed=5)
    r, one = _rand(300, 2048, seed=6), torch.ones(2048, dtype=BF, device="cuda")
    jobs = [lambda: linear_w4(x, a), lambda: linear_w4(y, b), lambda: gemm_bf16(y, w), lambda: post_pre_norm(r, r, one, one)[1]]
    expect = [j() for j in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(60):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                k = (i + 2 * s) % 4
                got.append((k, jobs[k]()))
    torch.cuda.synchronize()
    assert all(torch.equal(v, expect[k]) for k, v in got) and w4_error_site() == 0 and gemm_error_site() == 0


def test_extreme_shapes():
    """One column and a million rows; a million columns of a few 4-bit rows; many rows of few columns."""
    from block_reference import close
    from roc_shmem_b200.ops.gemm_w4 import W4Tensor, linear_w4
    from roc_shmem_b200.ops.norms import rms_norm
    x = _rand(1000003, 1, seed=1).requires_grad_(True)
    w = torch.full((1,), 0.5, dtype=torch.float32, device="cuda", requires_grad=True)
    h = rms_norm(x, w, 1e-3)
    d = x.detach().double()
    n = d / (d * d + 1e-3).sqrt()
    close(h, n * 0.5, (n * 0.5).abs())
    gw, = torch.autograd.grad(h, w, torch.ones_like(h))
    close(gw, n.sum().view(1), n.abs().sum().view(1), 64 + 1000003 // 4)
    K = 1 << 20
    q = torch.randint(0, 256, (24, K // 2), device="cuda", dtype=torch.uint8, generator=torch.Generator(device="cuda").manual_seed(2))
    t = W4Tensor(q, torch.full((24, K // 128), 0.01, dtype=BF, device="cuda"))
    v = _rand(3, K, seed=3)
    m = ((torch.stack((q & 15, q >> 4), 2).flatten(1).double() - 8) * t.scales[0, 0].double())
    close(linear_w4(v, t), v.double() @ m.t(), v.double().abs() @ m.abs().t(), 2 * (K // 16 + 16))
    tall = W4Tensor(q.view(-1, 32)[:100003].contiguous(), torch.full((100003, 1), 0.01, dtype=BF, device="cuda"))
    u = _rand(2, 64, seed=4)
    m = ((torch.stack((tall.q & 15, tall.q >> 4), 2).flatten(1).double() - 8) * tall.scales[0, 0].double())
    close(linear_w4(u, tall), u.double() @ m.t(), u.double().abs() @ m.abs().t(), 2 * (64 // 16 + 16))


def test_kept_of_another_block_is_refused(rt):
    from roc_shmem_b200.models.llama import LlamaMLP
    M, H = 512, 512
    one, other = LlamaMLP(rt, H, 768, M), LlamaMLP(rt, H, 1024, M)
    x = _rand(M, H, seed=1)
    one.forward(x), other.forward(x)
    a, b = one.keep(), other.keep()
    for kept in (b, (a[0], b[1]), (a[1], a[0])):
        with pytest.raises(ValueError, match="forward"):
            one.backward(x, kept)


def test_no_gradient_nothing_kept(rt, monkeypatch):
    from roc_shmem_b200.models.llama import LlamaMLPModule
    mod = LlamaMLPModule(rt, 512, 768, 512, norms=True, checkpoint=True)
    mod.block.load(_rand(768, 512, seed=1, scale=0.05), _rand(768, 512, seed=2, scale=0.05), _rand(512, 768, seed=3, scale=0.05))
    x = _rand(512, 512, seed=4)
    expect = mod(x).detach()
    monkeypatch.setattr(mod.block, "keep", lambda: pytest.fail("kept without a gradient"))
    with torch.no_grad():
        assert torch.equal(mod(x), expect)


def test_two_threads_at_once():
    """Widths whose kernels are the same but for their shared memory, from two threads: what one asks for does not become the other's."""
    import threading
    from roc_shmem_b200.ops.norms import post_pre_norm
    inputs = [torch.randn(rows, n, device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(BF) for rows, n in ((1300, 4096), (700, 8192))]
    weights = [torch.ones(x.shape[1], dtype=BF, device="cuda") for x in inputs]
    expect = [post_pre_norm(x, x, w, w)[1] for x, w in zip(inputs, weights)]
    torch.cuda.synchronize()
    start, failed = threading.Barrier(2), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(3000):
                    got = post_pre_norm(inputs[i], inputs[i], weights[i], weights[i])[1]
                assert torch.equal(got, expect[i])
        except Exception as e:
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
