"""Norms, 8-bit activations and 4-bit products that somebody traces, compiles, transforms or watches give what the plain calls give, and refuse what they do not have."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from roc_shmem_b200.ops import torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _rand(*shape, seed, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _operands(seed=0):
    return _rand(6, 40, 264, seed=seed), _rand(6, 40, 264, seed=seed + 1), _rand(264, seed=seed + 2), _rand(6, 40, 1, seed=seed + 3)


def _step(y, x, w, g, checkpoint=False, form="post_pre"):
    from roc_shmem_b200.ops.norms import post_norm, post_pre_norm, rms_norm
    if form == "pre":
        return rms_norm(x, w, checkpoint=checkpoint),
    if form == "post":
        return post_norm(y, x, w, gate=g, scale=0.75, checkpoint=checkpoint),
    return post_pre_norm(y, x, w, w, gate=g, scale=0.75, checkpoint=checkpoint)


FORMS = ["pre", "post", "post_pre"]


class Watch(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("form", FORMS)
def test_traced_norms(form):
    from torch.fx.experimental.proxy_tensor import make_fx
    first, other = _operands(), _operands(10)
    f = lambda *t: _step(*t, form=form)  # noqa: E731
    expect = f(*other)
    for traced in (make_fx(f)(*first), torch.jit.trace(f, first)):
        got = traced(*other)
        got = got if isinstance(got, tuple) else (got,)
        assert len(got) == len(expect) and all(torch.equal(a, b) for a, b in zip(got, expect))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("checkpoint", [False, True])
def test_watched_training_equals_plain_training(form, checkpoint):
    """Under a mode, compiled without a code generator, and a plain forward pass with a watched backward pass."""
    leaves = [t.requires_grad_(True) for t in _operands()]
    used = [t for t, unused in zip(leaves, (form == "pre", False, False, form == "pre")) if not unused]
    dys = [_rand(6, 40, 264, seed=20 + i) for i in range(2 if form == "post_pre" else 1)]
    def forward():
        return _step(*leaves, checkpoint, form)
    outs = forward()
    expect = (*[o.detach() for o in outs], *torch.autograd.grad(outs, used, dys))

    def same(outs, grads):
        assert all(torch.equal(a, b) for a, b in zip((*outs, *grads), expect))
    with Watch() as watch:
        outs = forward()
        same(outs, torch.autograd.grad(outs, used, dys))
    assert "bshmem.norm.default" in watch.seen and "bshmem.norm_backward.default" in watch.seen
    outs = forward()
    with Watch() as watch:
        same(outs, torch.autograd.grad(outs, used, dys))
    assert "bshmem.norm_backward.default" in watch.seen
    compiled = torch.compile(lambda *t: _step(*t, checkpoint, form), backend="aot_eager", fullgraph=True)
    outs = compiled(*leaves)
    same(outs, torch.autograd.grad(outs, used, dys))
    outs = forward()
    batched = torch.autograd.grad(outs, used, [torch.stack([d, 2 * d]) for d in dys], is_grads_batched=True)
    same(outs, [b[0] for b in batched])


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("used", [0, 1])
def test_one_result_of_a_watched_call_unused(checkpoint, used):
    leaves = [t.requires_grad_(True) for t in _operands()]
    dy = _rand(6, 40, 264, seed=20)

    def gradients(f):
        return torch.autograd.grad(f(*leaves)[used], leaves, dy)
    f = lambda *t: _step(*t, checkpoint)  # noqa: E731
    expect = gradients(f)
    with Watch():
        got = gradients(f)
    assert all(torch.equal(a, b) for a, b in zip(got, expect)) and dy.data_ptr() != got[0].data_ptr()
    out = f(*leaves)[used]
    with Watch():
        got = torch.autograd.grad(out, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    got = gradients(torch.compile(f, backend="aot_eager", fullgraph=True))
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    y, x, w, g = [t.detach() for t in leaves]
    _, _, rstd, kept = torch.ops.bshmem.norm(y, x, w, w, g, None, 0.75, 1e-6, 2, True)
    before = dy.clone()
    found = torch.ops.bshmem.norm_backward(dy, None, w, w, g, None, rstd, kept, None, 0.75, 2, True, 0b11111)      # the operator itself
    assert found[1].data_ptr() != dy.data_ptr() and torch.equal(found[1], dy) and torch.equal(dy, before) and not found[3].any()


def test_compiled_for_any_number_of_rows():
    from roc_shmem_b200.ops.norms import RMSNorm
    norm = RMSNorm(264, device="cuda")
    compiled = torch.compile(norm, backend="aot_eager", fullgraph=True, dynamic=True)
    for rows in (7, 40, 41):
        x, dy = _rand(rows, 264, seed=rows).requires_grad_(True), _rand(rows, 264, seed=99)
        a, b = (torch.autograd.grad(f(x), (x, norm.weight), dy) for f in (norm, compiled))
        assert torch.equal(compiled(x), norm(x)) and all(torch.equal(u, v) for u, v in zip(a, b))


def test_fake_norms():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        leaves = [mode.from_tensor(t).requires_grad_(True) for t in _operands()]
        for form in FORMS:
            for checkpoint in (False, True):
                outs = _step(*leaves, checkpoint, form)
                assert all(o.shape == (6, 40, 264) and o.dtype is BF for o in outs)
                dx, = torch.autograd.grad(outs, leaves[1], [torch.empty_like(o) for o in outs])
                assert dx.shape == (6, 40, 264)


def test_batched_and_dual_norms():
    from torch.autograd import forward_ad

    from roc_shmem_b200.ops.norms import rms_norm
    y, x, w, g = _operands()
    assert torch.equal(torch.func.vmap(lambda v: rms_norm(v, w))(x), rms_norm(x, w))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        rms_norm(forward_ad.make_dual(x, y), w)
    leaf = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(torch.ops.bshmem.norm(None, leaf, None, w, None, None, 1.0, 1e-6, 0, False)[1], leaf, y, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.float().sum(), leaf)


def test_watched_eight_bits():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    from roc_shmem_b200.ops.checkpoint8 import restore, store, swiglu, swiglu_backward, swiglu_store
    x, gu, d = _rand(40, 200, seed=1), _rand(40, 192, seed=2), _rand(40, 96, seed=3)
    there = lambda t: restore(store(t))  # noqa: E731

    def both(t, e):
        act, kept = swiglu_store(t)
        return (act, *swiglu_backward(kept, e, act=True))
    expect, pair = there(x), both(gu, d)
    for traced in (make_fx(there)(torch.zeros_like(x)), torch.jit.trace(there, (torch.zeros_like(x),)),
                   torch.compile(there, backend="aot_eager", fullgraph=True)):
        assert torch.equal(traced(x), expect)
    for traced in (make_fx(both)(torch.zeros_like(gu), d), torch.compile(both, backend="aot_eager", fullgraph=True)):
        assert all(torch.equal(a, b) for a, b in zip(traced(gu, d), pair))
    assert torch.equal(torch.func.vmap(there)(x.view(5, 8, 200)).view(40, 200), expect)
    leaf = gu.clone().requires_grad_(True)
    grad, = torch.autograd.grad(swiglu(leaf), leaf, d)
    assert torch.equal(grad, pair[1])
    compiled = torch.compile(swiglu, backend="aot_eager", fullgraph=True)
    assert torch.equal(torch.autograd.grad(compiled(leaf), leaf, d)[0], grad)
    act = swiglu(leaf)
    with Watch():
        assert torch.equal(torch.autograd.grad(act, leaf, d, retain_graph=True)[0], grad)
        assert torch.equal(swiglu(gu), pair[0]) and torch.equal(restore(store(x), out=torch.empty_like(x)), expect)
    assert torch.equal(torch.autograd.grad(act, leaf, torch.stack([d, d]), is_grads_batched=True)[0][1], grad)
    with FakeTensorMode() as mode:
        f = mode.from_tensor(gu).requires_grad_(True)
        assert torch.autograd.grad(swiglu(f), f, mode.from_tensor(d))[0].shape == gu.shape


def test_watched_backward_of_a_linear_layer_with_kept_input():
    from roc_shmem_b200.ops.torch_ops import Linear
    layer = Linear(200, 264, device="cuda", checkpoint=True)
    x, dy = _rand(40, 200, seed=1).requires_grad_(True), _rand(40, 264, seed=2)
    y = layer(x)
    expect = torch.autograd.grad(y, (x, layer.weight), dy, retain_graph=True)
    with Watch():
        got = torch.autograd.grad(y, (x, layer.weight), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    got = torch.autograd.grad(y, (x, layer.weight), torch.stack([dy, dy]), is_grads_batched=True)
    assert all(torch.equal(a[1], b) for a, b in zip(got, expect))


@pytest.mark.parametrize("zeros", [False, True])
def test_watched_four_bits(zeros):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    from roc_shmem_b200.ops.gemm_w4 import LinearW4, W4Tensor, linear_w4, quantize_w4, widen_w4
    w = _rand(264, 512, seed=1)
    t = quantize_w4(w, 64, zeros=zeros)
    layer = LinearW4(t)
    for rows in (5, 200):                                     # the 4-bit kernel and the bf16 GEMM
        x, other = _rand(rows, 512, seed=2), _rand(rows, 512, seed=3)
        expect = linear_w4(x, t)
        for traced in (make_fx(lambda v: linear_w4(v, t))(other), torch.jit.trace(lambda v: linear_w4(v, t), (other,)),
                       torch.compile(layer, backend="aot_eager", fullgraph=True)):
            assert torch.equal(traced(x), expect)
    assert torch.equal(torch.func.vmap(layer)(x.view(5, -1, 512)).view(rows, 264)[:40], linear_w4(x[:40], t))      # of 40 tokens each
    with Watch() as watch:
        again = quantize_w4(w, 64, zeros=zeros)
        wide = widen_w4(again)
    assert torch.equal(again.q, t.q) and torch.equal(again.scales, t.scales) and (not zeros or torch.equal(again.zeros, t.zeros))
    assert torch.equal(wide, widen_w4(t)) and {"bshmem.quantize_w4.default", "bshmem.widen_w4.default"} <= set(watch.seen)
    with FakeTensorMode() as mode:
        f = W4Tensor(*[None if v is None else mode.from_tensor(v) for v in (t.q, t.scales, t.zeros)])
        assert linear_w4(mode.from_tensor(x), f).shape == (200, 264) and widen_w4(f).shape == (264, 512)
        assert LinearW4(quantize_w4(mode.from_tensor(w), 64, zeros=zeros))(mode.from_tensor(x)).shape == (200, 264)


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_norm_operators_keep_torchs_rules(mode, checkpoint):
    """Schema, fake results and gradients, with fixed and with any sizes."""
    y, x, w, g = _operands()
    op, back = torch.ops.bshmem.norm, torch.ops.bshmem.norm_backward
    for grad in (False, True):
        leaf = [t.clone().requires_grad_(grad) for t in (y, x, w, w, g)]
        operands = (leaf[0] if mode else None, leaf[1], leaf[2] if mode else None, leaf[3] if mode != 1 else None, leaf[4] if mode else None, None)
        torch.library.opcheck(op, (*operands, 0.75, 1e-6, mode, checkpoint))
    plain = [None if t is None else t.detach() for t in operands]
    out, _, rstd, kept = op(*plain, 0.75, 1e-6, mode, checkpoint)
    saved = (kept, None) if checkpoint else (plain[0], (x, None, out)[mode])
    need = (0b001010, 0b010101, 0b011111)[mode]
    torch.library.opcheck(back, (y if mode else None, x if mode != 1 else None, *plain[2:], rstd, *saved, 0.75, mode, checkpoint, need))


def test_other_operators_keep_torchs_rules():
    ops = torch.ops.bshmem
    x, gu, d, w = _rand(40, 200, seed=1), _rand(40, 192, seed=2), _rand(40, 96, seed=3), _rand(264, 512, seed=4)
    torch.library.opcheck(ops.store8, (x,))
    torch.library.opcheck(ops.restore8, (ops.store8(x), 200, torch.float32))
    torch.library.opcheck(ops.swiglu8, (gu, False))
    torch.library.opcheck(ops.swiglu8, (gu.clone().requires_grad_(True), True))
    for act in (False, True):
        torch.library.opcheck(ops.swiglu8_backward, (ops.swiglu8(gu, True)[1], d, act))
    for zeros in (False, True):
        torch.library.opcheck(ops.quantize_w4, (w, 64, zeros))
        q, s, z = ops.quantize_w4(w, 64, zeros)
        torch.library.opcheck(ops.widen_w4, (q, s, z if zeros else None))
        for tokens in (5, 200):
            torch.library.opcheck(ops.linear_w4, (_rand(tokens, 512, seed=5), q, s, z if zeros else None))
