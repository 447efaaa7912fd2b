"""Norms that somebody traces, compiles, transforms or watches give what the plain calls give, and refuse what they do not have."""
import pytest
import torch

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
    from torch.utils._python_dispatch import TorchDispatchMode
    leaves = [t.requires_grad_(True) for t in _operands()]
    used = [t for t, unused in zip(leaves, (form == "pre", False, False, form == "pre")) if not unused]
    dys = [_rand(6, 40, 264, seed=20 + i) for i in range(2 if form == "post_pre" else 1)]
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    def forward():
        return _step(*leaves, checkpoint, form)
    outs = forward()
    expect = (*[o.detach() for o in outs], *torch.autograd.grad(outs, used, dys))

    def same(outs, grads):
        assert all(torch.equal(a, b) for a, b in zip((*outs, *grads), expect))
    with Watch():
        outs = forward()
        same(outs, torch.autograd.grad(outs, used, dys))
    assert "bshmem.norm.default" in seen and "bshmem.norm_backward.default" in seen
    outs = forward()
    seen.clear()
    with Watch():
        same(outs, torch.autograd.grad(outs, used, dys))
    compiled = torch.compile(lambda *t: _step(*t, checkpoint, form), backend="aot_eager", fullgraph=True)
    outs = compiled(*leaves)
    same(outs, torch.autograd.grad(outs, used, dys))
    outs = forward()
    batched = torch.autograd.grad(outs, used, [torch.stack([d, 2 * d]) for d in dys], is_grads_batched=True)
    same(outs, [b[0] for b in batched])


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
