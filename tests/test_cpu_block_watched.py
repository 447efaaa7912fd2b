"""Norms, 8-bit activations and 4-bit products on anything but plain tensors that nobody watches: fake tensors, tracing, transforms, modes that see operators and
forward-mode derivatives, with the formulas in the kernels' place.  Nothing there may reach a native entry, which would read addresses that
are not there."""
from types import SimpleNamespace

import numpy
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

from roc_shmem_b200.ops import checkpoint8, gemm_w4, norms, torch_ops  # noqa: F401

BF, F32 = torch.bfloat16, torch.float32


def _native(*_):
    pytest.fail("a native entry was reached")


@pytest.fixture(autouse=True)
def no_native(monkeypatch):
    for entry in ("_fwd", "_bwd", "_groups", "_finish"):
        monkeypatch.setattr(norms, entry, _native)
    for entry in ("_store", "_restore", "_swiglu_store", "_swiglu_backward"):
        monkeypatch.setattr(checkpoint8, entry, _native)
    for entry in ("_few", "_widen", "_lib", "gemm_bf16"):
        monkeypatch.setattr(gemm_w4, entry, _native)


def _n(v, eps):
    return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + eps)


@pytest.fixture
def formulas(monkeypatch):
    """The operators' own bodies on the CPU; the gradients are the norm's before a block."""
    def forward(y, x, w1, w2, gate, scale, number, eps, mode, checkpoint):
        one = lambda t: 1.0 if t is None else t  # noqa: E731
        out = h = None
        z = x
        if mode != norms.PRE:
            out = z = x + (number if scale is None else scale) * one(gate) * one(w1) * _n(y, eps)
        if mode != norms.POST:
            h = one(w2) * _n(z, eps)
        return tuple(x.new_empty(0) if t is None else t for t in (out, h, x.new_full((1,), eps), None))

    def backward(dout, dh, w1, w2, gate, scale, rstd, a, b, number, mode, checkpoint, need):
        assert mode == norms.PRE
        r = torch.rsqrt(b.pow(2).mean(-1, keepdim=True) + rstd[0])
        n, t = b * r, dh * w2
        found = (None, r * (t - n * (t * n).mean(-1, keepdim=True)), None, (dh * n).sum(0), None, None)
        return tuple(f if n else dh.new_empty(0) for f, n in zip(found, norms._asked(need)))
    monkeypatch.setattr(norms, "operator_forward", forward)
    monkeypatch.setattr(norms, "operator_backward", backward)


def _fakes(*shapes, dtype=BF):
    return [torch.empty(s, dtype=dtype, device="cuda") for s in shapes]


@pytest.mark.parametrize("checkpoint", [False, True])
def test_fake_norms_launch_nothing(checkpoint):
    with FakeTensorMode():
        x, y, w, g = _fakes((4, 6, 72), (4, 6, 72), (72,), (4, 6, 1))
        h = norms.rms_norm(x, w, checkpoint=checkpoint)
        out = norms.post_norm(y, x, w, gate=g, scale=0.5)
        both = norms.post_pre_norm(y, x, w, w, checkpoint=checkpoint)
        assert all(t.shape == x.shape and t.dtype is BF and t.device.type == "cuda" for t in (h, out, *both))
        s = torch.ones(1, device="cuda")                         # the backward pass as autograd calls it (its engine asks for a GPU)
        for mode, grads, need in ((norms.POST_PRE, (x, y), [True] * 6), (norms.POST_PRE, (x, None), [True] * 6),
                                  (norms.POST, (x, None), [True, True, True, False, True, True]), (norms.PRE, (None, y), [False, True, False, True, False, False])):
            operands = (y if mode != norms.PRE else None, x, w if mode != norms.PRE else None, w if mode != norms.POST else None,
                        g if mode != norms.PRE else None, s if mode != norms.PRE else None)
            _, _, rstd, kept = torch.ops.bshmem.norm(*operands, 1.0, 1e-6, mode, checkpoint)
            saved = (*operands[2:], rstd, *((kept, None) if checkpoint else (operands[0], x if mode != norms.POST else None)))
            found = norms._registered_gradients(mode, checkpoint, 1.0, need, saved, *grads)
            assert [None if t is None else t.shape for t in found] == [t.shape if n else None for t, n in zip(operands, need)]
        for bad in (lambda: norms.rms_norm(x, w[:71]), lambda: norms.post_norm(y[:3], x), lambda: norms.rms_norm(x, w.double()), lambda: norms.rms_norm(x, eps=0.0)):
            with pytest.raises(ValueError):
                bad()


def _close(a, b):
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_norms_are_traced(formulas):
    from torch.fx.experimental.proxy_tensor import make_fx
    x, y, w = torch.randn(5, 8), torch.randn(5, 8), torch.randn(8)
    cases = (lambda a, b: norms.rms_norm(a, w), lambda a, b: norms.post_norm(b, a, w, scale=0.5), lambda a, b: norms.post_pre_norm(b, a, w, w)[1])
    expect = (w * _n(x, 1e-6), x + 0.5 * w * _n(y, 1e-6), w * _n(x + w * _n(y, 1e-6), 1e-6))
    for f, e in zip(cases, expect):
        for traced in (make_fx(f)(torch.zeros(5, 8), torch.zeros(5, 8)), torch.jit.trace(f, (torch.zeros(5, 8), torch.zeros(5, 8)), check_trace=False)):
            assert "bshmem" in str(traced.graph) and "norm" in str(traced.graph)
            _close(traced(x, y), e)


def test_norms_with_gradients_are_traced(formulas):
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(a, b):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        return torch.autograd.grad(norms.rms_norm(a, b), (a, b), torch.ones_like(a))
    x, w = torch.randn(5, 8), torch.randn(8)
    graph = make_fx(step)(torch.zeros(5, 8), torch.zeros(8))
    assert "norm_backward" in str(graph.graph)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    for got, e in zip(graph(x, w), torch.autograd.grad(b * _n(a, 1e-6), (a, b), torch.ones_like(a))):
        _close(got, e)


def test_nothing_is_kept_without_a_gradient(formulas, monkeypatch):
    asked, body = [], norms.operator_forward
    monkeypatch.setattr(norms, "operator_forward", lambda *a: (asked.append(a[-1]), body(*a))[1])

    class Other(torch.Tensor):
        pass
    x, w = torch.randn(5, 8).as_subclass(Other), torch.randn(8, requires_grad=True)
    norms.rms_norm(x, w, checkpoint=True)
    norms.rms_norm(x, w)
    norms.rms_norm(x, w.detach(), checkpoint=True)
    with torch.no_grad():
        norms.rms_norm(x, w, checkpoint=True)
    assert asked == [True, False, False, False]


def test_transforms_and_modes(formulas):
    from torch.utils._python_dispatch import TorchDispatchMode
    x, w = torch.randn(3, 5, 8), torch.randn(8)
    e = w * _n(x, 1e-6)
    _close(torch.func.vmap(lambda v: norms.rms_norm(v, w))(x), e)
    with pytest.raises(RuntimeError, match="functorch"):      # torch's own refusal of a registered operator's gradient there
        torch.func.grad(lambda v: norms.rms_norm(v, w).pow(2).sum())(x)
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    with Watch():
        _close(norms.rms_norm(x, w), e)
    assert "bshmem.norm.default" in seen


def test_no_forward_mode_derivative():
    """A tangent is refused, not dropped; tensors without one pass on to the usual checks."""
    x, w = torch.randn(5, 8), torch.randn(8)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        g = forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: norms.rms_norm(d, w), lambda: norms.rms_norm(x, g), lambda: norms.post_norm(d, x), lambda: norms.post_norm(x, x, gate=d),
                     lambda: norms.post_pre_norm(x, x, scale=forward_ad.make_dual(w[:1], w[:1]))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="CUDA"):
            norms.rms_norm(x, w)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: norms.rms_norm(v, w), (x,), (x,))


def test_when_a_call_is_direct():
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    from roc_shmem_b200.ops.watched import direct

    class Other(torch.Tensor):
        pass
    x, p = torch.zeros(3), torch.nn.Parameter(torch.zeros(3))
    assert direct("it", x, p, None, 0.5, 1) and direct("it")
    assert not direct("it", x.as_subclass(Other)) and not direct("it", x, None, torch.empty(3, device="meta").as_subclass(Other))
    assert direct("it", x, True, numpy.float64(0.5))         # numbers of any kind
    with torch.device("cpu"):                                # a default device is no observer
        assert direct("it", x)
    with forward_ad.dual_level():                            # nor is a level that none of the operands is of
        assert direct("it", x, None, 0.5)
    for mode in (TorchFunctionMode, TorchDispatchMode):
        with mode():
            assert not direct("it", x)
    inside = []
    for f in (torch.func.vmap, torch.func.functionalize):
        f(lambda v: (inside.append(direct("it", v)), v)[1])(torch.zeros(2))
    torch.jit.trace(lambda v: (inside.append(direct("it", v)), v)[1], (x,), check_trace=False)
    assert inside == [False] * 3 and direct("it", x)


def _graph(monkeypatch, x, w):
    """A result of the direct call whose backward pass is still to come, with the formula in the kernel's place."""
    def forward(c, mode, train):
        return None, w.detach() * _n(x.detach(), 1e-6), torch.full((1,), 1e-6), None
    monkeypatch.setattr(norms, "_forward", forward)
    return norms._NormFn.apply(None, x, None, w, None, None, SimpleNamespace(what=2, n=8, rows=5, kind=norms.NO_GATE, number=1.0), norms.PRE)


def test_watched_backward_of_a_direct_call(formulas, monkeypatch):
    """The forward pass went past the dispatcher, the backward pass is batched, fake or of dual numbers."""
    x, w = torch.randn(5, 8, requires_grad=True), torch.randn(8, requires_grad=True)
    h = _graph(monkeypatch, x, w)
    d = torch.randn(3, 5, 8)
    got = torch.autograd.grad(h, (x, w), d, is_grads_batched=True, retain_graph=True)
    e = [torch.autograd.grad(w * _n(x, 1e-6), (x, w), v) for v in d]
    _close(got[0], torch.stack([v[0] for v in e]))
    _close(got[1], torch.stack([v[1] for v in e]))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.autograd.grad(h, x, forward_ad.make_dual(d[0], d[1]), retain_graph=True)


def test_operators_refuse_what_does_not_belong_together():
    with FakeTensorMode():
        x, w = _fakes((4, 8), (8,))
        r, two = torch.empty(1, 4, device="cuda"), torch.empty(2, 4, device="cuda")
        op, back = torch.ops.bshmem.norm, torch.ops.bshmem.norm_backward
        need = 2
        assert back(None, x, None, w, None, None, r, None, x, 1.0, norms.PRE, False, need)[1].shape == x.shape
        for bad in (lambda: op(None, x, None, w, None, None, 1.0, 1e-6, 3, False), lambda: op(x, x, None, w, None, None, 1.0, 1e-6, norms.PRE, False),
                    lambda: op(None, x, None, w, None, None, 1.0, 1e-6, norms.POST, False), lambda: op(None, x, w, w, None, None, 1.0, 1e-6, norms.PRE, False),
                    lambda: back(None, x, None, w, None, None, two, None, x, 1.0, norms.PRE, False, need),
                    lambda: back(None, x, None, w, None, None, r, None, x[:3], 1.0, norms.PRE, False, need),
                    lambda: back(None, x, None, w, None, None, r, x, None, 1.0, norms.PRE, True, need),
                    lambda: back(x, x, None, w, None, None, r, None, x, 1.0, norms.PRE, False, need),
                    lambda: back(None, None, None, w, None, None, r, None, x, 1.0, norms.PRE, False, need),
                    lambda: back(None, x, None, None, None, None, r, None, x, 1.0, norms.PRE, False, 2 | 8)):
            with pytest.raises(ValueError):
                bad()


def test_fake_eight_bits_launch_nothing():
    from roc_shmem_b200.ops.checkpoint8 import kept_bytes, restore, store, swiglu, swiglu_backward, swiglu_store
    with FakeTensorMode():
        x, gu, d = _fakes((3, 5, 200), (3, 5, 192), (3, 5, 96))
        kept = store(x)
        assert kept.data.shape == (kept_bytes(15, 200),) and kept.shape == x.shape and kept.dtype is BF
        assert restore(kept).shape == x.shape and restore(kept, F32).dtype is F32 and kept.restore().dtype is BF
        out = torch.empty(15, 300, device="cuda")[:, 4:204]
        assert restore(kept, out=out) is out
        act, kept = swiglu_store(gu)
        assert act.shape == d.shape and kept.data.shape == (kept_bytes(15, 192),)
        dgu, again = swiglu_backward(kept, d, act=True)
        assert dgu.shape == gu.shape and again.shape == d.shape and swiglu_backward(kept, d, dgu_out=gu) is gu
        assert swiglu_backward(kept, d, act_out=d)[1] is d
        assert swiglu(gu).shape == d.shape and swiglu(gu.requires_grad_(True)).requires_grad
        for bad in (lambda: store(x.double()), lambda: restore(kept, torch.float64), lambda: restore(store(x), out=x), lambda: swiglu(x),
                    lambda: swiglu_backward(kept, d[:2]), lambda: swiglu_backward(kept, d, dgu_out=d)):
            with pytest.raises(ValueError):
                bad()


def test_eight_bits_are_traced(monkeypatch):
    from torch.fx.experimental.proxy_tensor import make_fx

    from roc_shmem_b200.ops.checkpoint8 import Checkpoint8, restore, store, swiglu
    monkeypatch.setattr(checkpoint8, "store_direct", lambda x: x.clone().view(torch.uint8).flatten())
    monkeypatch.setattr(checkpoint8, "operator_restore", lambda data, cols, dtype: data.clone().view(F32).view(-1, cols))
    monkeypatch.setattr(checkpoint8, "_held", lambda kept, *_: (kept.data, kept.shape[:-1].numel(), kept.shape[-1]))
    monkeypatch.setattr(checkpoint8, "operator_swiglu", lambda gu, keep: ((torch.sigmoid(gu) * gu)[:, 32:], gu.new_empty((0,), dtype=torch.uint8)))
    x, gu = torch.randn(5, 8), torch.randn(5, 64)
    for f, v, names in ((lambda t: restore(store(t)), x, ("store8", "restore8")), (swiglu, gu, ("swiglu8",))):
        for traced in (make_fx(f)(torch.zeros_like(v)), torch.jit.trace(f, (torch.zeros_like(v),), check_trace=False)):
            assert all(n in str(traced.graph) for n in names)
            _close(traced(v), v if f is not swiglu else (torch.sigmoid(v) * v)[:, 32:])
    kept = Checkpoint8(x.view(torch.uint8).flatten(), x.shape, F32)
    with forward_ad.dual_level():
        d, g = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, gu))
        for call in (lambda: store(d), lambda: swiglu(g), lambda: checkpoint8.swiglu_store(g), lambda: checkpoint8.swiglu_backward(kept, d), lambda: restore(kept, out=d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_watched_backward_of_kept_activations(monkeypatch):
    """A plain forward pass whose backward pass is batched."""
    from roc_shmem_b200.ops import torch_ops
    gu, d = torch.randn(5, 64, dtype=torch.float32).to(BF), torch.randn(3, 5, 32).to(BF)
    monkeypatch.setattr(checkpoint8, "_swiglu_forward", lambda gu, keep: (gu[:, 32:].clone(), gu.view(torch.uint8).flatten().clone()))
    monkeypatch.setattr(checkpoint8, "operator_swiglu_backward",
                        lambda data, dact, act: (data.view(BF).view(-1, 64) * dact.repeat(1, 2), dact.new_empty(0)))
    leaf = gu.clone().requires_grad_(True)
    got, = torch.autograd.grad(checkpoint8._SwigluFn.apply(leaf), leaf, d, is_grads_batched=True)
    assert torch.equal(got, gu * d.repeat(1, 1, 2))

    def product(a, b, out=None, *, a_mn=False, b_mn=False):
        return ((a.t() if a_mn else a).float() @ (b if b_mn else b.t()).float()).to(BF)
    monkeypatch.setattr(torch_ops, "gemm_bf16", product)
    monkeypatch.setattr(checkpoint8, "store_direct", lambda x: x.detach().clone().view(torch.uint8).flatten())
    monkeypatch.setattr(checkpoint8, "operator_restore", lambda data, cols, dtype: data.clone().view(BF).view(-1, cols))
    x, w, dy = torch.randn(5, 16).to(BF).requires_grad_(True), torch.randn(8, 16).to(BF).requires_grad_(True), torch.randn(3, 5, 8).to(BF)
    dx, dw = torch.autograd.grad(torch_ops._LinearKeptFn.apply(x, w), (x, w), dy, is_grads_batched=True)
    for i in range(3):
        assert torch.equal(dx[i], product(dy[i], w, b_mn=True)) and torch.equal(dw[i], product(dy[i], x, a_mn=True, b_mn=True))


@pytest.mark.parametrize("zeros", [False, True])
def test_fake_four_bits_launch_nothing(zeros):
    from roc_shmem_b200.ops.gemm_w4 import LinearW4, linear_w4, quantize_w4, widen_w4
    with FakeTensorMode():
        w, x = _fakes((24, 256), (3, 5, 256))
        t = quantize_w4(w, 64, zeros=zeros)
        assert t.q.shape == (24, 128) and t.scales.shape == (24, 4) and t.scales.dtype is BF and t.group == 64
        assert t.zeros is None if not zeros else t.zeros.shape == (24, 4) and t.zeros.dtype is torch.uint8
        assert widen_w4(t).shape == (24, 256) and linear_w4(x, t).shape == (3, 5, 24) and linear_w4(x.new_empty(500, 256), t).shape == (500, 24)
        assert LinearW4(t)(x).shape == (3, 5, 24)
        for bad in (lambda: quantize_w4(w, 48), lambda: quantize_w4(w.float()), lambda: linear_w4(x[..., :128], t), lambda: linear_w4(x.float(), t),
                    lambda: linear_w4(x.clone().requires_grad_(True), t)):
            with pytest.raises(ValueError):
                bad()


def test_four_bits_are_traced(monkeypatch):
    from torch.fx.experimental.proxy_tensor import make_fx

    from roc_shmem_b200.ops.gemm_w4 import W4Tensor, linear_w4, quantize_w4, widen_w4
    t = W4Tensor(torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1, dtype=BF))
    monkeypatch.setattr(gemm_w4, "linear_direct", lambda x, w: x @ w.dequantize().t())
    monkeypatch.setattr(gemm_w4, "_check_x", lambda *_: None)
    monkeypatch.setattr(gemm_w4, "_checked", lambda *_: (8, 64, 64))
    x = torch.randn(5, 64)
    for traced in (make_fx(lambda v: linear_w4(v, t))(torch.zeros(5, 64)), torch.jit.trace(lambda v: linear_w4(v, t), (torch.zeros(5, 64),), check_trace=False)):
        assert "linear_w4" in str(traced.graph)
        _close(traced(x), x @ t.dequantize().t())
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        s = forward_ad.make_dual(t.scales, t.scales)
        for call in (lambda: linear_w4(d, t), lambda: linear_w4(x, W4Tensor(t.q, s)), lambda: widen_w4(W4Tensor(t.q, s)), lambda: quantize_w4(d)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
