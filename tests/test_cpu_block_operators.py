"""The norms', the 8-bit activations' and the 4-bit weights' operators without a GPU: what they refuse before any launch, their formulas against
differences, and the layouts that the kernels choose."""
import ctypes as C

import pytest
import torch

from block_reference import round8, rstd_of, through


def test_python_refuses_what_is_not_on_a_gpu():
    from roc_shmem_b200.ops.checkpoint8 import store, swiglu_store
    from roc_shmem_b200.ops.gemm_w4 import LinearW4, W4Tensor, linear_w4, quantize_w4, widen_w4
    from roc_shmem_b200.ops.norms import post_norm, post_pre_norm, rms_norm
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    q = W4Tensor(torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1, dtype=torch.bfloat16))
    for call in (lambda: rms_norm(x, w), lambda: post_norm(x, x, w), lambda: post_pre_norm(x, x, w, w), lambda: store(x), lambda: swiglu_store(x),
                 lambda: linear_w4(x, q), lambda: widen_w4(q), lambda: quantize_w4(x, 32), lambda: LinearW4(q)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    assert q.group == 64 and torch.equal(q.dequantize(), torch.full((8, 64), -8.0))
    z = W4Tensor(torch.full((2, 32), 0xA3, dtype=torch.uint8), torch.full((2, 2), 0.5, dtype=torch.bfloat16), torch.tensor([[3, 10], [0, 15]], dtype=torch.uint8))
    assert torch.equal(z.dequantize()[0, :4], torch.tensor([0.0, 3.5, 0.0, 3.5])) and z.dequantize()[1, 63] == -2.5


def test_native_entries_refuse_bad_sizes():
    """Sizes and types are looked at before CUDA is."""
    from roc_shmem_b200.ops import checkpoint8, gemm_w4, norms
    n, c, w = norms._lib(), checkpoint8._lib(), gemm_w4._lib()
    assert n.bshmem_norm_fwd(3, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 8, 0) == 1          # type
    assert n.bshmem_norm_fwd(3 << 2, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 8, 0) == 1     # mode
    for rows, cols in ((1, 0), (1, 16385), (1 << 31, 8)):
        assert n.bshmem_norm_fwd(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, rows, cols, 0) == 1
        assert n.bshmem_norm_bwd(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, rows, cols, 0) == 1
    assert b"16384" in n.bshmem_norm_last_error()
    assert n.bshmem_norm_fwd(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 8, 0) == 0           # no rows: nothing to do
    assert n.bshmem_norm_bwd_groups(0, 8) < 0 and n.bshmem_norm_bwd_groups(1, 16385) < 0
    assert c.bshmem_ckpt8_store(3, 0, 8, 0, 1, 8, 0) == 1 and c.bshmem_ckpt8_store(0, 0, 8, 0, 1, 0, 0) == 1
    assert c.bshmem_ckpt8_store(0, 0, 8, 0, 0, 8, 0) == 0 and c.bshmem_ckpt8_restore(3, 0, 0, 8, 1, 8, 0) == 1
    for F in (0, 31, 48):
        assert c.bshmem_ckpt8_swiglu_store(0, 0, 0, 1, F, 0) == 1 and c.bshmem_ckpt8_swiglu_backward(0, 0, 0, 0, 1, F, 0) == 1
    assert c.bshmem_ckpt8_swiglu_store(8, 0, 0, 1, 64, 0) == 1                                    # off a 16-byte boundary
    for N, K, group in ((0, 64, 32), (8, 48, 48), (8, 96, 64), (8, 192, 128), (8, 64, 0), (8, 1 << 25, 128)):
        assert w.bshmem_w4_few(0, K, 0, 0, 0, 0, 1, N, K, group, 0, 0) == 1
        assert w.bshmem_w4_widen(0, 0, 0, 0, N, K, group, 0) == 1 and w.bshmem_w4_quant(0, K, 0, 0, 0, N, K, group, 0) == 1
    assert w.bshmem_w4_few(8, 64, 0, 0, 0, 0, 1, 8, 64, 32, 0, 0) == 1 and w.bshmem_w4_few(0, 60, 0, 0, 0, 0, 1, 8, 64, 32, 0, 0) == 1
    assert w.bshmem_w4_few(0, 64, 0, 0, 0, 0, 0, 8, 64, 32, 0, 0) == 0                               # no tokens


def test_formula_of_the_gradient_against_autograd():
    """`through` at the true values is the derivative of v * rstd(v) u, by autograd in 64 bits."""
    g = torch.Generator().manual_seed(0)
    v = torch.randn(5, 37, generator=g, dtype=torch.float64, requires_grad=True)
    u = torch.randn(5, 37, generator=g, dtype=torch.float64)
    expect, = torch.autograd.grad(v * rstd_of(v, 1e-5), v, u)
    got, size = through(v.detach(), rstd_of(v.detach(), 1e-5), u, u.abs())
    # some forty roundings of 2^-53 of terms of `size`
    assert ((got - expect).abs() <= 64 * 2.0 ** -53 * size).all()


def test_eight_bits_in_the_oracle():
    """The oracle's own values: representable ones come back, ties go to the even neighbour, the scale is the smallest that holds."""
    x = torch.tensor([[448.0, 1.0, 1.0625, 1.1875, -2.0 ** -6, 2.0 ** -10, 0.0, 449.0]], dtype=torch.float32)
    a = round8(x[:, :7])
    assert a.tolist() == [[448.0, 1.0, 1.0, 1.25, -2.0 ** -6, 0.0, 0.0]]
    b = round8(x)                                              # 449 needs steps of twice the size
    assert b[0, 0] == 448.0 and b[0, 7] == 448.0 and b[0, 4] == -2.0 ** -6 and b[0, 5] == 0.0
    big = torch.tensor([[torch.finfo(torch.bfloat16).max, 1e38]], dtype=torch.bfloat16)
    assert round8(big)[0, 0] == 240 * 2.0 ** 120
    half = torch.tensor([[65504.0, 1.0]], dtype=torch.float16)
    assert round8(half)[0, 0] == 240 * 256


def test_few_tokens_rule():
    from roc_shmem_b200.ops.gemm_w4 import few_tokens
    assert [few_tokens(g) for g in (32, 64, 128, 256)] == [32, 128, 128, 128]
    assert C.sizeof(C.c_longlong) == 8


def test_checkpoints_that_do_not_hold_their_shape():
    """The kernels write as many rows as the shape has, so bytes for another number of them are refused, and whatever is not on a GPU."""
    from roc_shmem_b200.ops.checkpoint8 import Checkpoint8, kept_bytes, restore, swiglu_backward
    bf, shape = torch.bfloat16, torch.Size((4, 64))
    data = torch.zeros(kept_bytes(4, 64) + 16, dtype=torch.uint8)
    size, dact = kept_bytes(4, 64), torch.zeros(4, 32, dtype=bf)
    assert size == 4 * 65 and Checkpoint8(data[:size], shape, bf).rows == 4
    for kept in (Checkpoint8(data, shape, bf), Checkpoint8(data[:size - 1], shape, bf), Checkpoint8(data[:size], torch.Size((5, 64)), bf),
                 Checkpoint8(data[:size], torch.Size((3, 64)), bf), Checkpoint8(data[:size], torch.Size(()), bf),
                 Checkpoint8(data[:size], torch.Size((4, 0)), bf), Checkpoint8(data[1:size + 1], shape, bf),
                 Checkpoint8(data[:size].view(torch.int8), shape, bf)):
        for call in (lambda: restore(kept), lambda: swiglu_backward(kept, dact)):
            with pytest.raises(ValueError, match="does not hold"):
                call()
    for call in (lambda: restore(Checkpoint8(data[:size], shape, bf)), lambda: swiglu_backward(Checkpoint8(data[:size], shape, bf), dact)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_modules_saved_before_there_were_checkpoints():
    """What unpickling makes of a layer that was saved without the attributes."""
    from roc_shmem_b200.models.llama import LlamaMLPModule
    from roc_shmem_b200.ops.torch_ops import Linear
    assert Linear.__new__(Linear).checkpoint is False
    old = LlamaMLPModule.__new__(LlamaMLPModule)
    assert old.checkpoint is False and old.norms is False


def test_kept_norms_hold_every_word_that_is_read(monkeypatch):
    """The backward pass reads an exponent by the aligned word of four bytes that it is in, the last one's too: the buffer that the call
    makes has them all."""
    from types import SimpleNamespace

    from roc_shmem_b200.ops import norms
    monkeypatch.setattr(norms, "_fwd", lambda *_: 0)
    monkeypatch.setattr(norms, "current_stream", lambda: 0)
    for mode in (norms.PRE, norms.POST, norms.POST_PRE):
        for rows in (1, 2, 3, 501):
            for n in (8, 128, 136, 232, 520, 8200):
                x = torch.empty(rows, n, dtype=torch.bfloat16)
                c = SimpleNamespace(rows=rows, n=n, like=x, what=norms.KEPT, y=x, x=x, w1=None, w2=None, gate=None, gate_ld=0, scale=None, eps=1e-6, number=1.0)
                kept = norms._forward(c, mode, True)[3]
                count = 2 if mode == norms.POST_PRE else 1
                last = count * rows * ((n + 15) // 16 * 16 + (n + 127) // 128) - 1
                assert last // 4 * 4 + 4 <= kept.numel() < last + 5


def test_layer_reports_a_wait_that_ran_out(monkeypatch):
    """Of either kernel that it runs on; a layer whose device no longer answers says so too."""
    from contextlib import nullcontext
    from types import SimpleNamespace

    from roc_shmem_b200.ops import gemm_w4
    monkeypatch.setattr(torch.cuda, "device", lambda d: nullcontext())
    layer = SimpleNamespace(q=torch.zeros(1))
    sites = {"w4_error_site": 0, "gemm_error_site": 0}
    for name in sites:
        monkeypatch.setattr(gemm_w4, name, lambda name=name: sites[name])
    gemm_w4.LinearW4.check(layer)
    for name, site in (("w4_error_site", 403), ("gemm_error_site", 7), ("w4_error_site", -1)):
        sites[name] = site
        with pytest.raises(RuntimeError, match=f"site {site}"):
            gemm_w4.LinearW4.check(layer)
        sites[name] = 0


def test_kept_norms_from_a_hook_are_aligned(monkeypatch):
    """What a hook on saved tensors brings back may lie anywhere; the kernels get kept bytes on a 16-byte boundary and 1 / sqrt(...) side by side."""
    from roc_shmem_b200.ops import norms
    seen = []
    monkeypatch.setattr(norms, "_bwd", lambda *a: seen.append((a[13], a[14])) or 0)
    monkeypatch.setattr(norms, "current_stream", lambda: 0)
    rows, n = 6, 200
    x = torch.zeros(rows, n, dtype=torch.bfloat16)
    buffer = torch.zeros(norms.kept_size(1, rows, n) + 16, dtype=torch.uint8)
    for off in (0, 1, 4, 8):
        a = buffer[off:off + norms.kept_size(1, rows, n)]
        for rstd in (torch.zeros(1, rows), torch.zeros(1, 2 * rows)[:, ::2]):
            seen.clear()
            norms._gradients((norms.PRE, norms.KEPT, n, rows, norms.NO_GATE, 0), (False, True) + (False,) * 4, (None, None, None, None, rstd, a, None), None, x)
            (r, k), = seen
            assert k % 16 == 0 and (k == a.data_ptr()) == (off == 0) and (r == rstd.data_ptr()) == rstd.is_contiguous()
