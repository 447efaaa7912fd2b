"""Activations kept in 8 bits between the forward and the backward pass.

An activation that is only read again for a gradient is stored as e4m3 with one power of two per row and 128 columns:
half the bytes of bf16, and a relative error of at most 2^-4 for values down to 2^-13 of their block's largest.  ``store``
and ``restore`` are the way there and back; ``swiglu`` is the gated activation that keeps its input so; ``Linear`` and the norms
take ``checkpoint=True``.  Values that e4m3 does not have come back as NaN (infinities too).  No gradient goes through ``store`` and
``restore``.  Traced, compiled, fake and watched calls are the registered operators ``torch.ops.bshmem.store8``, ``restore8``, ``swiglu8`` and
``swiglu8_backward``; there is no forward-mode derivative.

The reference is a communication runtime without activations, so there is no parity citation.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _native
from .gemm import current_stream
from .watched import direct, direct_gradients

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_declared = False
_store = _restore = _swiglu_store = _swiglu_backward = None


def block_lib() -> C.CDLL:
    """The library of the norms, the 8-bit activations and the 4-bit weights."""
    return _native.load("libbshmem_block.so")


def _lib() -> C.CDLL:
    global _declared, _store, _restore, _swiglu_store, _swiglu_backward
    lib = block_lib()
    if not _declared:
        VP, I, L = C.c_void_p, C.c_int, C.c_longlong
        lib.bshmem_ckpt8_last_error.restype = C.c_char_p
        for name, args in (("store", [I, VP, L, VP, L, I, VP]), ("restore", [I, VP, VP, L, L, I, VP]),
                           ("swiglu_store", [VP, VP, VP, L, I, VP]), ("swiglu_backward", [VP, VP, VP, VP, L, I, VP])):
            fn = getattr(lib, "bshmem_ckpt8_" + name)
            fn.restype, fn.argtypes = I, args
        _swiglu_store, _swiglu_backward = _native.fast(lib, "bshmem_ckpt8_swiglu_store"), _native.fast(lib, "bshmem_ckpt8_swiglu_backward")
        _restore, _store = _native.fast(lib, "bshmem_ckpt8_restore"), _native.fast(lib, "bshmem_ckpt8_store")
        _declared = True
    return lib


def _check(st: int, what: str) -> None:
    if st != 0:
        raise RuntimeError(f"{what} failed ({st}): {_lib().bshmem_ckpt8_last_error().decode()}")


def on_current_device(t: torch.Tensor) -> bool:
    """Whether `t` is on the current CUDA device, whose current stream the kernels are launched on."""
    return t.get_device() == torch._C._cuda_getDevice()


def kept_bytes(rows: int, cols: int) -> int:
    """Bytes of a [rows, cols] activation in 8 bits: its values, rows padded to 16 columns, then an exponent per row and 128 columns."""
    return rows * ((cols + 15) // 16 * 16 + (cols + 127) // 128)


@dataclass
class Checkpoint8:
    """An activation in 8 bits.  ``data`` holds ``q`` [rows, columns rounded up to 16], e4m3 bytes (zeros in the columns more), and behind it ``e`` [rows, blocks of 128
    columns], biased exponents: the value of a byte is e4m3 * 2^(e - 127).  ``shape`` and ``dtype`` are those of the tensor that was stored."""
    data: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    @property
    def rows(self) -> int:
        return self.data.numel() // kept_bytes(1, self.shape[-1])

    @property
    def q(self) -> torch.Tensor:
        width = (self.shape[-1] + 15) // 16 * 16
        return self.data[:self.rows * width].view(-1, width)

    @property
    def e(self) -> torch.Tensor:
        return self.data[self.rows * ((self.shape[-1] + 15) // 16 * 16):].view(-1, (self.shape[-1] + 127) // 128)

    def restore(self, dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        return restore(self, dtype, out)

    @property
    def nbytes(self) -> int:
        return self.data.nbytes


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as [rows, columns] with neighbouring columns side by side; rows may be apart."""
    if not x.is_cuda or x.dtype not in _TYPES:
        raise ValueError(f"{what} needs a bf16, fp16 or fp32 CUDA tensor, got {x.dtype} on {x.device}")
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] >= 1 << 30:
        raise ValueError(f"{what} needs rows of 1 to 2^30 columns, got {tuple(x.shape)}")
    m = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return m if m.stride(1) == 1 else m.contiguous()


def _held(kept: Checkpoint8, what: str, addressed: bool = True) -> tuple[torch.Tensor, int, int]:
    """(bytes, rows, columns) of `kept`, whose shape says what the kernels write.  Not `addressed`: it is not for a kernel of this call."""
    data, shape = kept.data, kept.shape
    cols = shape[-1] if shape else 0
    rows = shape.numel() // cols if cols else 0
    if (not cols or data.numel() != kept_bytes(rows, cols) or data.dtype is not torch.uint8 or not data.is_contiguous()
            or (addressed and data.data_ptr() % 16)):
        raise ValueError(f"{what}: the checkpoint does not hold a {tuple(shape)}")
    if not data.is_cuda and addressed:
        raise ValueError(f"{what} needs a checkpoint of a CUDA tensor, got one on {data.device}")
    return data, rows, cols


def store(x: torch.Tensor) -> Checkpoint8:
    """bf16, fp16 or fp32 [..., columns] → 8 bits."""
    return Checkpoint8(store_direct(x) if direct("store", x) else _operators().store8(x), x.shape, x.dtype)


def store_direct(x: torch.Tensor) -> torch.Tensor:
    m = _rows(x, "store")
    if not on_current_device(x):
        with torch.cuda.device(x.device):
            return store_direct(x)
    if _store is None:
        _lib()
    rows, cols = m.shape
    data = x.new_empty((kept_bytes(rows, cols),), dtype=torch.uint8)
    st = _store(_TYPES[x.dtype], m.data_ptr(), m.stride(0), data.data_ptr(), rows, cols, current_stream())
    if st != 0:
        _check(st, "store")
    return data


def restore(kept: Checkpoint8, dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The stored values in `dtype` (default: what was stored), into `out` if given ([rows, columns] with columns side by side)."""
    dtype = dtype or (out.dtype if out is not None else kept.dtype)
    if direct("restore", kept.data, out):
        return restore_direct(kept, dtype, out)
    _check_dtype(dtype)
    _, rows, cols = _held(kept, "restore", False)
    if out is not None:
        _check_out(out, rows, cols, dtype, kept.data)
    got = _operators().restore8(kept.data, cols, dtype)
    return got.view(kept.shape) if out is None else out.copy_(got)


def _check_dtype(dtype: torch.dtype) -> None:
    if dtype not in _TYPES:
        raise ValueError(f"restore gives bf16, fp16 or fp32, not {dtype}")


def _check_out(out: torch.Tensor, rows: int, cols: int, dtype: torch.dtype, data: torch.Tensor) -> None:
    if out.shape != (rows, cols) or out.dtype != dtype or out.device != data.device or out.stride(1) != 1 or (rows > 1 and out.stride(0) < cols):
        raise ValueError("bad output tensor")


def restore_direct(kept: Checkpoint8, dtype: torch.dtype, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    data, rows, cols = _held(kept, "restore")
    if dtype not in _TYPES:
        _check_dtype(dtype)
    if not on_current_device(data):
        with torch.cuda.device(data.device):
            return restore_direct(kept, dtype, out)
    if _restore is None:
        _lib()
    if out is None:
        out = data.new_empty(kept.shape, dtype=dtype)
        ld = cols
    else:
        _check_out(out, rows, cols, dtype, data)
        ld = out.stride(0)
    st = _restore(_TYPES[dtype], data.data_ptr(), out.data_ptr(), ld, rows, cols, current_stream())
    if st != 0:
        _check(st, "restore")
    return out


def _check_gu(gu: torch.Tensor) -> None:
    if not gu.is_cuda or gu.dtype is not torch.bfloat16 or gu.dim() < 1 or gu.shape[-1] < 64 or gu.shape[-1] % 64:
        raise ValueError(f"swiglu needs bf16 CUDA rows of 32 gate and 32 up columns in turn, got {gu.dtype} {tuple(gu.shape)} on {gu.device}")


def _aligned(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _swiglu_forward(gu: torch.Tensor, keep: bool) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    _check_gu(gu)
    if not on_current_device(gu):
        with torch.cuda.device(gu.device):
            return _swiglu_forward(gu, keep)
    if _swiglu_store is None:
        _lib()
    g = _aligned(gu)
    F = gu.shape[-1] // 2
    rows = gu.numel() // (2 * F)
    act = gu.new_empty((*gu.shape[:-1], F))
    data = gu.new_empty((kept_bytes(rows, 2 * F),), dtype=torch.uint8) if keep else None
    st = _swiglu_store(g.data_ptr(), act.data_ptr(), None if data is None else data.data_ptr(), rows, F, current_stream())
    if st != 0:
        _check(st, "swiglu_store")
    return act, data


def swiglu_store(gu: torch.Tensor) -> tuple[torch.Tensor, Checkpoint8]:
    """act [..., F] = silu(gate) * up of gu [..., 2F] (32 columns of the gate, then the 32 of ``up``, see
    ``interleave_gate_up``), and gu in 8 bits, in one pass."""
    act, data = _swiglu_forward(gu, True) if direct("swiglu_store", gu) else _operators().swiglu8(gu.detach(), True)
    return act, Checkpoint8(data, gu.shape, gu.dtype)


def swiglu_backward(kept: Checkpoint8, dact: torch.Tensor, *, act: bool = False, dgu_out: Optional[torch.Tensor] = None,
                    act_out: Optional[torch.Tensor] = None):
    """Gradient of gu from its 8 bits and the activation's gradient; with `act` also the activation again, of the same 8 bits (what
    the next layer's weight gradient reads).  `dgu_out`, `act_out`: contiguous buffers for them."""
    act = act or act_out is not None
    if direct("swiglu_backward", kept.data, dact, dgu_out, act_out):
        return swiglu_backward_direct(kept, dact, act, dgu_out, act_out)
    _check_dact(kept, _held(kept, "swiglu_backward", False)[2], dact)
    for given, like in ((dgu_out, kept.shape), (act_out, dact.shape)):
        if given is not None:
            _check_buffer(given, like, dact)
    dgu, again = _operators().swiglu8_backward(kept.data, dact, act)
    dgu = dgu if dgu_out is None else dgu_out.copy_(dgu)
    return (dgu, again if act_out is None else act_out.copy_(again)) if act else dgu


def _check_dact(kept: Checkpoint8, cols: int, dact: torch.Tensor) -> None:
    like = (*kept.shape[:-1], cols // 2)
    if cols % 64 or dact.dtype is not torch.bfloat16 or dact.shape != like or dact.get_device() != kept.data.get_device():
        raise ValueError(f"swiglu_backward: a bf16 gradient of {like} belongs to this checkpoint, got {dact.dtype} {tuple(dact.shape)}")


def _check_buffer(given: torch.Tensor, like: torch.Size, d: torch.Tensor) -> None:
    if given.shape != like or given.dtype is not torch.bfloat16 or given.device != d.device or not given.is_contiguous():
        raise ValueError("bad output tensor")


def swiglu_backward_direct(kept: Checkpoint8, dact: torch.Tensor, act: bool, dgu_out: Optional[torch.Tensor] = None,
                           act_out: Optional[torch.Tensor] = None):
    data, rows, cols = _held(kept, "swiglu_backward")
    if not on_current_device(data):
        with torch.cuda.device(data.device):
            return swiglu_backward_direct(kept, dact, act, dgu_out, act_out)
    _check_dact(kept, cols, dact)
    if _swiglu_backward is None:
        _lib()
    d = _aligned(dact)

    def buffer(given, like):
        if given is None:
            return d.new_empty(like)
        _check_buffer(given, like, d)
        if given.data_ptr() % 16:
            raise ValueError("bad output tensor")
        return given
    dgu = buffer(dgu_out, kept.shape)
    again = buffer(act_out, dact.shape) if act else None
    st = _swiglu_backward(data.data_ptr(), d.data_ptr(), dgu.data_ptr(), None if again is None else again.data_ptr(), rows, cols // 2,
                          current_stream())
    if st != 0:
        _check(st, "swiglu_backward")
    return dgu if again is None else (dgu, again)


class _SwigluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu):
        act, data = _swiglu_forward(gu, True)
        ctx.save_for_backward(data)
        ctx.shape = gu.shape
        return act

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dact):
        data, = ctx.saved_tensors
        if not direct_gradients("swiglu", dact):
            return _operators().swiglu8_backward(data, dact, False)[0]
        return swiglu_backward_direct(Checkpoint8(data, ctx.shape, torch.bfloat16), dact, False)


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up of the interleaved gu [..., 2F]; what the gradient needs of gu is kept in 8 bits."""
    train = torch.is_grad_enabled() and gu.requires_grad
    if not direct("swiglu", gu):
        return _operators().swiglu8(gu, train)[0]
    return _SwigluFn.apply(gu) if train else _swiglu_forward(gu, False)[0]


# ---- registered operators: calls that somebody watches, traces or transforms ------------------------------------------------

def _operators():
    from . import torch_ops  # noqa: F401
    return torch.ops.bshmem


def operator_store_fake(x):
    rows, cols = _rows(x, "store").shape
    return x.new_empty((kept_bytes(rows, cols),), dtype=torch.uint8)


def _kept_rows(data, cols, dtype):
    if cols < 1 or data.numel() % kept_bytes(1, cols):
        raise ValueError(f"restore8: the checkpoint does not hold rows of {cols}")
    return Checkpoint8(data, torch.Size((data.numel() // kept_bytes(1, cols), cols)), dtype)


def operator_restore(data, cols, dtype):
    return restore_direct(_kept_rows(data, cols, dtype), dtype)


def operator_restore_fake(data, cols, dtype):
    _check_dtype(dtype)
    return data.new_empty(_kept_rows(data, cols, dtype).shape, dtype=dtype)


def operator_swiglu(gu, keep):
    act, data = _swiglu_forward(gu, keep)
    return act, gu.new_empty((0,), dtype=torch.uint8) if data is None else data


def operator_swiglu_fake(gu, keep):
    _check_gu(gu)
    cols = gu.shape[-1]
    size = kept_bytes(gu.numel() // cols, cols) if keep else 0
    return gu.new_empty((*gu.shape[:-1], cols // 2)), gu.new_empty((size,), dtype=torch.uint8)


def _kept_gu(data, dact):
    if dact.dim() < 1:
        raise ValueError("swiglu8_backward needs rows")
    return Checkpoint8(data, torch.Size((*dact.shape[:-1], 2 * dact.shape[-1])), torch.bfloat16)


def operator_swiglu_backward(data, dact, act):
    got = swiglu_backward_direct(_kept_gu(data, dact), dact, act)
    return got if act else (got, dact.new_empty((0,)))


def operator_swiglu_backward_fake(data, dact, act):
    kept = _kept_gu(data, dact)
    _check_dact(kept, _held(kept, "swiglu_backward", False)[2], dact)
    return dact.new_empty(kept.shape), dact.new_empty(dact.shape if act else (0,))
