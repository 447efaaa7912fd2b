"""RMS norms before and after a block, fused with the block's gate, its residual scale and the residual sum.

    rms_norm       h   = weight * n(x)                                     n(v) = v / sqrt(mean(v^2) + eps) over the last dimension
    post_norm      out = residual + scale * gate * weight * n(y)           y: what the block returned
    post_pre_norm  both in one pass: out, and the next block's h = next_weight * n(out)

Rows are bf16, fp16 or fp32, sums fp32.  A weight is one value per column, of the rows' type or fp32; the gate one per column
``[H]``, per row ``[..., 1]`` or per element (weights and gates may be left out); the scale a number or a tensor with one
element.  Every tensor has a gradient; sums over rows are added in a fixed order, so a call gives the same bits again.
``checkpoint=True`` keeps the norms' inputs for the backward pass in 8 bits (``checkpoint8``): n(v) is then the kept v times the true
row's 1 / sqrt(mean + eps) wherever a gradient has it.  Rows have 1 to 16384 columns and may be apart (any stride of the leading dimension); rows of a multiple of 8 columns on
16-byte boundaries are the fast ones.  A backward pass that a CUDA graph captures wants every eager graph of the same leaves gone: torch
keeps their gradients' accumulators as long, and with them the stream that they were made on.  Squares are fp32: rows whose squares leave its range give what that gives.
Traced, compiled, fake and watched calls are the registered operators ``torch.ops.bshmem.norm`` and ``norm_backward``; there is no forward-mode
derivative.

The reference is a communication runtime without models, so there is no parity citation.
"""
from __future__ import annotations

import ctypes as C
import struct
from functools import lru_cache
from typing import Optional, Union

import torch

from .. import _native
from .checkpoint8 import _TYPES, block_lib, kept_bytes, on_current_device
from .gemm import current_stream
from .watched import direct, direct_gradients

PRE, POST, POST_PRE = range(3)
NO_GATE, COLUMN, ROW, ELEMENT = range(4)
MAX_COLUMNS = 16384
KEPT = 1 << 12                                           # the call keeps its norms' inputs in 8 bits
_NAMES = ("rms_norm", "post_norm", "post_pre_norm")
_F32, _CONTIGUOUS, _new_like = torch.float32, torch.contiguous_format, torch.empty_like
_declared = False
_fwd = _bwd = _groups = _finish = None


def _lib() -> C.CDLL:
    global _declared, _fwd, _bwd, _groups, _finish
    lib = block_lib()
    if not _declared:
        VP, I, L, U = C.c_void_p, C.c_int, C.c_longlong, C.c_uint64
        lib.bshmem_norm_last_error.restype = C.c_char_p
        lib.bshmem_norm_fwd.restype = I
        lib.bshmem_norm_fwd.argtypes = [I, VP, L, VP, L, VP, VP, VP, VP, VP, L, VP, U, VP, VP, L, I, VP]
        lib.bshmem_norm_bwd.restype = I
        lib.bshmem_norm_bwd.argtypes = [I, VP, VP, VP, L, VP, L, VP, VP, VP, L, VP, U, VP, VP, I, VP, VP, VP, VP, L, I, VP]
        lib.bshmem_norm_bwd_finish.restype = I
        lib.bshmem_norm_bwd_finish.argtypes = [I, VP, VP, VP, VP, U, VP, VP, VP, VP, L, I, VP]
        lib.bshmem_norm_bwd_groups.restype = I
        lib.bshmem_norm_bwd_groups.argtypes = [L, I]
        _bwd, _groups = _native.fast(lib, "bshmem_norm_bwd"), _native.fast(lib, "bshmem_norm_bwd_groups")
        _finish, _fwd = _native.fast(lib, "bshmem_norm_bwd_finish"), _native.fast(lib, "bshmem_norm_fwd")
        _declared = True
    return lib


def _check(st: int, what: str) -> None:
    if st != 0:
        raise RuntimeError(f"{what} failed ({st}): {_lib().bshmem_norm_last_error().decode()}")


@lru_cache(maxsize=256)
def _bits(value: float) -> int:
    return struct.unpack("<I", struct.pack("<f", value))[0]


@lru_cache(maxsize=256)
def _numbers(eps: float, scale: float) -> int:
    return _bits(eps) | _bits(scale) << 32


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _matrix(t: torch.Tensor, cols: int) -> torch.Tensor:
    m = t if t.dim() == 2 else t.reshape(-1, cols)
    return m if m.stride(1) == 1 or cols == 1 else m.contiguous()


def _refuse_vector(name, label, t, x):
    raise ValueError(f"{name}: {label} must be {x.dtype} or fp32 of shape ({x.shape[-1]},) on {x.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


class _Call:
    """A call's operands, checked: what they are in one word, and their addresses and pitches."""
    __slots__ = ("what", "y", "x", "w1", "w2", "gate", "scale", "number", "eps", "rows", "n", "like", "gate_ld", "kind")

    def __init__(self, name, mode, y, x, w1, w2, gate, scale, eps, checkpoint):
        dt, shape = x.dtype, x.shape
        what = _TYPES.get(dt)
        if what is None or not x.is_cuda:
            raise ValueError(f"{name} needs bf16, fp16 or fp32 CUDA tensors, got {dt} on {x.device}")
        if not shape or not 1 <= shape[-1] <= MAX_COLUMNS:
            raise ValueError(f"{name} needs rows of 1 to {MAX_COLUMNS} columns, got {tuple(shape)}")
        if not 1.2e-38 < eps < 3.4e38:
            raise ValueError(f"{name} needs eps > 0, a normal fp32 number")
        n, dev = shape[-1], x.get_device()
        what |= mode << 2
        if checkpoint:
            what |= KEPT
        self.eps, self.n, self.like, self.kind = eps, n, x, NO_GATE
        self.x, self.y = _matrix(x, n), None
        self.rows = self.x.shape[0]
        if self.rows > 0x7fffffff:
            raise ValueError(f"{name} takes less than 2^31 rows")

        column = (n,)
        if w1 is not None:
            if w1.shape != column or w1.get_device() != dev or (w1.dtype is not dt and w1.dtype is not _F32):
                _refuse_vector(name, "weight", w1, x)
            if w1.dtype is _F32:
                what |= 1 << 8
            if not w1.is_contiguous():
                w1 = w1.contiguous()
        if w2 is not None:
            if w2.shape != column or w2.get_device() != dev or (w2.dtype is not dt and w2.dtype is not _F32):
                _refuse_vector(name, "weight" if mode == PRE else "next_weight", w2, x)
            if w2.dtype is _F32:
                what |= 1 << 9
            if not w2.is_contiguous():
                w2 = w2.contiguous()
        self.w1, self.w2, self.gate, self.gate_ld, self.scale, self.number = w1, w2, None, 0, None, 1.0
        if mode != PRE:
            if y.shape != shape or y.dtype is not dt or y.get_device() != dev:
                raise ValueError(f"{name}: y and residual must be alike, got {y.dtype} {tuple(y.shape)} on {y.device} and {dt} {tuple(shape)} on {x.device}")
            self.y = _matrix(y, n)
            if gate is not None:
                if gate.get_device() != dev or (gate.dtype is not dt and gate.dtype is not _F32):
                    raise ValueError(f"{name}: gate must be {dt} or fp32 on {x.device}, got {gate.dtype} on {gate.device}")
                if gate.dtype is _F32:
                    what |= 1 << 10
                if gate.shape == column:
                    self.kind, self.gate = COLUMN, gate.contiguous()
                else:
                    if gate.shape == shape:
                        self.kind, self.gate = ELEMENT, _matrix(gate, n)
                    elif gate.shape == (*shape[:-1], 1):
                        self.kind, self.gate = ROW, _matrix(gate, 1)
                    else:
                        raise ValueError(f"{name}: gate must be ({n},), {(*shape[:-1], 1)} or {tuple(shape)}, got {tuple(gate.shape)}")
                    self.gate_ld = self.gate.stride(0)
                what |= self.kind << 4
            if scale is None:
                pass
            elif isinstance(scale, torch.Tensor):
                if scale.numel() != 1 or scale.get_device() != dev or (scale.dtype is not dt and scale.dtype is not _F32):
                    raise ValueError(f"{name}: scale must be a number or one element of {dt} or fp32 on {x.device}")
                self.scale = scale
                if scale.dtype is _F32:
                    what |= 1 << 11
            else:
                self.number = float(scale)
        self.what = what


def kept_size(norms: int, rows: int, n: int) -> int:
    """Bytes that a call of `norms` norms keeps in 8 bits: values, then exponents, which the backward pass
    reads in whole words; what has no value is zero."""
    return (norms * kept_bytes(rows, n) + 3) // 4 * 4


def _forward(c: _Call, mode: int, train: bool):
    """(out, h, rstd, kept); what the call does not give is None."""
    if _fwd is None:
        _lib()
    rows, n, like, what = c.rows, c.n, c.like, c.what
    out = _new_like(like, memory_format=_CONTIGUOUS) if mode != PRE else None
    h = _new_like(like, memory_format=_CONTIGUOUS) if mode != POST else None
    rstd = kept = None
    if train:
        norms = 2 if mode == POST_PRE else 1
        rstd = torch.empty((norms, rows), dtype=_F32, device=like.device)
        if what & KEPT:
            kept = like.new_empty((kept_size(norms, rows, n),), dtype=torch.uint8)
    else:
        what &= ~KEPT
    y, x = c.y, c.x
    st = _fwd(what, None if y is None else y.data_ptr(), 0 if y is None else y.stride(0), x.data_ptr(), x.stride(0),
              None if out is None else out.data_ptr(), None if h is None else h.data_ptr(), None if c.w1 is None else c.w1.data_ptr(),
              None if c.w2 is None else c.w2.data_ptr(), None if c.gate is None else c.gate.data_ptr(), c.gate_ld, _p(c.scale),
              _numbers(c.eps, c.number), _p(rstd), _p(kept), rows, n, current_stream())
    if st != 0:
        _check(st, "norm")
    return out, h, rstd, kept


def _gradients(call, need, saved, dout, dh):
    """Gradients of y, x, w1, w2, gate and scale, as far as `need` asks for them, from what _NormFn keeps."""
    w1, w2, gate, scale, rstd, a, b = saved
    need_y, need_x, need_w1, need_w2, need_gate, need_scale = need[:6]
    mode, what, n, rows, kind, number = call
    if dout is None and dh is None:
        return (None,) * 6
    like = dout if dout is not None else dh
    dw_next = None
    if mode == POST_PRE and dh is None:                 # nobody used h: the first norm alone
        mode, what = POST, what & ~(3 << 2) | POST << 2
        dw_next = torch.zeros_like(w2) if need_w2 else None
        need_w2 = False
    if rows == 0:
        return (torch.zeros_like(like) if need_y else None, torch.zeros_like(like) if need_x else None, torch.zeros_like(w1) if need_w1 else None,
                dw_next if dw_next is not None else torch.zeros_like(w2) if need_w2 else None, torch.zeros_like(gate) if need_gate else None,
                torch.zeros_like(scale) if need_scale else None)
    if dout is not None and not dout.is_contiguous():
        dout = dout.contiguous()
    if dh is not None and not dh.is_contiguous():
        dh = dh.contiguous()
    kept8 = what & KEPT
    if not rstd.is_contiguous():                        # a hook on saved tensors may have brought them back some other way
        rstd = rstd.contiguous()
    if kept8 and (a.data_ptr() % 16 or not a.is_contiguous()):
        a = a.clone(memory_format=_CONTIGUOUS)
    y = None if kept8 or a is None else _matrix(a, n)
    z = None if kept8 or b is None else _matrix(b, n)
    dz = _new_like(like, memory_format=_CONTIGUOUS) if mode != POST else dout
    dy = _new_like(like, memory_format=_CONTIGUOUS) if need_y and mode != PRE else None
    dgate = _new_like(gate, memory_format=_CONTIGUOUS) if need_gate else None
    column = kind == COLUMN
    gate_m, gate_ld = gate, 0
    if gate is not None:
        if column:
            gate_m = gate if gate.is_contiguous() else gate.contiguous()
        else:
            gate_m = _matrix(gate, 1 if kind == ROW else n)
            gate_ld = gate_m.stride(0)
    if w1 is not None and not w1.is_contiguous():
        w1 = w1.contiguous()
    if w2 is not None and not w2.is_contiguous():
        w2 = w2.contiguous()
    sums = need_w1 or need_w2 or need_scale or (need_gate and column)
    work = None
    if sums:
        groups = _groups(rows, n)
        if groups < 1:
            _check(-groups, "norm backward")
        work = torch.empty((groups * ((n + 7) // 8 * 8 * (2 if mode == POST_PRE else 1) + 1),), dtype=_F32, device=like.device)
    stream = current_stream()
    if mode != POST or dy is not None or sums or dgate is not None:
        st = _bwd(what, _p(dout), _p(dh), _p(z), 0 if z is None else z.stride(0), _p(y), 0 if y is None else y.stride(0), _p(w1), _p(w2),
                  _p(gate_m), gate_ld, _p(scale), number, rstd.data_ptr(), _p(a) if kept8 else None, 2 if call[0] == POST_PRE else 1,
                  _p(dz) if mode != POST else None, _p(dy), None if column else _p(dgate), _p(work), rows, n, stream)
        if st != 0:
            _check(st, "norm backward")
    dw1 = dw2 = dscale = None
    if sums:
        dw1 = _new_like(w1) if need_w1 else None
        dw2 = _new_like(w2) if need_w2 else None
        dscale = _new_like(scale) if need_scale else None
        st = _finish(what, work.data_ptr(), _p(w1), _p(gate_m) if column else None, _p(scale), number, _p(dw1), _p(dw2),
                     _p(dgate) if column else None, _p(dscale), rows, n, stream)
        if st != 0:
            _check(st, "norm backward")
    return dy, dz if need_x else None, dw1, dw2 if dw_next is None else dw_next, dgate, dscale


@torch.autograd.function.once_differentiable
def _backward_once(ctx, dout, dh):
    return *_gradients(ctx.call, ctx.needs_input_grad, ctx.saved_tensors, dout, dh), None, None


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, w1, w2, gate, scale, c, mode):
        ctx.set_materialize_grads(False)
        out, h, rstd, kept = _forward(c, mode, True)
        ctx.call = mode, c.what, c.n, c.rows, c.kind, _bits(c.number)
        if kept is not None:
            ctx.save_for_backward(w1, w2, gate, scale, rstd, kept, None)
        else:
            ctx.save_for_backward(w1, w2, gate, scale, rstd, y, x if mode == PRE else None if mode == POST else out)
        return (out, h) if mode == POST_PRE else out if mode == POST else h

    @staticmethod
    def backward(ctx, *grads):
        call = ctx.call
        mode = call[0]
        dout, dh = grads[0] if mode != PRE else None, grads[-1] if mode != POST else None
        if not direct_gradients(_NAMES[mode], dout, dh):
            number = struct.unpack("<f", struct.pack("<I", call[5]))[0]
            return *_registered_gradients(mode, bool(call[1] & KEPT), number, ctx.needs_input_grad[:6], ctx.saved_tensors, dout, dh), None, None
        if torch.is_grad_enabled():
            return _backward_once(ctx, dout, dh)
        return *_gradients(call, ctx.needs_input_grad, ctx.saved_tensors, dout, dh), None, None


# ---- registered operators: calls that somebody watches, traces or transforms ------------------------------------------------

def _registered(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint):
    from . import torch_ops  # noqa: F401
    number = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        scale, number = None, float(scale)
    checkpoint = bool(checkpoint) and torch.is_grad_enabled() and any([t.requires_grad for t in (y, x, w1, w2, gate, scale) if t is not None])
    out, h, _, _ = torch.ops.bshmem.norm(y, x, w1, w2, gate, scale, number, float(eps), mode, checkpoint)
    return (out, h) if mode == POST_PRE else out if mode == POST else h


def _registered_gradients(mode, checkpoint, number, need, saved, dout, dh):
    from . import torch_ops  # noqa: F401
    need = list(need)
    if dout is None and dh is None:
        return (None,) * 6
    alone = mode == POST or (mode == POST_PRE and dh is None)
    dx = dout if alone and need[1] else None             # an operator may not return what it was given
    need[1] = need[1] and not alone
    found = torch.ops.bshmem.norm_backward(dout, dh, *saved, number, mode, checkpoint, sum(1 << i for i, wanted in enumerate(need) if wanted))
    found = [g if wanted else None for g, wanted in zip(found, need)]
    return found[0], found[1] if dx is None else dx, *found[2:]


def _only_its_own(what, mode, w1, w2, gate, scale) -> None:
    if (mode == PRE and not (w1 is gate is scale is None)) or (mode == POST and w2 is not None):
        raise ValueError(f"{what}: operands that do not belong to the mode")


def _whole_call(mode, y, x, w1, w2, gate, scale, number, eps, checkpoint) -> _Call:
    if mode not in (PRE, POST, POST_PRE) or (y is None) != (mode == PRE):
        raise ValueError("norm: unknown mode, or y does not belong to it")
    _only_its_own("norm", mode, w1, w2, gate, scale)
    return _Call(_NAMES[mode], mode, y, x, w1, w2, gate, number if scale is None else scale, eps, checkpoint)


def operator_forward(y, x, w1, w2, gate, scale, number, eps, mode, checkpoint):
    """torch.ops.bshmem.norm: (out, h, rstd, kept) of a call; what it does not have is empty."""
    c = _whole_call(mode, y, x, w1, w2, gate, scale, number, eps, checkpoint)
    with torch.cuda.device(x.device):
        found = _forward(c, mode, True)
    return tuple(x.new_empty(0) if t is None else t for t in found)


def operator_forward_fake(y, x, w1, w2, gate, scale, number, eps, mode, checkpoint):
    c = _whole_call(mode, y, x, w1, w2, gate, scale, number, eps, checkpoint)
    norms = 2 if mode == POST_PRE else 1
    return (_new_like(x, memory_format=_CONTIGUOUS) if mode != PRE else x.new_empty(0), _new_like(x, memory_format=_CONTIGUOUS) if mode != POST else x.new_empty(0),
            x.new_empty((norms, c.rows), dtype=_F32),
            x.new_empty((kept_size(norms, c.rows, c.n),), dtype=torch.uint8) if checkpoint else x.new_empty(0))


def _asked(need: int) -> list[bool]:
    return [bool(need >> i & 1) for i in range(6)]


def _whole_gradients(dout, dh, w1, w2, gate, scale, rstd, a, b, number, mode, checkpoint, need):
    """The call that these belong to, checked: the kernels go by its sizes."""
    like = dout if dout is not None else dh
    if mode not in (PRE, POST, POST_PRE) or like is None or (mode == PRE and dout is not None) or (mode == POST and dh is not None) or not 0 <= need < 64:
        raise ValueError("norm_backward: unknown mode, or gradients that do not belong to it")
    _only_its_own("norm_backward", mode, w1, w2, gate, scale)
    y = like if mode != PRE else None
    c = _Call("norm_backward", mode, y, like, w1, w2, gate, number if scale is None else scale, 1.0, checkpoint)
    norms = 2 if mode == POST_PRE else 1
    alike = [t for t in (dout, dh) if t is not None]
    if checkpoint:
        sized = a is not None and b is None and a.dtype is torch.uint8 and a.shape == (kept_size(norms, c.rows, c.n),) and a.is_contiguous()
        sized = sized and a.get_device() == like.get_device()
    else:
        sized = (a is not None) == (mode != PRE) and (b is not None) == (mode != POST)
        alike += [t for t in (a, b) if t is not None]
    if not (sized and rstd.shape == (norms, c.rows) and rstd.dtype is _F32 and rstd.is_contiguous() and rstd.get_device() == like.get_device()
            and all([t.shape == like.shape and t.dtype is like.dtype and t.get_device() == like.get_device() for t in alike])):
        raise ValueError("norm_backward: these are not what a call of this form kept")
    if any([wanted and t is None for wanted, t in zip(_asked(need), (y, like if mode != POST else None, w1, w2, gate, scale))]):
        raise ValueError("norm_backward: a gradient of an operand that the call does not have")
    return c


def operator_backward(dout, dh, w1, w2, gate, scale, rstd, a, b, number, mode, checkpoint, need):
    """torch.ops.bshmem.norm_backward: gradients of y, x, w1, w2, gate and scale; what the bits of `need` do not ask for is empty."""
    c = _whole_gradients(dout, dh, w1, w2, gate, scale, rstd, a, b, number, mode, checkpoint, need)
    with torch.cuda.device(rstd.device):
        found = _gradients((mode, c.what, c.n, c.rows, c.kind, _bits(number)), _asked(need), (w1, w2, gate, scale, rstd, a, b), dout, dh)
    return tuple(rstd.new_empty(0) if not wanted else g.clone() if g is dout else g for g, wanted in zip(found, _asked(need)))


def operator_backward_fake(dout, dh, w1, w2, gate, scale, rstd, a, b, number, mode, checkpoint, need):
    c = _whole_gradients(dout, dh, w1, w2, gate, scale, rstd, a, b, number, mode, checkpoint, need)
    return tuple(_new_like(t, memory_format=_CONTIGUOUS) if wanted else rstd.new_empty(0) for t, wanted in zip((c.like, c.like, w1, w2, gate, scale), _asked(need)))


def _run(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint):
    if not direct(name, y, x, w1, w2, gate, scale):
        return _registered(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint)
    c = _Call(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint)
    if not on_current_device(x):
        with torch.cuda.device(x.device):
            return _run(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint)
    if torch.is_grad_enabled() and any([t.requires_grad for t in (x, y, w1, w2, gate, c.scale) if t is not None]):
        return _NormFn.apply(y, x, w1, w2, gate, c.scale, c, mode)
    out, h, _, _ = _forward(c, mode, False)
    return (out, h) if mode == POST_PRE else out if mode == POST else h


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6, *, checkpoint: bool = False) -> torch.Tensor:
    """weight * x / sqrt(mean(x^2) + eps) over the last dimension."""
    return _run("rms_norm", PRE, None, x, None, weight, None, None, eps, checkpoint)


def post_norm(y: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, *, gate: Optional[torch.Tensor] = None,
              scale: Union[None, float, torch.Tensor] = None, eps: float = 1e-6, checkpoint: bool = False) -> torch.Tensor:
    """residual + scale * gate * weight * y / sqrt(mean(y^2) + eps)."""
    return _run("post_norm", POST, y, residual, weight, None, gate, scale, eps, checkpoint)


def post_pre_norm(y: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, next_weight: Optional[torch.Tensor] = None, *,
                  gate: Optional[torch.Tensor] = None, scale: Union[None, float, torch.Tensor] = None, eps: float = 1e-6,
                  checkpoint: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, h): ``post_norm`` and the next block's ``rms_norm(out, next_weight)`` in one pass."""
    return _run("post_pre_norm", POST_PRE, y, residual, weight, next_weight, gate, scale, eps, checkpoint)


class RMSNorm(torch.nn.Module):
    """``rms_norm`` with a learned weight."""

    def __init__(self, hidden: int, eps: float = 1e-6, device=None, dtype: torch.dtype = torch.bfloat16, checkpoint: bool = False):
        super().__init__()
        self.eps, self.checkpoint = eps, checkpoint
        self.weight = torch.nn.Parameter(torch.ones((hidden,), dtype=dtype, device=device))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return rms_norm(x, self.weight, self.eps, checkpoint=self.checkpoint)
