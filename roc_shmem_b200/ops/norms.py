"""RMS norms before and after a block, fused with the block's gate, its residual scale and the residual sum.

    rms_norm       h   = weight * n(x)                                     n(v) = v / sqrt(mean(v^2) + eps) over the last dimension
    post_norm      out = residual + scale * gate * weight * n(y)           y: what the block returned
    post_pre_norm  both in one pass: out, and the next block's h = next_weight * n(out)

Rows are bf16, fp16 or fp32, sums fp32.  A weight is one value per column, of the rows' type or fp32; the gate one per column
``[H]``, per row ``[..., 1]`` or per element (weights and gates may be left out); the scale a number or a tensor with one
element.  Every tensor has a gradient; sums over rows are added in a fixed order, so a call gives the same bits again.
``checkpoint=True`` keeps the norms' inputs for the backward pass in 8 bits (``checkpoint8``): the gradients are then those at the
kept values.  Rows have 1 to 16384 columns and may be apart (any stride of the leading dimension); rows of a multiple of 8 columns on
16-byte boundaries are the fast ones.  Squares are fp32: rows whose squares leave its range give what that gives.

The reference is a communication runtime without models, so there is no parity citation.
"""
from __future__ import annotations

import ctypes as C
import struct
from functools import lru_cache
from typing import Optional, Union

import torch

from .. import _native
from .checkpoint8 import _TYPES, _empty_kept, block_lib, on_current_device
from .gemm import current_stream

PRE, POST, POST_PRE = range(3)
NO_GATE, COLUMN, ROW, ELEMENT = range(4)
MAX_COLUMNS = 16384
_declared = False
_fwd = _bwd = _groups = _finish = None


def _lib() -> C.CDLL:
    global _declared, _fwd, _bwd, _groups, _finish
    lib = block_lib()
    if not _declared:
        VP, I, L, U = C.c_void_p, C.c_int, C.c_longlong, C.c_uint64
        lib.bshmem_norm_last_error.restype = C.c_char_p
        lib.bshmem_norm_fwd.restype = I
        lib.bshmem_norm_fwd.argtypes = [I, VP, L, VP, L, VP, VP, VP, VP, VP, L, VP, U, VP, VP, VP, L, I, VP]
        lib.bshmem_norm_bwd.restype = I
        lib.bshmem_norm_bwd.argtypes = [I, VP, VP, VP, L, VP, L, VP, VP, VP, L, VP, U, VP, VP, VP, VP, VP, VP, VP, L, I, VP]
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


def _p(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _matrix(t: torch.Tensor, cols: int) -> torch.Tensor:
    m = t if t.dim() == 2 else t.reshape(-1, cols)
    return m if m.stride(1) == 1 or cols == 1 else m.contiguous()


class _Call:
    """A call's operands, checked: what they are in one word, and their addresses and pitches."""
    __slots__ = ("what", "y", "x", "w1", "w2", "gate", "scale", "number", "eps", "rows", "n", "shape", "dtype", "device", "gate_ld", "kind")

    def __init__(self, name, mode, y, x, w1, w2, gate, scale, eps, checkpoint):
        dt = x.dtype
        kind = _TYPES.get(dt)
        if kind is None or not x.is_cuda:
            raise ValueError(f"{name} needs bf16, fp16 or fp32 CUDA tensors, got {dt} on {x.device}")
        shape = x.shape
        if len(shape) < 1 or not 1 <= shape[-1] <= MAX_COLUMNS:
            raise ValueError(f"{name} needs rows of 1 to {MAX_COLUMNS} columns, got {tuple(shape)}")
        if not eps > 0:
            raise ValueError(f"{name} needs eps > 0")
        n, dev = shape[-1], x.device
        what = kind | mode << 2 | (checkpoint << 12)
        self.eps, self.n, self.shape, self.dtype, self.device, self.kind = float(eps), n, shape, dt, dev, NO_GATE
        self.x, self.y = _matrix(x, n), None
        self.rows = self.x.shape[0]
        if self.rows > 0x7fffffff:
            raise ValueError(f"{name} takes less than 2^31 rows")

        def vector(t, label, bit):
            nonlocal what
            if t is None:
                return None
            if t.shape != (n,) or t.device != dev or (t.dtype is not dt and t.dtype is not torch.float32):
                raise ValueError(f"{name}: {label} must be {dt} or fp32 of shape ({n},) on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
            if t.dtype is torch.float32:
                what |= 1 << bit
            return t if t.stride(0) == 1 else t.contiguous()
        self.w1, self.w2 = vector(w1, "weight", 8), vector(w2, "weight" if mode == PRE else "next_weight", 9)
        self.gate, self.gate_ld, self.scale, self.number = None, 0, None, 1.0
        if mode != PRE:
            if y.shape != shape or y.dtype is not dt or y.device != dev:
                raise ValueError(f"{name}: y and residual must be alike, got {y.dtype} {tuple(y.shape)} on {y.device} and {dt} {tuple(shape)} on {dev}")
            self.y = _matrix(y, n)
            if gate is not None:
                if gate.shape == (n,):
                    self.kind, self.gate = COLUMN, vector(gate, "gate", 10)
                else:
                    if gate.device != dev or (gate.dtype is not dt and gate.dtype is not torch.float32):
                        raise ValueError(f"{name}: gate must be {dt} or fp32 on {dev}, got {gate.dtype} on {gate.device}")
                    if gate.shape == shape:
                        self.kind, self.gate = ELEMENT, _matrix(gate, n)
                    elif gate.shape == (*shape[:-1], 1):
                        self.kind, self.gate = ROW, _matrix(gate, 1)
                    else:
                        raise ValueError(f"{name}: gate must be ({n},), {(*shape[:-1], 1)} or {tuple(shape)}, got {tuple(gate.shape)}")
                    if gate.dtype is torch.float32:
                        what |= 1 << 10
                    self.gate_ld = self.gate.stride(0)
            if isinstance(scale, torch.Tensor):
                if scale.numel() != 1 or scale.device != dev or (scale.dtype is not dt and scale.dtype is not torch.float32):
                    raise ValueError(f"{name}: scale must be a number or one element of {dt} or fp32 on {dev}")
                self.scale = scale
                if scale.dtype is torch.float32:
                    what |= 1 << 11
            elif scale is not None:
                self.number = float(scale)
        self.what = what | self.kind << 4


def _forward(c: _Call, mode: int, train: bool):
    """(out, h, rstd, q, e); what the call does not give is None."""
    if _fwd is None:
        _lib()
    rows, n = c.rows, c.n
    out = torch.empty(c.shape, dtype=c.dtype, device=c.device) if mode != PRE else None
    h = torch.empty(c.shape, dtype=c.dtype, device=c.device) if mode != POST else None
    rstd = q = e = None
    if train:
        norms = 2 if mode == POST_PRE else 1
        rstd = torch.empty((norms, rows), dtype=torch.float32, device=c.device)
        if c.what >> 12 & 1:
            q, e = _empty_kept(rows, n, c.device, norms)
    what = c.what if q is not None else c.what & ~(1 << 12)
    y = c.y
    _check(_fwd(what, _p(y), 0 if y is None else y.stride(0), c.x.data_ptr(), c.x.stride(0), _p(out), _p(h), _p(c.w1), _p(c.w2), _p(c.gate),
                c.gate_ld, _p(c.scale), _bits(c.eps) | _bits(c.number) << 32, _p(rstd), _p(q), _p(e), rows, n, current_stream()), "norm")
    return out, h, rstd, q, e


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, w1, w2, gate, scale, c, mode):
        ctx.set_materialize_grads(False)
        out, h, rstd, q, e = _forward(c, mode, True)
        ctx.mode, ctx.what, ctx.n, ctx.rows, ctx.number, ctx.kind = mode, c.what, c.n, c.rows, c.number, c.kind
        ctx.gate_shape = None if gate is None else gate.shape
        z = x if mode == PRE else out
        kept = (q, e) if q is not None else (y if mode != PRE else None, z if mode != POST else None)
        ctx.save_for_backward(w1, w2, gate, scale, rstd, *kept)
        return (out, h) if mode == POST_PRE else out if mode == POST else h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        w1, w2, gate, scale, rstd, a, b = ctx.saved_tensors
        need_y, need_x, need_w1, need_w2, need_gate, need_scale = ctx.needs_input_grad[:6]
        mode, what, n, rows = ctx.mode, ctx.what, ctx.n, ctx.rows
        dout = grads[0] if mode != PRE else None
        dh = grads[-1] if mode != POST else None
        if dout is None and dh is None:
            return (None,) * 8
        given = dout if dout is not None else dh
        shape, dt, dev = given.shape, given.dtype, given.device
        dw_next = None
        if mode == POST_PRE and dh is None:                 # nobody used h: the first norm alone
            mode, what = POST, what & ~(3 << 2) | POST << 2
            dw_next = torch.zeros_like(w2) if need_w2 else None
            need_w2 = False
        if rows == 0:
            new = [None if not need else torch.zeros(s, dtype=t, device=dev) for need, s, t in (
                (need_y, shape, dt), (need_x, shape, dt), (need_w1, (n,), w1 is not None and w1.dtype), (need_w2, (n,), w2 is not None and w2.dtype),
                (need_gate, ctx.gate_shape, gate is not None and gate.dtype), (need_scale, scale is not None and scale.shape, scale is not None and scale.dtype))]
            if dw_next is not None:
                new[3] = dw_next
            return (*new, None, None)

        def flat(g):
            return None if g is None else g.contiguous()
        dout, dh = flat(dout), flat(dh)
        kept8 = what >> 12 & 1
        y = z = None
        if not kept8:
            y = None if a is None else _matrix(a, n)
            z = None if b is None else _matrix(b, n)
        new = torch.empty
        dz = new(shape, dtype=dt, device=dev) if mode != POST else dout
        dy = new(shape, dtype=dt, device=dev) if need_y and mode != PRE else None
        dgate = torch.empty(ctx.gate_shape, dtype=gate.dtype, device=dev) if need_gate else None
        column = ctx.kind == COLUMN
        gate_m = gate if gate is None or column else _matrix(gate, 1 if ctx.kind == ROW else n)
        if column and gate_m.stride(0) != 1:
            gate_m = gate_m.contiguous()
        w1 = None if w1 is None else w1.contiguous()
        w2 = None if w2 is None else w2.contiguous()
        sums = need_w1 or need_w2 or need_scale or (need_gate and column)
        work = None
        if sums:
            groups = _groups(rows, n)
            if groups < 1:
                _check(-groups, "norm backward")
            work = new((groups * ((n + 7) // 8 * 8 * (2 if mode == POST_PRE else 1) + 1),), dtype=torch.float32, device=dev)
        stream, number = current_stream(), _bits(ctx.number)
        ld = 0 if gate_m is None or column else gate_m.stride(0)
        if mode != POST or dy is not None or sums or dgate is not None:
            _check(_bwd(what, _p(dout), _p(dh), _p(z), 0 if z is None else z.stride(0), _p(y), 0 if y is None else y.stride(0), _p(w1), _p(w2),
                        _p(gate_m), ld, _p(scale), number, rstd.data_ptr(), _p(a) if kept8 else 0, _p(b) if kept8 else 0,
                        _p(dz) if mode != POST else 0, _p(dy), 0 if column else _p(dgate), _p(work), rows, n, stream), "norm backward")
        dw1 = dw2 = dscale = None
        if sums:
            dw1 = torch.empty_like(w1) if need_w1 else None
            dw2 = torch.empty_like(w2) if need_w2 else None
            dscale = torch.empty_like(scale) if need_scale else None
            _check(_finish(what, work.data_ptr(), _p(w1), _p(gate_m) if column else 0, _p(scale), number, _p(dw1), _p(dw2),
                           _p(dgate) if column else 0, _p(dscale), rows, n, stream), "norm backward")
        return dy, dz if need_x else None, dw1, dw2 if dw_next is None else dw_next, dgate, dscale, None, None


def _run(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint):
    c = _Call(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint)
    if not on_current_device(x):
        with torch.cuda.device(x.device):
            return _run(name, mode, y, x, w1, w2, gate, scale, eps, checkpoint)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, x, w1, w2, gate, c.scale)):
        return _NormFn.apply(y, x, w1, w2, gate, c.scale, c, mode)
    out, h = _forward(c, mode, False)[:2]
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
