"""Linear layers with weights of 4 bits: ``out = x @ w.T``, w[n, k] = (q[n, k] - z) * s with one bf16 scale s, and optionally one zero
point z of 4 bits, per row and group of columns.

Few tokens (a decode step) run on a kernel that streams the 4 bits and multiplies them as they are; with many the weights are
widened to bf16 once and the bf16 tcgen05 GEMM takes them.  That GEMM wants a number of rows that is a multiple of 8: weights with another
stay on the first kernel, which reads them again for every 64 tokens (32 in groups of 32).  Traced, compiled, fake and watched calls are the registered operators
``torch.ops.bshmem.linear_w4``, ``widen_w4`` and ``quantize_w4``; there is no derivative of either mode.  The reference contains no GEMM, so there
is no parity citation.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _native
from .checkpoint8 import block_lib, on_current_device
from .gemm import current_stream, gemm_bf16, gemm_error_site
from .watched import direct

_U8, _BF16 = torch.uint8, torch.bfloat16


def few_tokens(group: int) -> int:
    """Tokens up to which the weights are multiplied as they are.  us, that kernel against widening and the bf16 GEMM, 8192 to 7168 columns,
    groups of 128: 64 tokens 23.2 / 56.6, 128 41.2 / 58.7, 192 72.6 / 63.0; 14336 to 4096, groups of 64: 128 47.0 / 58.2, 192 78.5 / 62.6.
    Groups of 32 have four accumulators for every 128 columns, so 32 tokens are a tile: 4096 to 14336, 33 tokens 60.5 / 54.3."""
    return 128 if group >= 64 else 32


_declared = False
_few = _widen = None


def _lib() -> C.CDLL:
    global _declared, _few, _widen
    lib = block_lib()
    if not _declared:
        VP, I, L = C.c_void_p, C.c_int, C.c_longlong
        lib.bshmem_w4_last_error.restype = C.c_char_p
        lib.bshmem_w4_few.restype = I
        lib.bshmem_w4_few.argtypes = [VP, L, VP, VP, VP, VP, I, I, I, I, VP, I]
        lib.bshmem_w4_error_site.restype = I
        lib.bshmem_w4_error_site.argtypes = [I]
        lib.bshmem_w4_widen.restype = I
        lib.bshmem_w4_widen.argtypes = [VP, VP, VP, VP, I, I, I, VP]
        lib.bshmem_w4_quant.restype = I
        lib.bshmem_w4_quant.argtypes = [VP, L, VP, VP, VP, I, I, I, VP]
        _widen, _few = _native.fast(lib, "bshmem_w4_widen"), _native.fast(lib, "bshmem_w4_few")
        _declared = True
    return lib


def _check(st: int, what: str) -> None:
    if st != 0:
        raise RuntimeError(f"{what} failed ({st}): {_lib().bshmem_w4_last_error().decode()}")


@dataclass
class W4Tensor:
    """A [N, K] weight in 4 bits: ``q`` [N, K/2] bytes (the column of even number in the low half), ``scales`` [N, K/group] bf16 and
    ``zeros`` [N, K/group] bytes 0..15, or None for 8 everywhere.  Groups have 32, 64 or a multiple of 128 columns."""
    q: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor] = None

    @property
    def group(self) -> int:
        return 2 * self.q.shape[1] // max(1, self.scales.shape[1])

    def dequantize(self) -> torch.Tensor:
        """fp32 [N, K] (for tests and reference computations)."""
        q = torch.stack((self.q & 15, self.q >> 4), dim=2).flatten(1).float()
        z = 8.0 if self.zeros is None else self.zeros.float().repeat_interleave(self.group, dim=1)
        return (q - z) * self.scales.float().repeat_interleave(self.group, dim=1)


def _checked(w: W4Tensor, what: str, addressed: bool = True) -> tuple[int, int, int]:
    """N, K and group of `w`.  Not `addressed`: it is not for a kernel of this call."""
    q, s, z = w.q, w.scales, w.zeros
    if not (q.dtype is _U8 and s.dtype is _BF16 and q.is_cuda and (z is None or z.dtype is _U8)):
        raise ValueError(f"{what} needs CUDA tensors q (uint8), scales (bf16) and zeros (uint8 or None)")
    qs, ss = q.shape, s.shape
    if len(qs) != 2 or len(ss) != 2 or qs[0] != ss[0] or ss[1] < 1 or (z is not None and z.shape != ss):
        raise ValueError(f"{what}: shapes do not belong together: q {tuple(qs)}, scales {tuple(ss)}")
    N, K = qs[0], 2 * qs[1]
    group = K // ss[1]
    if N < 1 or group * ss[1] != K or not (group in (32, 64) or (group and group % 128 == 0)) or K > 1 << 24:
        raise ValueError(f"{what} needs whole groups of 32, 64 or a multiple of 128 columns, got K {K} in {ss[1]} groups")
    if s.get_device() != q.get_device() or (z is not None and z.get_device() != q.get_device()):
        raise ValueError(f"{what}: q, scales and zeros must be on one device")
    if not (q.is_contiguous() and s.is_contiguous() and (z is None or z.is_contiguous())) or (addressed and q.data_ptr() % 16):
        raise ValueError(f"{what} needs contiguous tensors and q on a 16-byte boundary")
    return N, K, group


def _check_weight(w: torch.Tensor, group: int) -> None:
    if not w.is_cuda or w.dtype is not torch.bfloat16 or w.dim() != 2 or w.stride(1) != 1:
        raise ValueError("quantize_w4 needs a K-major bf16 CUDA matrix")
    N, K = w.shape
    if N < 1 or not (group in (32, 64) or (group > 0 and group % 128 == 0)) or K < group or K % group:
        raise ValueError(f"quantize_w4 needs rows of whole groups of 32, 64 or a multiple of 128 columns, got K {K}, group {group}")


def quantize_w4(w: torch.Tensor, group: int = 128, *, zeros: bool = False) -> W4Tensor:
    """bf16 [N, K] → 4 bits.  Without zero points a group's scale is (largest magnitude) / 7; with them (largest - smallest) / 15, of a range
    that holds zero; both rounded to bf16, and every value goes to the nearest that they can say.  A group with an infinity or a NaN becomes NaN."""
    if not direct("quantize_w4", w):
        q, s, z = _operators().quantize_w4(w, group, zeros)
        return W4Tensor(q, s, z if zeros else None)
    return quantize_direct(w, group, zeros)


def quantize_direct(w: torch.Tensor, group: int, zeros: bool) -> W4Tensor:
    _check_weight(w, group)
    if not on_current_device(w):
        with torch.cuda.device(w.device):
            return quantize_direct(w, group, zeros)
    N, K = w.shape
    lib = _lib()
    q = torch.empty((N, K // 2), dtype=torch.uint8, device=w.device)
    s = torch.empty((N, K // group), dtype=torch.bfloat16, device=w.device)
    z = torch.empty((N, K // group), dtype=torch.uint8, device=w.device) if zeros else None
    _check(lib.bshmem_w4_quant(w.data_ptr(), w.stride(0), q.data_ptr(), s.data_ptr(), 0 if z is None else z.data_ptr(), N, K, group,
                               current_stream()), "quantize_w4")
    return W4Tensor(q, s, z)


def widen_w4(w: W4Tensor) -> torch.Tensor:
    """The weight in bf16 [N, K], each value rounded once."""
    if not direct("widen_w4", w.q, w.scales, w.zeros):
        return _operators().widen_w4(w.q, w.scales, w.zeros)
    return widen_direct(w)


def widen_direct(w: W4Tensor) -> torch.Tensor:
    N, K, group = _checked(w, "widen_w4")
    if not on_current_device(w.q):
        with torch.cuda.device(w.q.device):
            return widen_direct(w)
    if _widen is None:
        _lib()
    out = torch.empty((N, K), dtype=torch.bfloat16, device=w.q.device)
    _check(_widen(w.q.data_ptr(), w.scales.data_ptr(), 0 if w.zeros is None else w.zeros.data_ptr(), out.data_ptr(), N, K, group,
                  current_stream()), "widen_w4")
    return out


def linear_w4(x: torch.Tensor, w: W4Tensor) -> torch.Tensor:
    """x [..., K] bf16 times the weight [N, K] of 4 bits, in bf16 [..., N] (forward only).

    Up to ``few_tokens(group)`` tokens, and for any number if N is no multiple of 8, the products are those of the weight as it stands, with sums in
    fp32.  Beyond, every weight is rounded to bf16 first, half a step (2^-8 of it) at most, as a layer that keeps its weights in bf16 has
    them: relative to the exact product's norm the result is off by 2.2e-3 then, 1.7e-3 (its own rounding to bf16) without.  So a token's
    result may differ with the number of tokens beside it.  2000 tokens, 4096 to 14340 columns, on the first kernel: 641 us in groups of 128 and 1270 in
    groups of 32, where 14336 columns take 184 and 209.

    A kernel whose bounded wait runs out leaves its result unfinished and says so on request: ``w4_error_site``, ``gemm_error_site`` (many
    tokens), or ``LinearW4.check``, which asks both."""
    if direct("linear_w4", x, w.q, w.scales, w.zeros):
        return linear_direct(x, w)
    _check_x(x, w, _checked(w, "linear_w4", False)[1])
    return _operators().linear_w4(x, w.q, w.scales, w.zeros)


def _check_x(x: torch.Tensor, w: W4Tensor, K: int) -> None:
    shape = x.shape
    if x.dtype is not _BF16 or not shape or shape[-1] != K or not x.is_cuda or x.get_device() != w.q.get_device():
        raise ValueError(f"linear_w4 needs bf16 [..., {K}] on {w.q.device}, got {x.dtype} {tuple(shape)} on {x.device}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("linear_w4 has no gradient: detach x, or call it under torch.no_grad()")


def linear_direct(x: torch.Tensor, w: W4Tensor) -> torch.Tensor:
    N, K, group = _checked(w, "linear_w4")
    shape = x.shape
    if x.dtype is not _BF16 or not shape or shape[-1] != K or x.get_device() != w.q.get_device() or x.requires_grad:
        _check_x(x, w, K)
    if not on_current_device(x):
        with torch.cuda.device(x.device):
            return linear_direct(x, w)
    m = x if len(shape) == 2 else x.reshape(-1, K)
    T = m.shape[0]
    ld, columns = m.stride()
    if T == 1:
        ld = K
    if columns != 1 or ld < K or ld % 8 or m.data_ptr() % 16:
        m = m.contiguous()
        if m.data_ptr() % 16:
            m = m.clone()
        ld = K
    if T > few_tokens(group) and N % 8 == 0:                 # the bf16 GEMM's columns come in eights
        out = gemm_bf16(m, widen_direct(w))
    else:
        if _few is None:
            _lib()
        out = m.new_empty((T, N))
        st = _few(m.data_ptr(), ld, w.q.data_ptr(), w.scales.data_ptr(), None if w.zeros is None else w.zeros.data_ptr(), out.data_ptr(), T, N, K,
                  group, current_stream(), 2000)
        if st != 0:
            _check(st, "linear_w4")
    return out if len(shape) == 2 else out.view(*shape[:-1], N)


# ---- registered operators: calls that somebody watches, traces or transforms ------------------------------------------------

def _operators():
    from . import torch_ops  # noqa: F401
    return torch.ops.bshmem


def operator_quantize(w, group, zeros):
    t = quantize_direct(w, group, zeros)
    return t.q, t.scales, t.q.new_empty((0,)) if t.zeros is None else t.zeros


def operator_quantize_fake(w, group, zeros):
    _check_weight(w, group)
    N, K = w.shape
    return (w.new_empty((N, K // 2), dtype=torch.uint8), w.new_empty((N, K // group)),
            w.new_empty((N, K // group) if zeros else (0,), dtype=torch.uint8))


def operator_widen_fake(q, scales, zeros):
    N, K, _ = _checked(W4Tensor(q, scales, zeros), "widen_w4", False)
    return scales.new_empty((N, K))


def operator_linear_fake(x, q, scales, zeros):
    w = W4Tensor(q, scales, zeros)
    N, K, _ = _checked(w, "linear_w4", False)
    _check_x(x, w, K)
    return x.new_empty((*x.shape[:-1], N))


def w4_error_site(clear: bool = True) -> int:
    """0 if no in-kernel bounded wait ran out since the last clear, else the site code."""
    return int(_lib().bshmem_w4_error_site(int(clear)))


class LinearW4(torch.nn.Module):
    """A linear layer (no bias) with a weight of 4 bits, for serving."""

    def __init__(self, weight: W4Tensor):
        super().__init__()
        N, K, _ = _checked(weight, "LinearW4", direct("LinearW4", weight.q, weight.scales, weight.zeros))
        self.in_features, self.out_features = K, N
        self.register_buffer("q", weight.q)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)

    @classmethod
    def from_linear(cls, layer: torch.nn.Module, group: int = 128, *, zeros: bool = False) -> "LinearW4":
        """The same layer in 4 bits; `layer` has a bf16 ``weight`` [out, in] and no bias."""
        if getattr(layer, "bias", None) is not None:
            raise ValueError("LinearW4 has no bias")
        return cls(quantize_w4(layer.weight.detach(), group, zeros=zeros))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear_w4(x, W4Tensor(self.q, self.scales, self.zeros))

    def check(self) -> None:
        """Raises if an in-kernel wait of the products on this device ran out since the last check; synchronises."""
        with torch.cuda.device(self.q.device):
            site = w4_error_site() or gemm_error_site()
        if site:
            raise RuntimeError(f"a bounded in-kernel wait ran out (site {site})")
