"""Whether a call may hand the addresses of its tensors to a kernel.

The layers' calls skip torch's dispatcher, which costs more than many of their kernels.  That is right for plain tensors that nobody watches;
fake tensors, tracing, transforms and modes that see operators get the registered operators of ``torch_ops``, with their fake
implementations and autograd formulas."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.utils._device import DeviceContext

from .. import _native

_PLAIN = (torch.Tensor, torch.nn.Parameter)
_compiling = torch.compiler.is_compiling
_dispatch_modes, _function_modes, _function_mode = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack, torch._C._get_function_stack_at
_batch = torch._C._functorch.is_legacy_batchedtensor
_transformed, _traced = torch._C._are_functorch_transforms_active, torch._C._is_tracing


def _unwatched() -> bool:
    """Nobody watches or rewrites operators: no compilation or tracing, no dispatch or function mode (fake tensors, make_fx,
    counters; the one of a default device only adds an argument to factories), no functorch transform (vmap, grad, jvp)."""
    if _compiling() or _dispatch_modes() or _transformed() or _traced():     # compilation first: nothing of the rest can be compiled
        return False
    modes = _function_modes()
    return not modes or modes == 1 and type(_function_mode(0)) is DeviceContext


def _first_plain(*operands) -> bool:
    """`plain` until the extension module is there: True if direct() is without looking further (see csrc/host/pycall.cc)."""
    global plain
    native = _native._pycall()
    native.watch((torch.Tensor, type(None), torch.nn.Parameter, float, int), (_dispatch_modes, _function_modes, _transformed, _traced), vars(forward_ad),
                 "_current_level")
    plain = native.plain
    return plain(*operands)


plain = _first_plain


def direct(what: str, *operands) -> bool:
    """Whether the kernels may read `operands` (tensors, and whatever else a call has) where they lie; False: through the registered operator.
    There is no forward-mode derivative, so an operand with a tangent is refused."""
    if _compiling():
        return False
    if plain(*operands):
        return True
    if forward_ad._current_level >= 0:
        for t in operands:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")
    return all([type(t) in _PLAIN for t in operands if isinstance(t, torch.Tensor)]) and _unwatched()


def direct_gradients(what: str, *grads) -> bool:
    """The same for the gradients that a backward pass gets, which may also be batches (``is_grads_batched``)."""
    if not direct(what, *grads):
        return False
    for g in grads:
        if g is not None and _batch(g):
            return False
    return True
