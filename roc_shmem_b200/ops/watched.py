"""Whether a call may hand the addresses of its tensors to a kernel.

The layers' calls skip torch's dispatcher, which costs more than many of their kernels.  That is right for plain tensors that nobody watches;
fake tensors, tracing, transforms and modes that see operators get the registered operators of ``torch_ops``, with their fake
implementations and autograd formulas."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.utils._device import DeviceContext

_PLAIN = (torch.Tensor, torch.nn.Parameter)
_DIRECT = frozenset((*_PLAIN, type(None), float, int))


def _unwatched() -> bool:
    """Nobody watches or rewrites operators: no compilation or tracing, no dispatch or function mode (fake tensors, make_fx,
    counters; the one of a default device only adds an argument to factories), no functorch transform (vmap, grad, jvp)."""
    if torch.compiler.is_compiling():                    # first: nothing of the rest can be compiled
        return False
    C = torch._C
    modes = C._len_torch_function_stack()
    return (C._len_torch_dispatch_stack() == 0 and C._functorch.peek_interpreter_stack() is None and C._get_tracing_state() is None
            and (modes == 0 or modes == 1 and type(C._get_function_stack_at(0)) is DeviceContext))


def direct(what: str, *operands) -> bool:
    """Whether the kernels may read `operands` (tensors, numbers, None) where they lie; False: through the registered operator.
    There is no forward-mode derivative, so an operand with a tangent is refused."""
    if torch.compiler.is_compiling():
        return False
    if forward_ad._current_level >= 0:
        for t in operands:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")
    return _DIRECT.issuperset(map(type, operands)) and _unwatched()


def direct_gradients(what: str, *grads) -> bool:
    """The same for the gradients that a backward pass gets, which may also be batches (``is_grads_batched``)."""
    batched = torch._C._functorch.is_legacy_batchedtensor
    return direct(what, *grads) and not any([batched(g) for g in grads if g is not None])
