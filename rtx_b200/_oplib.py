"""Operator registration for the `rtx::` custom ops.

`torch.library.custom_op` wraps every call of the device implementation in several Python layers (an
aliasing check, a compile-disable frame, an autograd trampoline even for ops without a backward): tens of
microseconds per call, more than a whole decode step takes on the device.  The ops here are declared with
the dispatcher directly instead — same inferred schema, same `pt2_compliant` tag, fake and autograd
registrations through the same `torch.library` functions — so an eager call costs one dispatch.
The returned handle offers the part of the `custom_op` object's interface the package uses.
"""

from __future__ import annotations

from typing import Callable, Optional

import torch
from torch.autograd import forward_ad

_LIB = torch.library.Library("rtx", "FRAGMENT")


# bound once: these stand on the launch path of calls that take 15 microseconds in all
_is_compiling = torch.compiler.is_compiling
_transforms_active = torch._C._are_functorch_transforms_active
_dispatch_modes = torch._C._len_torch_dispatch_stack
_is_tracing = torch._C._is_tracing
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))


def interposed() -> bool:
    """Whether something has to see an op's call before the CUDA implementation runs: `torch.compile`, a `torch.func`
    transform, a dispatch mode (`make_fx`, a FLOP counter, a checkpointing policy, fake tensors) or `torch.jit.trace`.  A
    launcher that is called past them writes through an address they know nothing of, and a graph they record lacks it."""
    return bool(_is_compiling() or _dispatch_modes() or _transforms_active() or _is_tracing())


def eager(t: torch.Tensor, *others) -> bool:
    """Whether an op on these operands would only be dispatched back into this package's CUDA implementation (plain CUDA
    tensors, nothing interposed): the package's own functions then call the launcher itself and save a dispatch of a few
    microseconds.  What is no tensor is the launcher's to refuse."""
    if not t.is_cuda or _is_compiling() or _dispatch_modes() or _transforms_active() or _is_tracing():
        return False
    if type(t) not in _PLAIN:
        return False
    for operand in others:
        if type(operand) not in _PLAIN and isinstance(operand, torch.Tensor):
            return False
    return True


def transformed() -> bool:
    """Whether a `torch.func` transform is active that differentiates or batches an `autograd.Function` with a
    `setup_context`; a formula registered for an op cannot be differentiated there.  (`functionalize` is the other way
    round: it takes ops and no such functions.)"""
    if _is_compiling() or not _transforms_active():
        return False
    levels = torch._C._functorch.get_interpreter_stack() or ()
    return all(level.key() != torch._C._functorch.TransformType.Functionalize for level in levels)


class _Once(torch.autograd.Function):
    generate_vmap_rule = True

    @staticmethod
    def forward(op, message, *args):
        return op(*args)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.message = inputs[1]

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError(ctx.message)


def call_without_derivative(op: "OpHandle", message: str, *args):
    """An op that has no derivative: `torch.func` transforms that ask for one get the error `message`, where the bare op
    would give zeros."""
    return _Once.apply(op, message, *args) if transformed() else op(*args)


def call_detached(op: "OpHandle", message: str, *args):
    """The same for a function whose results carry no gradient, whatever its operands: as in an eager call, also where a
    graph is recorded."""
    if transformed():
        return _Once.apply(op, message, *args)
    return op(*(a.detach() if isinstance(a, torch.Tensor) else a for a in args))


def refuse_tangents(name: str, *tensors) -> None:
    """Forward-mode differentiation of an op without a formula for it would drop the tangents: refuse it.  (A tangent below
    a `vmap` cannot be looked at; the graph nodes of `torch.func` transforms refuse it where the batch is unpacked.)"""
    if forward_ad._current_level >= 0 and not _is_compiling():
        for t in tensors:
            if isinstance(t, torch.Tensor) and not torch._C._functorch.is_batchedtensor(t):
                if forward_ad.unpack_dual(t).tangent is not None:
                    raise NotImplementedError(f"{name} has no forward-mode derivative")


def no_tangents(name: str) -> Callable:
    """The `jvp` of a graph node without one."""
    def jvp(ctx, *tangents):
        raise NotImplementedError(f"{name} has no forward-mode derivative")

    return jvp


class OpHandle:
    """Callable handle of one registered op (`torch.ops.rtx.<name>.default`)."""

    def __init__(self, qualname: str, fn: Callable):
        namespace, name = qualname.split("::")
        self.qualname = qualname
        self.fn = fn                                  # the device implementation, for direct in-package calls
        self.overload = getattr(getattr(torch.ops, namespace), name).default
        self.__name__ = getattr(fn, "__name__", name)
        self.__doc__ = fn.__doc__

    def __call__(self, *args, **kwargs):
        return self.overload(*args, **kwargs)

    def register_fake(self, fn: Callable) -> Callable:
        torch.library.register_fake(self.qualname, fn, lib=_LIB)
        return fn

    def refuse_derivative(self, message: str) -> None:
        """Differentiating the op raises, where an op without a formula would warn and give zeros."""
        def backward(ctx, *grads):
            raise NotImplementedError(message)

        self.register_autograd(backward)

    def register_autograd(self, backward: Callable, *, setup_context: Optional[Callable] = None) -> None:
        torch.library.register_autograd(self.qualname, backward, setup_context=setup_context, lib=_LIB)


def custom_op(qualname: str, *, mutates_args=(), device_types: str = "cuda") -> Callable[[Callable], OpHandle]:
    """Decorator with the call signature of `torch.library.custom_op` (schema inferred from the annotations)."""
    if device_types != "cuda":
        raise ValueError("the rtx:: ops have CUDA implementations only")

    def register(fn: Callable) -> OpHandle:
        schema = torch.library.infer_schema(fn, mutates_args=mutates_args)
        torch.library.define(qualname, schema, lib=_LIB, tags=(torch.Tag.pt2_compliant_tag,))
        torch.library.impl(qualname, "CUDA", fn, lib=_LIB)
        return OpHandle(qualname, fn)

    return register
