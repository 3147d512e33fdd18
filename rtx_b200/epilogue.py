"""MXFP8 linear with bias, activation and residual in the GEMM's epilogue.

    z = q(x) q(w)^T + bias        y = act(z) + residual        one BF16 rounding of the FP32 result

Operand formats and gradient orientation as `mxfp8_linear` (whose modules are no-bias, rtx/fp8.py:2389).  Training keeps
z in BF16 (not at all for activation "none"); the backward forms dz = dy act'(z), rounds it to BF16 as the gradient
tensor between an activation and a linear would be, and quantizes it for dX and dW in the same pass that sums dbias.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import fp8 as _fp8
from . import ops
from ._oplib import (call_detached, call_without_derivative, custom_op, eager, no_tangents, refuse_tangents,
                     transformed)
from .formats import (PACKED_OPERAND_SCHEMA_VERSION, SCALE_LAYOUT_CODES, MXFP8Tensor, make_mxfp8_tensor,
                      mxfp8_kernel_operands, mxfp8_matrix_shape, mxfp8_qdata_2d, mxfp8_scales_for_kernel,
                      mxfp8_state_for_kernel, reject_packed_dtype_conversion)


_FROZEN = "a prequantized MXFP8 weight is inference-only; keep the BF16 master weight to train"


def _check(x, n, k, bias, residual, activation) -> None:
    ops.activation_code(activation)
    if x.dtype is not torch.bfloat16 or x.ndim != 2:
        raise TypeError(f"x must be BF16 [M, K], got {x.dtype} with {x.ndim} dimensions")
    if x.shape[1] != k:
        raise ValueError(f"K mismatch: x has {x.shape[1]}, weight has {k}")
    if n == 0 or k == 0:
        raise ValueError("N and K must be positive")
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError(f"bias must be [{n}]")
    if residual is not None and tuple(residual.shape) != (x.shape[0], n):
        raise ValueError(f"residual must be [{x.shape[0]}, {n}]")


@custom_op("rtx::mxfp8_linear_epilogue", mutates_args=(), device_types="cuda")
def mxfp8_linear_epilogue_op(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                             residual: Optional[torch.Tensor], activation: str) -> torch.Tensor:
    _check(x, *weight.shape, bias, residual, activation)
    return ops.mxfp8_linear_epilogue_fwd(x, weight.contiguous(), bias, residual, activation=activation)[0]


@mxfp8_linear_epilogue_op.register_fake
def _(x, weight, bias, residual, activation):
    return x.new_empty((x.shape[0], weight.shape[0]), dtype=torch.bfloat16)


@custom_op("rtx::mxfp8_linear_epilogue_prequant_w", mutates_args=(), device_types="cuda")
def mxfp8_linear_epilogue_prequant_w(x: torch.Tensor, weight_data: torch.Tensor, weight_scales: torch.Tensor,
                                     bias: Optional[torch.Tensor], residual: Optional[torch.Tensor], n: int, k: int,
                                     activation: str) -> torch.Tensor:
    _check(x, n, k, bias, residual, activation)
    return ops.mxfp8_linear_epilogue_fwd_prequant_w(x, weight_data, weight_scales, n, bias, residual, activation=activation)


@mxfp8_linear_epilogue_prequant_w.register_fake
def _(x, weight_data, weight_scales, bias, residual, n, k, activation):
    return x.new_empty((x.shape[0], n), dtype=torch.bfloat16)


@custom_op("rtx::mxfp8_linear_epilogue_fwd", mutates_args=(), device_types="cuda")
def mxfp8_linear_epilogue_fwd(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                              residual: Optional[torch.Tensor], activation: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, z): z is what the backward needs of the forward, empty for activation "none"."""
    _check(x, *weight.shape, bias, residual, activation)
    y, z = ops.mxfp8_linear_epilogue_fwd(x, weight.contiguous(), bias, residual, activation=activation,
                                         keep_z=activation != "none")
    return y, (z if z is not None else y.new_empty(0))


def _fake_fwd(x, weight, bias, residual, activation):
    y = x.new_empty((x.shape[0], weight.shape[0]), dtype=torch.bfloat16)
    return y, (torch.empty_like(y) if activation != "none" else y.new_empty(0))


mxfp8_linear_epilogue_fwd.register_fake(_fake_fwd)


@custom_op("rtx::mxfp8_linear_epilogue_train", mutates_args=(), device_types="cuda")
def mxfp8_linear_epilogue_train(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                                residual: Optional[torch.Tensor], activation: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """The differentiable op."""
    return mxfp8_linear_epilogue_fwd.fn(x, weight, bias, residual, activation)


mxfp8_linear_epilogue_train.register_fake(_fake_fwd)


@custom_op("rtx::mxfp8_linear_epilogue_bwd", mutates_args=(), device_types="cuda")
def mxfp8_linear_epilogue_bwd(grad_output: torch.Tensor, z: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                              activation: str, need_dx: bool, need_dw: bool,
                              need_dbias: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dX, dW, dbias); what is not needed is an empty tensor."""
    n, k = weight.shape
    _check(x, n, k, None, None, activation)
    if grad_output.dtype is not torch.bfloat16 or tuple(grad_output.shape) != (x.shape[0], n):
        raise ValueError(f"grad_output must be BF16 [{x.shape[0]}, {n}]")
    grads = ops.mxfp8_linear_epilogue_bwd(grad_output, z, x, weight.contiguous() if need_dx else None, k,
                                          activation=activation, need_dx=need_dx, need_dw=need_dw, need_dbias=need_dbias)
    return tuple(g if g is not None else x.new_empty(0) for g in grads)


@mxfp8_linear_epilogue_bwd.register_fake
def _(grad_output, z, x, weight, activation, need_dx, need_dw, need_dbias):
    new = x.new_empty
    return (new(x.shape) if need_dx else new(0), new(weight.shape) if need_dw else new(0),
            new((weight.shape[0],)) if need_dbias else new(0))


_TWICE = "the backward of mxfp8_linear_epilogue has no derivative of its own"
mxfp8_linear_epilogue_bwd.refuse_derivative(_TWICE)


def _train_setup(ctx, inputs, output):
    x, weight, _bias, _residual, activation = inputs
    _y, z = output
    ctx.save_for_backward(x, weight, z)
    ctx.activation = activation
    ctx.mark_non_differentiable(z)
    ctx.set_materialize_grads(False)


def _train_backward(ctx, grad_y, _grad_z):
    need_dx, need_dw, need_db, need_dr = ctx.needs_input_grad[:4]
    if grad_y is None or not (need_dx or need_dw or need_db):
        return None, None, None, grad_y if need_dr else None, None
    x, weight, z = ctx.saved_tensors
    if not eager(grad_y, x, weight, z):
        return _dispatched_backward(ctx, grad_y, None)
    weight = weight.contiguous() if need_dx else weight
    return (*ops.mxfp8_linear_epilogue_bwd(grad_y, z, x, weight, weight.shape[1], activation=ctx.activation, need_dx=need_dx,
                                           need_dw=need_dw, need_dbias=need_db), grad_y if need_dr else None, None)


def _dispatched_backward(ctx, grad_y, _grad_z):
    need_dx, need_dw, need_db, need_dr = ctx.needs_input_grad[:4]
    if grad_y is None or not (need_dx or need_dw or need_db):
        return None, None, None, grad_y if need_dr else None, None
    x, weight, z = ctx.saved_tensors
    dx, dw, db = call_without_derivative(mxfp8_linear_epilogue_bwd, _TWICE, grad_y, z, x, weight, ctx.activation, need_dx,
                                         need_dw, need_db)
    return (dx if need_dx else None, dw if need_dw else None, db if need_db else None, grad_y if need_dr else None, None)


mxfp8_linear_epilogue_train.register_autograd(_train_backward, setup_context=_train_setup)


class _LinearEpilogueFunction(torch.autograd.Function):
    """The same graph node for eager calls, without the host time of an op's registered autograd formula."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, z = mxfp8_linear_epilogue_fwd.fn(x, weight, bias, residual, activation)
        ctx.save_for_backward(x, weight, z)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        return _train_backward(ctx, grad_y, None)


class _TransformedLinearEpilogue(torch.autograd.Function):
    """The same node in the form that `torch.func` transforms take."""

    generate_vmap_rule = True

    @staticmethod
    def forward(x, weight, bias, residual, activation):
        return mxfp8_linear_epilogue_fwd(x, weight, bias, residual, activation)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _train_setup(ctx, inputs, output)
        ctx.save_for_forward(inputs[0], inputs[1], output[1])   # a batched `jvp` looks for them

    backward = staticmethod(_dispatched_backward)
    jvp = staticmethod(no_tangents("mxfp8_linear_epilogue"))


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def mxfp8_linear_epilogue(x: torch.Tensor, weight, bias: Optional[torch.Tensor] = None,
                          residual: Optional[torch.Tensor] = None, *, activation: str = "none") -> torch.Tensor:
    """act(x weight^T + bias) + residual with MXFP8 operands.

    x           BF16 [..., K]; leading dimensions are flattened and restored
    weight      BF16 [N, K] (quantized in the call; differentiable), or an `MXFP8Tensor` of that shape (inference)
    bias        BF16 [N] or None
    residual    BF16 [..., N], the shape of the result, or None
    activation  "none", "relu", "relu2" (max(z, 0)^2), "silu", "gelu" (erf) or "gelu_tanh"
    """
    if isinstance(weight, MXFP8Tensor):
        n, k = mxfp8_matrix_shape(weight)
        return _apply_packed(x, weight, n, k, bias, residual, activation)
    refuse_tangents("mxfp8_linear_epilogue", x, weight, bias, residual)
    n, k = weight.shape
    shape, x, residual = _matrices(x, residual, n, k)
    direct = eager(x, weight, bias, residual)
    if not direct and transformed():
        y = _TransformedLinearEpilogue.apply(x, weight, bias, residual, activation)[0]
    elif not _needs_grad(x, weight, bias, residual):
        y = (mxfp8_linear_epilogue_op.fn if direct else mxfp8_linear_epilogue_op)(x, weight, bias, residual, activation)
    elif direct:
        y = _LinearEpilogueFunction.apply(x, weight, bias, residual, activation)
    else:
        y = mxfp8_linear_epilogue_train(x, weight, bias, residual, activation)[0]
    return y if len(shape) == 2 else y.reshape(shape)


def _matrices(x, residual, n, k):
    """(shape of the result, x and residual as matrices)"""
    if x.ndim < 1 or x.shape[-1] != k:
        raise ValueError(f"K mismatch: x has {x.shape[-1] if x.ndim else 'no dimension'}, weight has {k}")
    shape = (*x.shape[:-1], n)
    if residual is not None:
        if tuple(residual.shape) != shape:
            raise ValueError(f"residual must have the result's shape {shape}, got {tuple(residual.shape)}")
        if residual.ndim != 2:
            residual = residual.reshape(-1, n)
    return shape, (x if x.ndim == 2 else x.reshape(-1, k)), residual


def _apply_packed(x, packed, n, k, bias, residual, activation):
    """`packed`: an MXFP8Tensor, or its (payload, scales) as the kernels take them"""
    refuse_tangents("mxfp8_linear_epilogue", x, bias, residual)
    shape, x, residual = _matrices(x, residual, n, k)
    if _needs_grad(x, bias, residual):
        raise RuntimeError(_FROZEN)
    data, scales = packed if isinstance(packed, tuple) else mxfp8_kernel_operands(packed)
    if eager(x, data, scales, bias, residual):
        y = ops.mxfp8_linear_epilogue_fwd_prequant_w(x, data, scales, n, bias, residual, activation=activation)
    else:
        y = call_without_derivative(mxfp8_linear_epilogue_prequant_w, _FROZEN, x, data, scales, bias, residual, n, k,
                                    activation)
    return y if len(shape) == 2 else y.reshape(shape)


def mxfp8_linear_epilogue_backward(grad_output: torch.Tensor, z: Optional[torch.Tensor], x: torch.Tensor,
                                   weight: torch.Tensor, *, activation: str = "none",
                                   bias: bool = True) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """BF16 (dX, dW, dbias) of `mxfp8_linear_epilogue`; `z` is the pre-activation in BF16 (None for activation "none"),
    `bias=False` leaves dbias out (None).  The residual's gradient is grad_output.  There is no FP32 dW for sums over ranks,
    as the dense linear's backward has one."""
    refuse_tangents("mxfp8_linear_epilogue_backward", grad_output, z, x, weight)
    n, k = weight.shape
    if activation != "none" and z is None:
        raise ValueError("an activation's backward needs the pre-activation z")
    for name, t, width in (("grad_output", grad_output, n), ("x", x, k), ("z", z if activation != "none" else None, n)):
        if t is not None and (t.ndim < 1 or t.shape[-1] != width):
            raise ValueError(f"{name} must have rows of {width} values, got shape {tuple(t.shape)}")
    z2d = z.reshape(-1, n).contiguous() if z is not None and activation != "none" else grad_output.new_empty(0)
    args = (grad_output.reshape(-1, n), z2d, x.reshape(-1, k), weight, activation, True, True, bias)
    if eager(x, grad_output, z2d, weight):
        dx, dw, db = mxfp8_linear_epilogue_bwd.fn(*args)
    else:
        dx, dw, db = call_detached(mxfp8_linear_epilogue_bwd, _TWICE, *args)
    return dx.reshape(x.shape), dw, db if bias else None


class MXFP8LinearEpilogue(nn.Module):
    """Linear with bias and activation, `forward(x, residual=None)`; parameters `weight` and `bias` in BF16 under
    nn.Linear's names.  `to_quantized_weight()` gives the inference copy with the weight packed."""

    __constants__ = ["in_features", "out_features", "activation", "weight_mode"]

    def __init__(self, in_features: int, out_features: int, bias: bool = True, *, activation: str = "none", device=None,
                 dtype: torch.dtype = torch.bfloat16, packed_weight=None) -> None:
        super().__init__()
        if dtype is not torch.bfloat16:
            raise TypeError(f"MXFP8LinearEpilogue parameters must be BF16, got {dtype}")
        ops.activation_code(activation)
        self.in_features, self.out_features, self.activation = int(in_features), int(out_features), activation
        self.weight_mode = "prequantized" if packed_weight is not None else "dynamic"
        if packed_weight is None:
            self.weight = nn.Parameter(torch.empty(self.out_features, self.in_features, device=device, dtype=torch.bfloat16))
        else:
            if mxfp8_matrix_shape(packed_weight) != (self.out_features, self.in_features):
                raise ValueError("packed weight does not have the module's shape")
            device = packed_weight.qdata.device
            self.register_parameter("weight", None)
            self.register_buffer("weight_data", mxfp8_qdata_2d(packed_weight).view(torch.uint8))
            self.register_buffer("weight_scales", mxfp8_scales_for_kernel(packed_weight))
            self.register_buffer("weight_packing_meta", torch.tensor(
                [PACKED_OPERAND_SCHEMA_VERSION, SCALE_LAYOUT_CODES["mma128"], self.in_features,
                 int(packed_weight.qdata.shape[-1])], dtype=torch.int64))
        if bias:
            self.bias = nn.Parameter(torch.zeros(self.out_features, device=device, dtype=torch.bfloat16),
                                     requires_grad=packed_weight is None)
        else:
            self.register_parameter("bias", None)
        if packed_weight is None:
            self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.kaiming_uniform_(self.weight, a=5 ** 0.5)
        if self.bias is not None:
            bound = self.in_features ** -0.5 if self.in_features > 0 else 0.0
            nn.init.uniform_(self.bias, -bound, bound)

    @classmethod
    def from_float(cls, module: nn.Linear, *, activation: str = "none") -> "MXFP8LinearEpilogue":
        out = cls(module.in_features, module.out_features, module.bias is not None, activation=activation,
                  device=module.weight.device)
        with torch.no_grad():
            out.weight.copy_(module.weight)
            if module.bias is not None:
                out.bias.copy_(module.bias)
        return out

    def to_quantized_weight(self) -> "MXFP8LinearEpilogue":
        if self.weight_mode == "prequantized":
            return self
        out = MXFP8LinearEpilogue(self.in_features, self.out_features, self.bias is not None, activation=self.activation,
                                  packed_weight=_fp8.quantize_mxfp8(self.weight.detach()))
        if self.bias is not None:
            with torch.no_grad():
                out.bias.copy_(self.bias)
        return out

    def packed_weight(self):
        if self.weight_mode != "prequantized":
            raise RuntimeError("module holds a BF16 weight; call to_quantized_weight() first")
        return make_mxfp8_tensor(self.weight_data, self.weight_scales, (self.out_features, self.in_features), "mma128")

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        if self.weight_mode == "prequantized":
            problem = mxfp8_state_for_kernel(state_dict, prefix, self.out_features, self.in_features)
            if problem is not None:
                error_msgs.append(problem)
                return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)

    def to(self, *args, **kwargs):
        if self.weight_mode == "prequantized":
            reject_packed_dtype_conversion(args, kwargs, format_name="MXFP8")
        return super().to(*args, **kwargs)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"activation={self.activation}, weight_mode={self.weight_mode}")

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.weight_mode == "prequantized":
            return _apply_packed(x, (self.weight_data, self.weight_scales), self.out_features, self.in_features, self.bias,
                                 residual, self.activation)
        return mxfp8_linear_epilogue(x, self.weight, self.bias, residual, activation=self.activation)


__all__ = ["MXFP8LinearEpilogue", "mxfp8_linear_epilogue", "mxfp8_linear_epilogue_backward"]
