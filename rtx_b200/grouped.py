"""Grouped MXFP8 linear: the products of a mixture's experts in one call.

    y[r] = q(x[r]) q(w[g])^T        rows offsets[g] .. offsets[g + 1] - 1 of x belong to group g

Same operand formats, rounding rules and gradient orientation as `mxfp8_linear` (both operands quantized in blocks of
32 along the contraction, FP32 accumulation, one BF16 rounding): a group's rows get bit for bit what `mxfp8_linear` of
those rows and that weight gives.  The reference has no grouped form; its linears are dense (rtx/fp8.py:2019-2193).

`offsets` stays on the device (int32, non-decreasing, inside [0, rows]): the host never learns the group sizes, nothing
synchronises, and a captured graph may be replayed with other offsets.  Rows of no group give zero and get a zero
gradient; a group without rows gets a zero weight gradient.
"""

from __future__ import annotations

from typing import Tuple

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import fp8 as _fp8
from . import ops
from ._oplib import call_detached, call_without_derivative, custom_op, eager, no_tangents, refuse_tangents, transformed
from .formats import (PACKED_OPERAND_SCHEMA_VERSION, SCALE_LAYOUT_CODES, MXFP8Tensor, make_mxfp8_tensor,
                      mxfp8_kernel_operands, mxfp8_qdata_2d, mxfp8_scales_for_kernel, mxfp8_state_for_kernel,
                      reject_packed_dtype_conversion)


_FROZEN = "a prequantized MXFP8 weight is inference-only; keep the BF16 master weight to train"


def _check_grouped(x: torch.Tensor, weight: torch.Tensor) -> None:
    if x.device.type != "cuda" or weight.device.type != "cuda":
        raise ValueError("MXFP8 grouped linear requires CUDA tensors")
    if x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16:
        raise TypeError(f"MXFP8 grouped linear requires BF16 operands, got {x.dtype} and {weight.dtype}")
    if x.ndim != 2 or weight.ndim != 3:
        raise ValueError("x must be [rows, K] and weight [groups, N, K]")
    if x.shape[1] != weight.shape[2]:
        raise ValueError(f"K mismatch: x has {x.shape[1]}, weight has {weight.shape[2]}")
    if min(weight.shape) == 0:
        raise ValueError("groups, N and K must be positive")


@custom_op("rtx::mxfp8_grouped_linear", mutates_args=(), device_types="cuda")
def mxfp8_grouped_linear_op(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    _check_grouped(x, weight)
    return ops.mxfp8_grouped_linear_fwd(x, weight, offsets)


@mxfp8_grouped_linear_op.register_fake
def _(x, weight, offsets):
    return x.new_empty((x.shape[0], weight.shape[1]), dtype=torch.bfloat16)


@custom_op("rtx::mxfp8_grouped_linear_prequant_w", mutates_args=(), device_types="cuda")
def mxfp8_grouped_linear_prequant_w(x: torch.Tensor, weight_data: torch.Tensor, weight_scales: torch.Tensor,
                                    offsets: torch.Tensor, n: int) -> torch.Tensor:
    return ops.mxfp8_grouped_linear_fwd_prequant_w(x, weight_data, weight_scales, offsets, n)


@mxfp8_grouped_linear_prequant_w.register_fake
def _(x, weight_data, weight_scales, offsets, n):
    return x.new_empty((x.shape[0], n), dtype=torch.bfloat16)


def _bwd(grad_output, x, weight, offsets, need_dx, need_dw):
    groups, _, k = (int(v) for v in weight.shape)
    return ops.mxfp8_grouped_linear_bwd(grad_output, x, weight, offsets, groups, k, need_dx=need_dx, need_dw=need_dw)


def _check_grad(grad_output, x, weight) -> None:
    _check_grouped(x, weight)
    if grad_output.dtype is not torch.bfloat16:
        raise TypeError(f"grad_output must be BF16, got {grad_output.dtype}")
    if tuple(grad_output.shape) != (x.shape[0], weight.shape[1]):
        raise ValueError(f"grad_output must be [{x.shape[0]}, {weight.shape[1]}]")


@custom_op("rtx::mxfp8_grouped_linear_bwd", mutates_args=(), device_types="cuda")
def mxfp8_grouped_linear_bwd(grad_output: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                             offsets: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    _check_grad(grad_output, x, weight)
    return _bwd(grad_output, x, weight, offsets, True, True)


@mxfp8_grouped_linear_bwd.register_fake
def _(grad_output, x, weight, offsets):
    return x.new_empty(x.shape), weight.new_empty(weight.shape)


@custom_op("rtx::mxfp8_grouped_linear_dx", mutates_args=(), device_types="cuda")
def mxfp8_grouped_linear_dx(grad_output: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                            offsets: torch.Tensor) -> torch.Tensor:
    """dX only; `x` gives the result's shape."""
    _check_grad(grad_output, x, weight)
    return _bwd(grad_output, x, weight, offsets, True, False)[0]


@mxfp8_grouped_linear_dx.register_fake
def _(grad_output, x, weight, offsets):
    return x.new_empty(x.shape)


@custom_op("rtx::mxfp8_grouped_linear_dw", mutates_args=(), device_types="cuda")
def mxfp8_grouped_linear_dw(grad_output: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                            offsets: torch.Tensor) -> torch.Tensor:
    """dW only; `weight` gives the result's shape."""
    _check_grad(grad_output, x, weight)
    return _bwd(grad_output, x, weight, offsets, False, True)[1]


@mxfp8_grouped_linear_dw.register_fake
def _(grad_output, x, weight, offsets):
    return weight.new_empty(weight.shape)


_TWICE = "the backward of mxfp8_grouped_linear has no derivative of its own"
mxfp8_grouped_linear_bwd.refuse_derivative(_TWICE)
mxfp8_grouped_linear_dx.refuse_derivative(_TWICE)
mxfp8_grouped_linear_dw.refuse_derivative(_TWICE)


@custom_op("rtx::mxfp8_grouped_linear_train", mutates_args=(), device_types="cuda")
def mxfp8_grouped_linear_train(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Forward of the differentiable op; saves its inputs."""
    return mxfp8_grouped_linear_op.fn(x, weight, offsets)


@mxfp8_grouped_linear_train.register_fake
def _(x, weight, offsets):
    return x.new_empty((x.shape[0], weight.shape[1]), dtype=torch.bfloat16)


def _train_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _train_backward(ctx, grad_output):
    x, weight, offsets = ctx.saved_tensors
    if eager(grad_output, x, weight, offsets):
        return (*_bwd(grad_output, x, weight, offsets, *ctx.needs_input_grad[:2]), None)
    return _dispatched_backward(ctx, grad_output)


def _dispatched_backward(ctx, grad_output):
    need_dx, need_dw = ctx.needs_input_grad[:2]
    args = (_TWICE, grad_output, *ctx.saved_tensors)
    if need_dx and need_dw:
        return (*call_without_derivative(mxfp8_grouped_linear_bwd, *args), None)
    if need_dx:
        return call_without_derivative(mxfp8_grouped_linear_dx, *args), None, None
    if need_dw:
        return None, call_without_derivative(mxfp8_grouped_linear_dw, *args), None
    return None, None, None


mxfp8_grouped_linear_train.register_autograd(_train_backward, setup_context=_train_setup)


class _GroupedLinearFunction(torch.autograd.Function):
    """The same graph node for eager calls: an op's registered autograd formula costs some 40 microseconds of host time
    per call more than this, longer than a small layer takes on the device."""

    @staticmethod
    def forward(ctx, x, weight, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return mxfp8_grouped_linear_op.fn(x, weight, offsets)

    backward = staticmethod(once_differentiable(_train_backward))


class _TransformedGroupedLinear(torch.autograd.Function):
    """The same node in the form that `torch.func` transforms take (30 microseconds of host time more than the one above).
    A pullback may be called after its transform has ended, with saved tensors that only the dispatcher can unwrap."""

    generate_vmap_rule = True

    @staticmethod
    def forward(x, weight, offsets):
        return mxfp8_grouped_linear_op(x, weight, offsets)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _train_setup(ctx, inputs, output)
        ctx.save_for_forward(*inputs)      # a batched `jvp` looks for them

    backward = staticmethod(_dispatched_backward)
    jvp = staticmethod(no_tangents("mxfp8_grouped_linear"))


def _packed_group_shape(weight) -> Tuple[int, int, int]:
    shape = weight._rtx_logical_shape
    if len(shape) != 3:
        raise ValueError(f"a packed group weight has the logical shape (groups, N, K), got {shape}")
    if shape[0] > 1 and shape[1] % 128:
        raise ValueError("packed group weights need N to be a multiple of 128 (scale tiles of 128 rows per group)")
    return shape


def mxfp8_grouped_linear(x: torch.Tensor, weight, offsets: torch.Tensor) -> torch.Tensor:
    """Rows `offsets[g] .. offsets[g + 1] - 1` of `x` times the weight of group g.

    x        BF16 [rows, K], any row pitch
    weight   BF16 [groups, N, K] (quantized in the call; differentiable), or an `MXFP8Tensor` of that logical shape, as
             `quantize_mxfp8(weight)` packs it (inference; N a multiple of 128 unless there is one group)
    offsets  int32 [groups + 1] on x's device, non-decreasing, inside [0, rows]; at most 512 groups
    returns  BF16 [rows, N]; rows of no group are zero
    """
    if isinstance(weight, MXFP8Tensor):
        groups, n, k = _packed_group_shape(weight)
        if x.ndim != 2 or x.shape[1] != k:
            raise ValueError(f"K mismatch: x has {x.shape[-1]}, weight has {k}")
        if isinstance(offsets, torch.Tensor) and offsets.shape != (groups + 1,):
            raise ValueError(f"offsets must be a contiguous vector of groups + 1 = {groups + 1} row numbers")
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(_FROZEN)
        return _packed(x, *mxfp8_kernel_operands(weight), offsets, n)
    return _dynamic(x, weight, offsets)


def _packed(x, weight_data, weight_scales, offsets, n) -> torch.Tensor:
    refuse_tangents("mxfp8_grouped_linear", x)
    if eager(x, weight_data, weight_scales, offsets):
        return ops.mxfp8_grouped_linear_fwd_prequant_w(x, weight_data, weight_scales, offsets, n)
    return call_without_derivative(mxfp8_grouped_linear_prequant_w, _FROZEN, x, weight_data, weight_scales, offsets, n)


def _dynamic(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    refuse_tangents("mxfp8_grouped_linear", x, weight)
    direct = eager(x, weight, offsets)
    if not direct and transformed():
        return _TransformedGroupedLinear.apply(x, weight, offsets)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return (_GroupedLinearFunction.apply if direct else mxfp8_grouped_linear_train)(x, weight, offsets)
    return (mxfp8_grouped_linear_op.fn if direct else mxfp8_grouped_linear_op)(x, weight, offsets)


def mxfp8_grouped_linear_backward(grad_output: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                                  offsets: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """BF16 dX [rows, K] and dW [groups, N, K] of `mxfp8_grouped_linear`, from independently quantized MXFP8 products
    (blocks along N for dX, along each group's rows for dW).  There is no FP32 dW for sums over ranks, as the dense linear's
    backward has one."""
    refuse_tangents("mxfp8_grouped_linear_backward", grad_output, x, weight)
    if eager(x, grad_output, weight, offsets):
        return mxfp8_grouped_linear_bwd.fn(grad_output, x, weight, offsets)
    return call_detached(mxfp8_grouped_linear_bwd, _TWICE, grad_output, x, weight, offsets)


class MXFP8GroupedLinear(nn.Module):
    """One no-bias linear per group, `weight` BF16 [groups, out_features, in_features]; `forward(x, offsets)`.

    `to_quantized_weight()` gives the inference copy with packed weights (buffers `weight_data`, `weight_scales`,
    `weight_packing_meta` as in `MXFP8Linear`)."""

    __constants__ = ["num_groups", "in_features", "out_features", "weight_mode"]

    def __init__(self, num_groups: int, in_features: int, out_features: int, *, device=None,
                 dtype: torch.dtype = torch.bfloat16, packed_weight=None) -> None:
        super().__init__()
        if dtype is not torch.bfloat16:
            raise TypeError(f"MXFP8GroupedLinear parameters must be BF16, got {dtype}")
        if not 1 <= int(num_groups) <= ops.MAX_GROUPS:
            raise ValueError(f"num_groups must be between 1 and {ops.MAX_GROUPS}")
        self.num_groups, self.in_features, self.out_features = int(num_groups), int(in_features), int(out_features)
        self.weight_mode = "prequantized" if packed_weight is not None else "dynamic"
        if packed_weight is None:
            self.weight = nn.Parameter(torch.empty(self.num_groups, self.out_features, self.in_features, device=device,
                                                   dtype=torch.bfloat16))
            self.reset_parameters()
        else:
            if _packed_group_shape(packed_weight) != (self.num_groups, self.out_features, self.in_features):
                raise ValueError("packed weight does not have the module's shape")
            self.register_parameter("weight", None)
            self.register_buffer("weight_data", mxfp8_qdata_2d(packed_weight).view(torch.uint8))
            self.register_buffer("weight_scales", mxfp8_scales_for_kernel(packed_weight))
            self.register_buffer("weight_packing_meta", torch.tensor(
                [PACKED_OPERAND_SCHEMA_VERSION, SCALE_LAYOUT_CODES["mma128"], self.in_features,
                 int(packed_weight.qdata.shape[-1])], dtype=torch.int64))

    def reset_parameters(self) -> None:
        for g in range(self.num_groups):
            nn.init.kaiming_uniform_(self.weight[g], a=5 ** 0.5)

    def to_quantized_weight(self) -> "MXFP8GroupedLinear":
        if self.weight_mode == "prequantized":
            return self
        return MXFP8GroupedLinear(self.num_groups, self.in_features, self.out_features,
                                  packed_weight=_fp8.quantize_mxfp8(self.weight.detach()))

    def packed_weight(self):
        if self.weight_mode != "prequantized":
            raise RuntimeError("module holds a BF16 weight; call to_quantized_weight() first")
        return make_mxfp8_tensor(self.weight_data, self.weight_scales,
                                 (self.num_groups, self.out_features, self.in_features), "mma128")

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        if self.weight_mode == "prequantized":
            problem = mxfp8_state_for_kernel(state_dict, prefix, self.num_groups * self.out_features, self.in_features)
            if problem is not None:
                error_msgs.append(problem)
                return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)

    def to(self, *args, **kwargs):
        if self.weight_mode == "prequantized":
            reject_packed_dtype_conversion(args, kwargs, format_name="MXFP8")
        return super().to(*args, **kwargs)

    def extra_repr(self) -> str:
        return (f"num_groups={self.num_groups}, in_features={self.in_features}, out_features={self.out_features}, "
                f"weight_mode={self.weight_mode}")

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"K mismatch: x has {x.shape[-1]}, weight has {self.in_features}")
        if self.weight_mode == "prequantized":
            if x.requires_grad and torch.is_grad_enabled():
                raise RuntimeError(_FROZEN)
            return _packed(x, self.weight_data, self.weight_scales, offsets, self.out_features)
        return _dynamic(x, self.weight, offsets)


__all__ = ["MXFP8GroupedLinear", "mxfp8_grouped_linear", "mxfp8_grouped_linear_backward"]
