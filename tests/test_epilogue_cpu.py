"""MXFP8 linear with bias, activation and residual: refusals and host logic (no GPU, no kernel launch)."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_entry_points_refuse_bad_arguments_before_any_launch(native_lib):
    from rtx_b200 import _native as N

    L = native_lib
    buf = (ctypes.c_uint8 * 8192)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256
    size = N.query("rtxb_mxfp8_linear_epilogue_workspace_bytes", 64, 128, 96, 1)
    assert size >= (64 + 128) * 96 > N.query("rtxb_mxfp8_linear_epilogue_workspace_bytes", 64, 128, 96, 0) - 4096

    def fwd(x=p, ldx=96, w=p, bias=p, res=p, ldr=128, out=p, z=p, m=64, n=128, k=96, act=0, ws=p, nbytes=size):
        return L.rtxb_mxfp8_linear_epilogue_fwd(x, ldx, w, bias, res, ldr, out, z, m, n, k, act, 1, ws, nbytes, None, None)

    assert fwd(x=None) == fwd(w=None) == fwd(out=None) == -1
    assert fwd(ldx=95) == fwd(ldr=127) == fwd(m=0) == fwd(n=0) == fwd(k=0) == fwd(act=6) == fwd(act=-1) == -1
    assert fwd(m=2 ** 31) == fwd(n=2 ** 31, ldr=2 ** 40) == fwd(k=2 ** 31, ldx=2 ** 40) == -2
    assert fwd(x=p + 1) == fwd(w=p + 1) == fwd(bias=p + 1) == fwd(res=p + 1) == fwd(out=p + 1) == fwd(z=p + 1) == -3
    assert fwd(ws=None) == fwd(nbytes=size - 1) == -4
    assert fwd(ws=p + 64) == -3

    def packed(qw=p, sw=p):
        return L.rtxb_mxfp8_linear_epilogue_fwd_prequant_w(p, 96, qw, sw, None, None, 0, p, 64, 128, 96, 0, 1, p, 0, None, None)

    assert packed(qw=None) == packed(sw=None) == -1 and packed(qw=p + 8) == packed(sw=p + 8) == -3 and packed() == -4
    full = N.query("rtxb_mxfp8_linear_epilogue_backward_workspace_bytes", 64, 128, 96, 1, 1, 1)
    assert full > N.query("rtxb_mxfp8_linear_epilogue_backward_workspace_bytes", 64, 128, 96, 1, 1, 0)

    def bwd(dy=p, lddy=128, z=p, x=p, ldx=96, w=p, dx=p, dw=p, db=p, act=3, ws=p, nbytes=full):
        return L.rtxb_mxfp8_linear_epilogue_bwd(dy, lddy, z, x, ldx, w, dx, dw, db, 64, 128, 96, act, ws, nbytes, None, None)

    assert bwd(dy=None) == bwd(z=None) == bwd(x=None) == bwd(w=None) == bwd(dx=None, dw=None, db=None) == -1
    assert bwd(lddy=127) == bwd(ldx=95) == bwd(act=9) == -1
    assert bwd(z=p + 1) == bwd(db=p + 1) == -3
    assert bwd(ws=None) == bwd(nbytes=full - 1) == bwd(z=None, act=0, nbytes=0) == -4


def test_activation_codes_agree_between_header_kernels_and_python():
    from rtx_b200 import ops

    header = open(os.path.join(ROOT, "include", "rtxb.h")).read()
    macros = {name.lower(): int(v) for name, v in re.findall(r"#define RTXB_ACT_([A-Z0-9_]+) (\d+)", header)}
    assert macros == ops.ACTIVATIONS
    device = open(os.path.join(ROOT, "rtx_b200", "csrc", "activation.cuh")).read()
    codes = [int(v) for _, v in re.findall(r"(kAct[A-Za-z0-9]+) = (\d+)", device)]
    assert sorted(codes) == sorted(macros.values())


def test_python_refusals():
    from rtx_b200.epilogue import MXFP8LinearEpilogue, mxfp8_linear_epilogue, mxfp8_linear_epilogue_backward
    from rtx_b200.formats import make_mxfp8_tensor
    from rtx_b200 import ops

    x, w = torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(128, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        mxfp8_linear_epilogue(x, w)                       # the op has a CUDA implementation only
    with pytest.raises(ValueError, match="K mismatch"):
        mxfp8_linear_epilogue(x[:, :32], w)
    with pytest.raises(ValueError, match="residual"):
        mxfp8_linear_epilogue(x, w, None, torch.zeros(128, dtype=torch.bfloat16))     # not broadcast
    with pytest.raises(ValueError, match="unknown activation"):
        ops.activation_code("tanh")
    with pytest.raises(ValueError, match="unknown activation"):
        MXFP8LinearEpilogue(64, 128, activation=None)
    with pytest.raises(TypeError, match="BF16"):
        MXFP8LinearEpilogue(64, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops._rows_of(x, 64, "x")
    for bad, error in ((torch.zeros(128), TypeError), (torch.zeros(64, dtype=torch.bfloat16), ValueError),
                       (torch.zeros(1, 128, dtype=torch.bfloat16), ValueError), (1.0, TypeError)):
        with pytest.raises(error, match="bias"):
            ops._vector_of(bad, 128, torch.device("cpu"), "bias")
    packed = make_mxfp8_tensor(torch.zeros(128, 64, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), (128, 64), "mma128")
    with pytest.raises(RuntimeError, match="inference-only"):
        mxfp8_linear_epilogue(x.clone().requires_grad_(True), packed)
    with pytest.raises(RuntimeError, match="inference-only"):
        mxfp8_linear_epilogue(x, packed, torch.zeros(128, dtype=torch.bfloat16, requires_grad=True))
    with pytest.raises(ValueError, match="pre-activation"):
        mxfp8_linear_epilogue_backward(torch.zeros(8, 128, dtype=torch.bfloat16), None, x, w, activation="gelu")
    m = MXFP8LinearEpilogue.from_float(torch.nn.Linear(64, 128), activation="gelu")
    assert sorted(m.state_dict()) == ["bias", "weight"] and m.weight.dtype is torch.bfloat16
    assert MXFP8LinearEpilogue(64, 128, bias=False).bias is None


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from rtx_b200 import epilogue

    with FakeTensorMode():
        # (autograd's engine itself needs a device: the gradients' shapes are taken from the backward)
        x = torch.empty(2, 4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        w = torch.empty(96, 64, dtype=torch.bfloat16, device="cuda")
        b = torch.empty(96, dtype=torch.bfloat16, device="cuda")
        y = epilogue.mxfp8_linear_epilogue(x, w, b, activation="silu")
        assert tuple(y.shape) == (2, 4, 96) and y.dtype is torch.bfloat16 and y.requires_grad
        dx, dw, db = epilogue.mxfp8_linear_epilogue_backward(y.detach(), y.detach(), x.detach(), w, activation="silu")
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape


def test_backward_takes_no_operand_by_its_number_of_values():
    """Rows of another width whose values happen to fill whole rows of the right one are refused, not reshaped."""
    from rtx_b200.epilogue import mxfp8_linear_epilogue_backward

    def zeros(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16)

    w = zeros(16, 32)
    for dy, z, x, name in ((zeros(4, 32), zeros(8, 16), zeros(8, 32), "grad_output"), (zeros(8, 16), zeros(8, 16), zeros(4, 64), "x"),
                           (zeros(8, 16), zeros(16, 8), zeros(8, 32), "z"), (zeros(8, 16), zeros(8, 16), zeros(()), "x")):
        with pytest.raises(ValueError, match=f"{name} must have rows of"):
            mxfp8_linear_epilogue_backward(dy, z, x, w, activation="silu")
    with pytest.raises(NotImplementedError):                    # the right widths reach the op (which needs a GPU)
        mxfp8_linear_epilogue_backward(zeros(2, 4, 16), zeros(8, 16), zeros(8, 32), w, activation="silu")
    with pytest.raises(NotImplementedError):                    # z is not looked at without an activation
        mxfp8_linear_epilogue_backward(zeros(8, 16), zeros(3), zeros(8, 32), w)
