"""Grouped MXFP8 linear: refusals and host logic (no GPU, no kernel launch)."""
import ctypes

import pytest
import torch


def test_entry_points_refuse_bad_arguments_before_any_launch(native_lib):
    from rtx_b200 import _native as N

    L = native_lib
    buf = (ctypes.c_uint8 * 8192)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256
    size = N.query("rtxb_mxfp8_grouped_linear_workspace_bytes", 64, 128, 64, 4, 1)
    assert size >= 64 * 64 + 4 * 128 * 64 > N.query("rtxb_mxfp8_grouped_linear_workspace_bytes", 64, 128, 64, 4, 0) - 8192

    def fwd(x=p, ldx=64, w=p, offsets=p, groups=4, out=p, ldo=128, rows=64, n=128, k=64, ws=p, nbytes=size):
        return L.rtxb_mxfp8_grouped_linear_fwd(x, ldx, w, offsets, groups, out, ldo, rows, n, k, 1, ws, nbytes, None, None)

    assert fwd(x=None) == fwd(w=None) == fwd(offsets=None) == fwd(out=None) == -1
    assert fwd(ldx=63) == fwd(ldo=127) == -1
    assert fwd(rows=0) == fwd(n=0) == fwd(k=0) == fwd(groups=0) == fwd(rows=-1) == -1
    assert fwd(groups=513) == -2
    assert fwd(rows=2 ** 31, ldx=2 ** 40) == fwd(n=2 ** 31, ldo=2 ** 40) == fwd(k=2 ** 31, ldx=2 ** 40) == -2
    assert fwd(groups=512, n=2 ** 23, ldo=2 ** 23) == -2            # weight rows beyond 32 bits
    assert fwd(x=p + 1) == fwd(out=p + 1) == fwd(w=p + 1) == fwd(offsets=p + 2) == -3
    assert fwd(ws=None) == fwd(nbytes=size - 1) == -4
    assert fwd(ws=p + 128) == -3

    def packed(qw=p, sw=p, n=128, groups=4, ldo=256):
        return L.rtxb_mxfp8_grouped_linear_fwd_prequant_w(p, 64, qw, sw, p, groups, p, ldo, 64, n, 64, 1, p, 0, None, None)

    assert packed(qw=None) == packed(sw=None) == -1
    assert packed(n=200) == -2 and packed(n=200, groups=1) == -4    # one group may have any width (refused here by size)
    assert packed(qw=p + 8) == packed(sw=p + 8) == -3
    both = N.query("rtxb_mxfp8_grouped_backward_workspace_bytes", 64, 128, 64, 4, 1, 1)
    assert both > N.query("rtxb_mxfp8_grouped_backward_workspace_bytes", 64, 128, 64, 4, 1, 0)

    def bwd(dy=p, lddy=128, x=p, ldx=64, w=p, offsets=p, groups=4, dx=p, dw=p, ws=p, nbytes=both):
        return L.rtxb_mxfp8_grouped_linear_bwd(dy, lddy, x, ldx, w, offsets, groups, dx, dw, 64, 128, 64, ws, nbytes, None, None)

    assert bwd(dy=None) == bwd(w=None) == bwd(x=None) == bwd(dx=None, dw=None) == bwd(offsets=None) == -1
    assert bwd(lddy=127) == bwd(ldx=63) == -1
    assert bwd(groups=600) == -2
    assert bwd(dx=p + 1) == bwd(dw=p + 1) == -3
    assert bwd(ws=None) == bwd(nbytes=both - 1) == -4


def test_python_refusals():
    from rtx_b200 import ops
    from rtx_b200.formats import make_mxfp8_tensor
    from rtx_b200.grouped import MXFP8GroupedLinear, mxfp8_grouped_linear

    x, w = torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(2, 128, 64, dtype=torch.bfloat16)
    o = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        mxfp8_grouped_linear(x, w, o)                       # the op has a CUDA implementation only
    with pytest.raises(ValueError, match="CUDA"):
        ops.mxfp8_grouped_linear_fwd(x, w, o)
    with pytest.raises(ValueError, match="groups, N, K"):
        ops._group_weight(w[0], torch.device("cpu"))
    for bad, error in ((torch.zeros(3, dtype=torch.int64), TypeError), (torch.zeros(4, dtype=torch.int32), ValueError),
                       (torch.zeros(1, 3, dtype=torch.int32), ValueError), (torch.zeros(6, dtype=torch.int32)[::2], ValueError),
                       ([0, 1, 2], TypeError)):
        with pytest.raises(error, match="offsets"):
            ops._require_offsets(bad, 2, torch.device("cpu"))
    with pytest.raises(ValueError, match="512"):
        ops._require_offsets(torch.zeros(514, dtype=torch.int32), 513, torch.device("cpu"))

    packed = make_mxfp8_tensor(torch.zeros(2 * 100, 64, dtype=torch.uint8), torch.zeros(2 * 512, dtype=torch.uint8),
                               (2, 100, 64), "mma128")
    with pytest.raises(ValueError, match="multiple of 128"):
        mxfp8_grouped_linear(x, packed, o)
    flat = make_mxfp8_tensor(torch.zeros(128, 64, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8), (128, 64), "mma128")
    with pytest.raises(ValueError, match="logical shape"):
        mxfp8_grouped_linear(x, flat, o)
    good = make_mxfp8_tensor(torch.zeros(256, 64, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8), (2, 128, 64), "mma128")
    with pytest.raises(ValueError, match="K mismatch"):
        mxfp8_grouped_linear(x[:, :32], good, o)
    with pytest.raises(RuntimeError, match="inference-only"):
        mxfp8_grouped_linear(x.clone().requires_grad_(True), good, o)

    with pytest.raises(TypeError, match="BF16"):
        MXFP8GroupedLinear(2, 64, 128, dtype=torch.float32)
    with pytest.raises(ValueError, match="num_groups"):
        MXFP8GroupedLinear(0, 64, 128)
    m = MXFP8GroupedLinear(2, 64, 128)
    assert tuple(m.weight.shape) == (2, 128, 64) and list(m.state_dict()) == ["weight"]
    with pytest.raises(ValueError, match="K mismatch"):
        m(x[:, :32], o)


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from rtx_b200 import grouped

    with FakeTensorMode():
        x = torch.empty(8, 64, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(2, 96, 64, dtype=torch.bfloat16, device="cuda")
        o = torch.empty(3, dtype=torch.int32, device="cuda")
        y = grouped.mxfp8_grouped_linear(x, w, o)
        assert tuple(y.shape) == (8, 96) and y.dtype is torch.bfloat16
        dx, dw = grouped.mxfp8_grouped_linear_backward(y, x, w, o)
        assert dx.shape == x.shape and dw.shape == w.shape
