"""Activations and slopes of the linear with an epilogue, for every BF16 pre-activation between 2^-20 and 128 in magnitude.

Tolerances, derived before the first run (u = 2^-24, half an FP32 step; the hardware's 2^x is within 2^-22 of the value,
its reciprocal within 2^-23):
  value  The exponent of e^(..) has at most three roundings of magnitude up to 126 (below, the power has left the normal
         range): 126 ln 2 * 3 u = 2^-16 of the result; the power, the reciprocal, the fit of gelu's tail (8.1e-7) and a dozen
         roundings less than 2^-18 together.  2^-15 in all, beside the BF16 rounding (2^-8).  No form cancels.  Below 2^-119
         a result may be zero: it is |z| times a power or reciprocal below 2^-126, and |z| < 88 < 2^7 there.
  slope  At z = -a.  gelu: the power 4 u and u for the exponent's put-back rounding, the fit 4.6e-8 < u, its evaluation
         2 u (the leading term is two thirds or more of the sum), 1 / (1 + 0.32 a) u, a0 - a 2 u, two products 2 u: 12 u of
         the slope with everything.  silu and gelu_tanh: q (g + q) / (1 + q)^2: q 5 u, which the sum g + q passes on in
         full where it cancels (5 u q beside a rounding of g + q), the other factors 7 u: 12 u |slope| + 8 u (q / (1 + q))^2.
         At z = a the slope is 1 less that, one more rounding (u) of a number below 2: 2 u more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev(native_lib):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    torch.cuda.set_device(0)
    return torch.device("cuda", 0)


def every_z():
    bits = torch.arange(107 << 7, (134 << 7) + 1, dtype=torch.int32)
    z = bits.to(torch.int16).view(torch.bfloat16)
    assert z[0] == 2.0 ** -20 and z[-1] == 128
    return torch.cat([z, -z])


def value64(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2))
    return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [3, 150])
def test_values_keep_their_relative_accuracy(dev, act, m):
    """Zero weights: z is the bias."""
    import rtx_b200

    z = every_z()
    x, w = torch.zeros(m, 32).bfloat16().to(dev), torch.zeros(z.numel(), 32).bfloat16().to(dev)
    y = rtx_b200.mxfp8_linear_epilogue(x, w, z.to(dev), activation=act).cpu()
    assert torch.equal(y, y[:1].expand_as(y))
    want = value64(z.double(), act)
    off = (y[0].double() - want).abs()
    live = want.abs() >= 2.0 ** -119
    rel = off[live] / want[live].abs()
    worst = rel.argmax()
    assert (rel <= 2.0 ** -8 + 2.0 ** -15).all(), (z[live][worst].item(), rel[worst].item() * 2 ** 8)
    assert (off[~live] <= 2.0 ** -119).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_slopes_are_held_to_fp32(dev, act):
    """dbias of four rows: the first has dy = 1 and the z in question; the others, with slope 1 (z = 200), subtract the
    exact slope in three BF16 parts.  What is left is the slope's error; the sums that lead to it are exact or off by u
    of what is left of the slope after the first part."""
    import rtx_b200

    z = every_z()
    v = z.double().requires_grad_(True)
    slope = torch.autograd.grad(value64(v, act).sum(), v)[0]
    if act == "gelu":   # (autograd's product form loses the tail's digits)
        a = z.double().abs()
        tail = 0.5 * torch.erfc(a / math.sqrt(2)) - a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
        slope = torch.where(z < 0, tail, 1 - tail)
    parts, rest = [], slope
    for _ in range(3):
        parts.append(rest.bfloat16())
        rest = rest - parts[-1].double()
    dy = torch.stack([torch.ones_like(z), *(-p for p in parts)])
    zs = torch.stack([z, *[torch.full_like(z, 200.0)] * 3])
    n = z.numel()
    x, w = torch.zeros(4, 32).bfloat16().to(dev), torch.zeros(n, 32).bfloat16().to(dev)
    db = rtx_b200.mxfp8_linear_epilogue_backward(dy.to(dev), zs.to(dev), x, w, activation=act)[2].double().cpu()
    at = torch.where(z < 0, slope, 1 - slope).abs()                     # the entry behind this z
    bound = 12 * U * at
    if act != "gelu":
        a = z.double().abs()
        s = torch.sigmoid(-(a if act == "silu" else 2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
        bound = bound + 8 * U * s * s
    bound = bound + torch.where(z < 0, 0.0, 2 * U) + rest.abs() + U * (slope - parts[0].double()).abs()
    live = at >= 2.0 ** -110
    over = db.abs()[live] / bound[live]
    assert (over <= 1 + 2.0 ** -8).all(), (z[live][over.argmax()].item(), over.max().item())
    assert (db.abs()[~live] <= 2.0 ** -108 + bound[~live]).all()
