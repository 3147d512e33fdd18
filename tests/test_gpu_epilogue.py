"""MXFP8 linear with bias, activation and residual against its definition in 64 bits.

Tolerances, derived before the first run (u = 2^-23, one FP32 step relative to a value in [1, 2)):
  z     FP32 accumulation of K products in any order, cut instead of rounded: K u S, S the sum of their magnitudes;
        the bias addition adds u (|z| + |bias|).
  y     act has slope at most L (1; 1.13 for silu and the gelus; 2 |z| for relu2), so z's error enters L-fold; the FP32
        evaluation of act is off by at most 16 u |z| (16 u z^2 for relu2); the residual addition by u (|act| + |r|); the
        BF16 rounding by 2^-8 of the value (finfo.eps / 2).
  dz    the FP32 slope is off by at most 8 u (1 + |z|), so dy act'(z) lies within a = |dy| 8 u (1 + |z|) (0 for none, relu
        and relu2, whose products are exact: 8 + 8 bits) of the exact one.  Rounding to BF16 and to MXFP8 is monotone
        for a given block scale, and the scale is one of those of the interval's ends, so the quantized value lies
        between the smallest and largest of the four combinations; delta is their distance.
  dx    delta @ |w| beside the accumulation and the rounding; dw likewise.
  db    FP32 sum of M values: M u sum |dz|, plus the sum of a, plus the rounding."""
import math

import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
ACTS = ["none", "relu", "relu2", "silu", "gelu", "gelu_tanh"]


@pytest.fixture(scope="module")
def dev(native_lib):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    torch.cuda.set_device(0)
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def no_status(request):
    yield
    if "dev" in request.fixturenames:
        from rtx_b200 import ops

        torch.cuda.synchronize()
        ops.check_device_status(torch.device("cuda", 0))


def mx(v):
    q, s = O.mxfp8_quantize(v.contiguous())
    return O.mxfp8_dequantize(q, s).double()


def act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "relu2": lambda: z.clamp(min=0) ** 2,
            "silu": lambda: z * torch.sigmoid(z), "gelu": lambda: 0.5 * z * torch.erfc(-z / math.sqrt(2)),
            "gelu_tanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}[act]()


def slope64(z, act):
    v = z.clone().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act64(v, act).sum(), v)[0]


def within(got, want, bound):
    assert got.dtype is torch.bfloat16 and got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (off - bound).max().item()


def inputs(m, n, k, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen)
    x = torch.where(torch.rand(m, k, generator=gen) < 0.01, 20 * x, x).bfloat16()
    w = (torch.randn(n, k, generator=gen) / k ** 0.5).bfloat16()
    b = torch.randn(n, generator=gen).bfloat16()
    r = torch.randn(m, n, generator=gen).bfloat16()
    dy = (0.1 * torch.randn(m, n, generator=gen)).bfloat16()
    return x, w, b, r, dy


def forward(x, w, b, r, act):
    """(y, its bound, z, its bound before the rounding)"""
    k = x.shape[1]
    xa, wa = mx(x), mx(w)
    z = xa @ wa.T
    ez = k * U * (xa.abs() @ wa.abs().T)
    if b is not None:
        z = z + b.double()
        ez = ez + U * (z.abs() + b.double().abs())
    a = act64(z, act)
    slope = {"none": 1.0, "relu": 1.0, "relu2": 2 * z.abs() + ez}.get(act, 1.13)
    ey = slope * ez + (0 if act in ("none", "relu") else 16 * U * (z ** 2 if act == "relu2" else z.abs()))
    y = a
    if r is not None:
        y = a + r.double()
        ey = ey + U * (a.abs() + r.double().abs())
    return y, 2.0 ** -8 * y.abs() + (1 + 2.0 ** -8) * ey, z, ez


def mx_span(lo, hi):
    """Of BF16 values between lo and hi (elementwise): the middle and the distance of the MXFP8 values they can get."""
    ends = []
    for scale_of in (lo, hi):
        code = O.mxfp8_quantize(scale_of.contiguous())[1]
        recip = O.e8m0_reciprocal(code).repeat_interleave(32, -1)
        kp = recip.shape[-1]
        for v in (lo, hi):
            vf = torch.nn.functional.pad(v.float(), (0, kp - v.shape[-1]))
            ends.append(O.mxfp8_dequantize(O.e4m3_encode(vf * recip), code).double())
    ends = torch.stack(ends)
    return ends.amin(0), ends.amax(0)


def backward(dy, z, x, w, act):
    """{name: (value, bound)} of dx, dw, db for the pre-activation z in BF16"""
    m, n = dy.shape
    dz = dy.double() * slope64(z.double(), act)
    a = torch.zeros_like(dz) if act in ("none", "relu", "relu2") else dy.double().abs() * 8 * U * (1 + z.double().abs())
    out = {}
    for name, turn, other, depth in (("dx", lambda t: t, mx(w.T), n), ("dw", lambda t: t.T, mx(x.T), m)):
        v = mx(turn(dz.bfloat16()))
        lo, hi = mx_span(turn((dz - a).bfloat16()), turn((dz + a).bfloat16()))
        delta = torch.maximum(hi - v, v - lo)
        assert (delta >= 0).all()
        want = v @ other.T
        off = delta @ other.abs().T + depth * U * (torch.maximum(lo.abs(), hi.abs()) @ other.abs().T)
        out[name] = want, 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * off
    want = dz.sum(0)
    out["db"] = want, 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * (m * U * dz.abs().sum(0) + a.sum(0))
    return out


SHAPES = [(1, 1, 1), (1, 128, 64), (5, 17, 33), (8, 256, 256), (64, 200, 96), (128, 72, 520), (129, 256, 128),
          (130, 40, 72), (257, 257, 65), (300, 520, 136)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_forward_shapes(dev, m, n, k, act):
    import rtx_b200

    x, w, b, r, _ = inputs(m, n, k)
    y = rtx_b200.mxfp8_linear_epilogue(x.to(dev), w.to(dev), b.to(dev), r.to(dev), activation=act)
    within(y, *forward(x, w, b, r, act)[:2])
    packed = rtx_b200.quantize_mxfp8(w.to(dev))
    assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x.to(dev), packed, b.to(dev), r.to(dev), activation=act), y)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("m", [7, 150])
def test_forward_parts(dev, act, bias, residual, m):
    from rtx_b200 import ops

    x, w, b, r, _ = inputs(m, 136, 160, seed=1)
    b, r = b if bias else None, r if residual else None
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y, none = ops.mxfp8_linear_epilogue_fwd(on(x), on(w), on(b), on(r), activation=act)
    assert none is None
    want, bound, z_want, ez = forward(x, w, b, r, act)
    within(y, want, bound)
    y2, z = ops.mxfp8_linear_epilogue_fwd(on(x), on(w), on(b), on(r), activation=act, keep_z=True)
    assert torch.equal(y, y2)
    within(z, z_want, 2.0 ** -8 * z_want.abs() + (1 + 2.0 ** -8) * ez)


def test_plain_epilogue_is_the_linear(dev):
    """No bias, no activation, no residual: the bits of mxfp8_linear, in every schedule."""
    import rtx_b200
    from rtx_b200 import ops

    for m, n in ((5, 256), (200, 384), (1, 20000)):
        x, w, *_ = (t.to(dev) for t in inputs(m, n, 96, seed=2))
        want = rtx_b200.mxfp8_linear(x, w)
        assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x, w), want)
        for schedule in ("single", "pair", "stream"):
            with ops.gemm_schedule(schedule):
                assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x, w), want)


@pytest.mark.parametrize("schedule", ["single", "pair", "stream"])
def test_schedules_give_the_same_bits(dev, schedule):
    from rtx_b200 import ops

    for m in (9, 140):
        x, w, b, r, _ = (t.to(dev) for t in inputs(m, 300, 128, seed=3))
        want = ops.mxfp8_linear_epilogue_fwd(x, w, b, r, activation="silu", keep_z=True)
        with ops.gemm_schedule(schedule):
            got = ops.mxfp8_linear_epilogue_fwd(x, w, b, r, activation="silu", keep_z=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_larger_than_one_wave(dev):
    """More tiles than resident CTAs, several chunks in flight per staging buffer."""
    from rtx_b200 import ops

    x, w, b, r, _ = inputs(2600, 2816, 64, seed=4)
    on = lambda t: t.to(dev)  # noqa: E731
    want, bound, z_want, ez = forward(x, w, b, r, "gelu_tanh")
    y, z = ops.mxfp8_linear_epilogue_fwd(on(x), on(w), on(b), on(r), activation="gelu_tanh", keep_z=True)
    within(y, want, bound)
    within(z, z_want, 2.0 ** -8 * z_want.abs() + (1 + 2.0 ** -8) * ez)


def test_pitches_and_unaligned_operands(dev):
    import rtx_b200

    x, w, b, r, _ = inputs(140, 120, 96, seed=5)
    want, bound = forward(x, w, b, r, "relu")[:2]
    wd = w.to(dev)
    for pad, lead in ((8, 0), (13, 0), (13, 1)):
        wide = torch.full((140, 96 + pad + lead), float("nan"), dtype=torch.bfloat16, device=dev)
        wide_r = torch.full((140, 120 + pad + lead), float("nan"), dtype=torch.bfloat16, device=dev)
        wide_b = torch.full((120 + lead,), float("nan"), dtype=torch.bfloat16, device=dev)
        xs, rs, bs = wide[:, lead:lead + 96], wide_r[:, lead:lead + 120], wide_b[lead:]
        xs.copy_(x), rs.copy_(r), bs.copy_(b)
        within(rtx_b200.mxfp8_linear_epilogue(xs, wd, bs, rs, activation="relu"), want, bound)
    # leading dimensions, a transposed residual, a broadcast bias
    y = rtx_b200.mxfp8_linear_epilogue(x.to(dev).view(7, 20, 96), wd, b.to(dev), r.T.contiguous().to(dev).T.reshape(7, 20, 120),
                                       activation="relu")
    assert y.shape == (7, 20, 120)
    within(y.view(140, 120), want, bound)
    one = torch.tensor([0.5], dtype=torch.bfloat16, device=dev).expand(120)
    within(rtx_b200.mxfp8_linear_epilogue(x.to(dev), wd, one, activation="relu"),
           *forward(x, w, one.cpu().contiguous(), None, "relu")[:2])


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("act", ["none", "relu2", "gelu"])
def test_backward_shapes(dev, m, n, k, act):
    import rtx_b200

    x, w, _, z, dy = inputs(m, n, k, seed=6)
    dx, dw, db = rtx_b200.mxfp8_linear_epilogue_backward(dy.to(dev), z.to(dev), x.to(dev), w.to(dev), activation=act)
    want = backward(dy, z, x, w, act)
    within(dx, *want["dx"])
    within(dw, *want["dw"])
    within(db, *want["db"])


@pytest.mark.parametrize("act", ACTS)
def test_backward_activations_and_wide_pre_activations(dev, act):
    import rtx_b200

    x, w, _, z, dy = inputs(200, 168, 96, seed=7)
    z = (z.float() * torch.exp(3 * torch.randn(z.shape, generator=torch.Generator().manual_seed(1)))).bfloat16()
    args = (dy.to(dev), z.to(dev), x.to(dev), w.to(dev))
    dx, dw, db = rtx_b200.mxfp8_linear_epilogue_backward(*args, activation=act)
    want = backward(dy, z, x, w, act)
    within(dx, *want["dx"])
    within(dw, *want["dw"])
    within(db, *want["db"])
    assert rtx_b200.mxfp8_linear_epilogue_backward(*args, activation=act, bias=False)[2] is None
    if act in ("none", "relu", "relu2"):   # dz is exact: the bits of the plain backward of that dz
        dz = (dy.double() * slope64(z.double(), act)).bfloat16().to(dev)
        want_dx, want_dw = rtx_b200.mxfp8_linear_backward(dz, x.to(dev), w.to(dev))
        assert torch.equal(dx, want_dx) and torch.equal(dw, want_dw)


@pytest.mark.parametrize("act", ACTS)
def test_extreme_pre_activations_give_the_limits(dev, act):
    """Infinities, the type's lowest and largest values and zeros: act and its slope take their limits, NaN stays NaN."""
    from rtx_b200 import ops

    top = torch.finfo(torch.bfloat16).max
    zs = torch.tensor([0.0, -0.0, top, -top, 1e-30, -1e-30, 200.0, -200.0], dtype=torch.bfloat16)
    n = zs.numel()
    x = torch.zeros(3, 32, dtype=torch.bfloat16, device=dev)
    w = torch.zeros(n, 32, dtype=torch.bfloat16, device=dev)
    y, z = ops.mxfp8_linear_epilogue_fwd(x, w, zs.to(dev), activation=act, keep_z=True)
    assert torch.equal(z.cpu(), zs.expand(3, n))
    limit = {"none": zs, "relu": zs.clamp(min=0)}.get(act)
    if limit is None:
        limit = torch.where(zs.abs() > 1, zs.clamp(min=0), act64(zs.double(), act).bfloat16())
        if act == "relu2":
            limit = (zs.float().clamp(min=0) ** 2).bfloat16()
    assert torch.equal(y.cpu(), limit.expand(3, n))
    # slopes through dbias: one row, dy = 1, dbias = act'(z)
    zi = torch.cat([zs, torch.tensor([float("inf"), -float("inf"), float("nan")], dtype=torch.bfloat16)])
    ones = torch.ones(1, n + 3, dtype=torch.bfloat16, device=dev)
    db = ops.mxfp8_linear_epilogue_bwd(ones, zi[None].contiguous().to(dev), None, None, 32, activation=act, need_dx=False,
                                       need_dw=False, need_dbias=True)[2].cpu()
    big = zi.abs() > 1
    want = {"none": torch.ones(n + 3), "relu": (zi > 0).float(), "relu2": 2 * zi.float().clamp(min=0)}.get(act)
    if want is None:
        want = torch.where(big, (zi > 0).float(), torch.full((n + 3,), 0.5))
    want = want.bfloat16()
    if act != "none":
        want[-1] = float("nan")
    assert torch.equal(db.isnan(), want.isnan())
    keep = ~want.isnan()
    assert torch.equal(db[keep], want[keep])


def test_autograd_matches_the_backward_and_differences(dev):
    """Autograd returns the backward's gradients; and they are the gradient: with relu2 on operands whose products and
    squares BF16 and MXFP8 hold exactly and z > 0, the loss is quadratic and a central difference is exact."""
    import rtx_b200

    gen = torch.Generator().manual_seed(8)
    eye = torch.eye(32)[torch.randint(0, 32, (6,), generator=gen)].bfloat16()
    w = torch.randint(-1, 2, (16, 32), generator=gen).bfloat16()
    b = torch.full((16,), 4.0, dtype=torch.bfloat16)
    r = torch.randint(-2, 3, (6, 16), generator=gen).bfloat16()
    c = torch.randint(-1, 2, (6, 16), generator=gen).bfloat16()
    leaves = [t.to(dev).requires_grad_(True) for t in (eye, w, b, r)]
    y = rtx_b200.mxfp8_linear_epilogue(*leaves, activation="relu2")
    gx, gw, gb, gr = torch.autograd.grad(y, leaves, c.to(dev))
    z = (eye.float() @ w.float().T + b.float()).bfloat16()
    dx, dw, db = rtx_b200.mxfp8_linear_epilogue_backward(c.to(dev), z.to(dev), eye.to(dev), w.to(dev), activation="relu2")
    assert torch.equal(gx, dx) and torch.equal(gw, dw) and torch.equal(gb, db) and torch.equal(gr.cpu(), c)

    def loss(*t):
        return (rtx_b200.mxfp8_linear_epilogue(*(v.to(dev) for v in t), activation="relu2").double() * c.to(dev).double()).sum().item()

    base = [eye, w, b, r]
    for i, g in enumerate((gx, gw, gb, gr)):
        for _ in range(3):
            step = torch.zeros_like(base[i])
            step.view(-1)[torch.randint(0, step.numel(), (1,), generator=gen)] = 1.0
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + step, base[i] - step
            assert loss(*up) - loss(*down) == 2 * (g.double().cpu() * step.double()).sum().item()


@pytest.mark.parametrize("act", ["none", "silu"])
def test_each_gradient_alone(dev, act):
    import rtx_b200

    x, w, b, r, dy = (t.to(dev) for t in inputs(70, 96, 64, seed=9))
    all_leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(rtx_b200.mxfp8_linear_epilogue(*all_leaves, activation=act), all_leaves, dy)
    for i in range(4):
        args = [x, w, b, r]
        args[i] = args[i].clone().requires_grad_(True)
        got = torch.autograd.grad(rtx_b200.mxfp8_linear_epilogue(*args, activation=act), args[i], dy)[0]
        assert torch.equal(got, want[i])
    # an expanded gradient, and no bias or residual
    a = x.clone().requires_grad_(True)
    rtx_b200.mxfp8_linear_epilogue(a, w, activation=act).sum().backward()
    b2 = x.clone().requires_grad_(True)
    rtx_b200.mxfp8_linear_epilogue(b2, w, activation=act).backward(torch.ones(70, 96, dtype=torch.bfloat16, device=dev))
    assert torch.equal(a.grad, b2.grad)
    # one tensor in two places: both gradients arrive
    sq = torch.randn(64, 64, device=dev).bfloat16().requires_grad_(True)
    parts = [sq.detach().clone().requires_grad_(True) for _ in range(3)]
    g = torch.autograd.grad(rtx_b200.mxfp8_linear_epilogue(sq, sq, None, sq, activation=act).float().sum(), sq)[0]
    gs = torch.autograd.grad(rtx_b200.mxfp8_linear_epilogue(parts[0], parts[1], None, parts[2], activation=act).float().sum(), parts)
    total = sum(t.double() for t in gs)
    assert ((g.double() - total).abs() <= 2 * 2.0 ** -8 * sum(t.double().abs() for t in gs)).all()


def test_captured_graph_and_streams(dev):
    import rtx_b200

    x, w, b, r, dy = inputs(260, 200, 96, seed=10)
    xd, wd, bd, rd, dyd = (t.to(dev) for t in (x, w, b, r, dy))
    leaves = [t.clone().requires_grad_(True) for t in (xd, wd, bd)]

    def step():
        y = rtx_b200.mxfp8_linear_epilogue(*leaves, rd, activation="gelu")
        return (y, *torch.autograd.grad(y, leaves, dyd))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
        graphs.append((graph, out))
    for graph, out in graphs:
        for t in out:
            t.detach().zero_()
    torch.cuda.synchronize()
    for graph, _ in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, e) for a, e in zip(out, eager))
    within(eager[0].detach(), *forward(x, w, b, r, "gelu")[:2])


def test_module_from_float_packed_and_state_dict(dev):
    import rtx_b200

    torch.manual_seed(0)
    ref = torch.nn.Linear(96, 72).to(dev)
    m = rtx_b200.MXFP8LinearEpilogue.from_float(ref, activation="silu")
    x = torch.randn(4, 9, 96, device=dev).bfloat16()
    r = torch.randn(4, 9, 72, device=dev).bfloat16()
    y = m(x, r)
    within(y.detach().view(36, 72), *forward(x.cpu().view(36, 96), m.weight.detach().cpu(), m.bias.detach().cpu(),
                                             r.cpu().view(36, 72), "silu")[:2])
    y.sum().backward()
    assert m.weight.grad.shape == m.weight.shape and m.bias.grad.shape == m.bias.shape
    packed = m.to_quantized_weight()
    with torch.no_grad():
        assert torch.equal(packed(x, r), y)
    other = rtx_b200.MXFP8LinearEpilogue(96, 72, activation="silu", device=dev)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x, r), y)
    assert rtx_b200.MXFP8LinearEpilogue(96, 72, bias=False, device=dev)(x).shape == (4, 9, 72)
    assert m(x[:0]).shape == (0, 9, 72)
    z = x[:0].clone().requires_grad_(True)
    m.zero_grad()
    m(z).sum().backward()
    assert (m.weight.grad == 0).all() and (m.bias.grad == 0).all()


def test_compiled_graph_gives_the_same_bits(dev):
    import rtx_b200

    x, w, b, r, dy = (t.to(dev) for t in inputs(40, 72, 64, seed=11))
    w.requires_grad_(True)
    fn = torch.compile(lambda *t: rtx_b200.mxfp8_linear_epilogue(*t, activation="gelu") * 2, fullgraph=True)
    y, want = fn(x, w, b, r), rtx_b200.mxfp8_linear_epilogue(x, w, b, r, activation="gelu") * 2
    assert torch.equal(y, want)
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], torch.autograd.grad(want, w, dy)[0])


def test_experts_and_epilogue_as_used_together(dev):
    """A feed-forward block with experts: projection with bias and activation, experts' up and down products, the output
    projection added to the residual stream; forward and every gradient against the same chain taken operator by
    operator in 64 bits (each operator on what the one before returned)."""
    import rtx_b200

    x, w_in, b_in, _, dy = inputs(100, 96, 96, seed=12)
    gen = torch.Generator().manual_seed(13)
    w_up = (torch.randn(3, 128, 96, generator=gen) / 96 ** 0.5).bfloat16()
    w_out = (torch.randn(96, 128, generator=gen) / 128 ** 0.5).bfloat16()
    offsets = torch.tensor([0, 30, 30, 100], dtype=torch.int32)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w_in, b_in, w_up, w_out)]
    xd, wi, bi, wu, wo = leaves
    h = rtx_b200.mxfp8_linear_epilogue(xd, wi, bi, activation="relu2")
    e = rtx_b200.mxfp8_grouped_linear(h, wu, offsets.to(dev))
    y = rtx_b200.mxfp8_linear_epilogue(e, wo, None, xd)
    h.retain_grad(), e.retain_grad()
    y.backward(dy.to(dev))
    within(h.detach(), *forward(x, w_in, b_in, None, "relu2")[:2])
    hc, ec = h.detach().cpu(), e.detach().cpu()
    for a, b, g in ((0, 30, 0), (30, 100, 2)):
        within(e.detach()[a:b], *forward(hc[a:b], w_up[g], None, None, "none")[:2])
    within(y.detach(), *forward(ec, w_out, None, x, "none")[:2])
    last = backward(dy, dy, ec, w_out, "none")
    within(e.grad, *last["dx"])
    within(wo.grad, *last["dw"])
    eg = e.grad.cpu()
    for a, b, g in ((0, 30, 0), (30, 100, 2)):
        part = backward(eg[a:b], eg[a:b], hc[a:b], w_up[g], "none")
        within(h.grad[a:b], *part["dx"])
        within(wu.grad[g], *part["dw"])
    assert (wu.grad[1] == 0).all()
    from rtx_b200 import ops

    z = ops.mxfp8_linear_epilogue_fwd(x.to(dev), w_in.to(dev), b_in.to(dev), activation="relu2", keep_z=True)[1].cpu()
    first = backward(h.grad.cpu(), z, x, w_in, "relu2")
    within(wi.grad, *first["dw"])
    within(bi.grad, *first["db"])
    # x has two uses: the residual's gradient dy and dx, added in BF16
    want, bound = first["dx"]
    total = want + dy.double()
    within(xd.grad, total, 2.0 ** -8 * total.abs() + (1 + 2.0 ** -8) * bound)


@pytest.mark.parametrize("m,n,k", [(300, 222, 386), (131, 255, 97), (257, 33, 520), (150, 129, 64)])
def test_every_alignment_gives_the_same_bits(dev, m, n, k):
    """Operands in wider tensors of NaN, at every two-byte place: the bits of the contiguous ones, which are right."""
    import rtx_b200

    x, w, b, r, dy = inputs(m, n, k, seed=22)
    xd, wd, bd, rd, dyd = (t.to(dev) for t in (x, w, b, r, dy))
    z = rtx_b200.mxfp8_linear_epilogue(xd, wd, bd)
    y = rtx_b200.mxfp8_linear_epilogue(xd, wd, bd, rd, activation="gelu")
    grads = rtx_b200.mxfp8_linear_epilogue_backward(dyd, z, xd, wd, activation="gelu")
    within(y, *forward(x, w, b, r, "gelu")[:2])
    for got, (want, bound) in zip(grads, backward(dy, z.cpu(), x, w, "gelu").values()):
        within(got, want, bound)

    def moved(t, pad, lead):
        flat = torch.full((t.shape[0] * (t.shape[1] + pad) + lead + 8,), float("nan"), dtype=torch.bfloat16, device=dev)
        view = flat.as_strided(t.shape, (t.shape[1] + pad, 1), lead)
        view.copy_(t)
        return view

    for pad, lead in ((0, 1), (0, 2), (1, 0), (1, 4), (1, 3), (2, 0), (2, 6), (7, 5), (8, 8)):
        xv, rv, dyv, wv = moved(xd, pad, lead), moved(rd, pad, lead), moved(dyd, pad, lead), moved(wd, 0, lead)
        bv = moved(bd[None], 0, lead)[0]
        zv = moved(z, 0, lead)
        assert torch.equal(rtx_b200.mxfp8_linear_epilogue(xv, wv, bv, rv, activation="gelu"), y), (pad, lead)
        got = rtx_b200.mxfp8_linear_epilogue_backward(dyv, zv, xv, wv, activation="gelu")
        for a, c in zip(got, grads):
            assert torch.equal(a, c), (pad, lead)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_small_slopes_keep_their_relative_accuracy(dev, act):
    """One row, so that dbias is dz: every BF16 z in [-64, -2], where the slopes fall from 0.1 to nothing.

    Beside the BF16 rounding: the exponent (up to z^2 / 2 = 90 where a slope above 1e-30 is left) is off by a rounding or
    two, 90 * 2^-22 = 2^-15 of the slope, a dozen other roundings less than that; gelu's Phi(z) is off by at most 0.08 of
    itself and 1 / z^2 of the slope there, at most 3e-4 over this range (at z = -12: 0.032 / 144).  2^-11 covers both."""
    import rtx_b200

    bits = torch.arange(0xC000, 0xC281, dtype=torch.int32)              # -2 ... -64
    z = (bits - 65536).to(torch.int16).view(torch.bfloat16)[None]
    assert z[0, 0] == -2 and z[0, -1] == -64
    n = z.shape[1]
    x, w = torch.zeros(1, 32, dtype=torch.bfloat16), torch.zeros(n, 32, dtype=torch.bfloat16)
    db = rtx_b200.mxfp8_linear_epilogue_backward(torch.ones(1, n, device=dev).bfloat16(), z.to(dev), x.to(dev), w.to(dev),
                                                 activation=act)[2].double().cpu()
    want = slope64(z[0].double(), act)
    live = want.abs() > 1e-30
    off = (db - want).abs()[live] / want.abs()[live]
    assert live.sum() > 150 and (off <= 2.0 ** -8 + 2.0 ** -11).all(), off.max().item()
    assert (db.abs() <= 2 * want.abs() + 1e-36).all()


def test_replaced_packed_storage_is_used(dev):
    """A packed weight whose storage is exchanged (a reload in place) is read where it now is."""
    import rtx_b200

    x, w, b, r, _ = (t.to(dev) for t in inputs(20, 64, 96, seed=18))
    packed, other = rtx_b200.quantize_mxfp8(w), rtx_b200.quantize_mxfp8(2 * w.flip(0))
    first = rtx_b200.mxfp8_linear_epilogue(x, packed, b, r)
    want = rtx_b200.mxfp8_linear_epilogue(x, other, b, r)
    packed.qdata.data, packed.scale.data = other.qdata.data, other.scale.data
    got = rtx_b200.mxfp8_linear_epilogue(x, packed, b, r)
    assert torch.equal(got, want) and not torch.equal(got, first)


def test_forward_mode_is_refused(dev):
    import rtx_b200
    from torch.autograd import forward_ad

    x, w, b, r, _ = (t.to(dev) for t in inputs(20, 32, 32, seed=19))
    with forward_ad.dual_level():
        rtx_b200.mxfp8_linear_epilogue(x, w, b, r)                      # no tangents: nothing to drop
        for i in range(4):
            args = [x, w, b, r]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                rtx_b200.mxfp8_linear_epilogue(*args)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rtx_b200.mxfp8_linear_epilogue(forward_ad.make_dual(x, torch.ones_like(x)), rtx_b200.quantize_mxfp8(w), b, r)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rtx_b200.mxfp8_linear_epilogue_backward(forward_ad.make_dual(r, torch.ones_like(r)), None, x, w)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: rtx_b200.mxfp8_linear_epilogue(t, w, b, r), (x,), (torch.ones_like(x),))


def test_vmap_runs_one_call_after_the_other(dev):
    import rtx_b200

    x, w, b, r, _ = (t.to(dev) for t in inputs(40, 32, 48, seed=20))
    got = torch.func.vmap(lambda a, c: rtx_b200.mxfp8_linear_epilogue(a, w, b, c, activation="silu"))(
        x.view(2, 20, 48), r.view(2, 20, 32))
    want = [rtx_b200.mxfp8_linear_epilogue(x[i:i + 20], w, b, r[i:i + 20], activation="silu") for i in (0, 20)]
    assert torch.equal(got, torch.stack(want))


def test_second_derivatives_are_refused(dev):
    import rtx_b200

    x, w, b, r, dy = (t.to(dev) for t in inputs(20, 32, 32, seed=14))
    x.requires_grad_(True)
    g = torch.autograd.grad(rtx_b200.mxfp8_linear_epilogue(x, w, b, activation="silu"), x, dy.requires_grad_(True),
                            create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_packed_module_under_compile_and_with_leading_dimensions(dev):
    import rtx_b200

    torch.manual_seed(1)
    m = rtx_b200.MXFP8LinearEpilogue(96, 72, activation="gelu", device=dev).to_quantized_weight()
    x = torch.randn(2, 3, 96, device=dev).bfloat16()
    r = torch.randn(2, 3, 72, device=dev).bfloat16()
    y = m(x, r)
    assert y.shape == (2, 3, 72)
    assert torch.equal(torch.compile(lambda a, c: m(a, c), fullgraph=True)(x, r), y)
    assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x, m.packed_weight(), m.bias, r, activation="gelu"), y)
    one = rtx_b200.mxfp8_linear_epilogue(x[0, 0], m.packed_weight(), m.bias, activation="gelu")
    assert one.shape == (72,) and torch.equal(one, m(x[0, 0]))


def test_row_major_packed_scales(dev):
    """A packed weight whose scales are stored row-major is re-tiled on the way in."""
    import rtx_b200
    from rtx_b200.formats import convert_mxfp8_scale_layout

    x, w, b, _, _ = (t.to(dev) for t in inputs(20, 200, 96, seed=15))
    packed = rtx_b200.quantize_mxfp8(w)
    rows = convert_mxfp8_scale_layout(packed, "row_major")
    want = rtx_b200.mxfp8_linear_epilogue(x, packed, b)
    assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x, rows, b), want)
    assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x, rows, b), want)


def test_replaced_packed_storage_is_noticed(dev):
    import rtx_b200

    x, w, _, _, _ = (t.to(dev) for t in inputs(20, 128, 96, seed=16))
    packed, other = rtx_b200.quantize_mxfp8(w), rtx_b200.quantize_mxfp8(-w)
    rtx_b200.mxfp8_linear_epilogue(x, packed)
    packed.qdata, packed.scale = other.qdata, other.scale
    assert torch.equal(rtx_b200.mxfp8_linear_epilogue(x, packed), rtx_b200.mxfp8_linear_epilogue(x, other))


@pytest.mark.parametrize("m,n,k", [(140_000, 64, 16_384), (70_000, 32_768, 32)])
def test_operands_beyond_32_bit_offsets(dev, m, n, k):
    """More than 2^31 values in x, respectively in the result: the last rows have the bits of a call on those rows alone."""
    import rtx_b200

    tail = slice(m - 200, m)
    x = torch.randn(m, k, device=dev, dtype=torch.bfloat16)
    w = torch.randn(n, k, device=dev, dtype=torch.bfloat16)
    b = torch.randn(n, device=dev, dtype=torch.bfloat16)
    r = torch.randn(m, n, device=dev, dtype=torch.bfloat16)
    y = rtx_b200.mxfp8_linear_epilogue(x, w, b, r, activation="silu")
    assert torch.equal(y[tail], rtx_b200.mxfp8_linear_epilogue(x[tail], w, b, r[tail], activation="silu"))
    dx = rtx_b200.mxfp8_linear_epilogue_backward(r, y, x, w, activation="silu", bias=False)[0]
    assert torch.equal(dx[tail], rtx_b200.mxfp8_linear_epilogue_backward(r[tail], y[tail].contiguous(), x[tail], w,
                                                                         activation="silu", bias=False)[0])


def test_two_threads_at_once(dev):
    """Two threads on two streams: launch state is per thread, scratch per call."""
    import threading

    import rtx_b200

    cases = [tuple(t.to(dev) for t in inputs(300, 256, 128, seed=s)[:4]) for s in (20, 21)]
    want = [rtx_b200.mxfp8_linear_epilogue(*c, activation="silu") for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got[i].append(rtx_b200.mxfp8_linear_epilogue(*cases[i], activation="silu"))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 50 and all(torch.equal(y, want[i]) for y in got[i])
