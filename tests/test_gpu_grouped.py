"""Grouped MXFP8 linear against its definition in 64 bits, at the group sizes, widths, pitches and streams where it can
go wrong.

Tolerance.  The quantized operands are exact in 64 bits, so a result differs from the definition by the FP32
accumulation and one BF16 rounding.  Summing K products in FP32 in any order is off by at most K u S with S the sum of
the products' magnitudes; u = 2^-23 allows for an accumulator that cuts instead of rounding.  The BF16 rounding is off
by at most half a step, 2^-8 of the value (finfo.eps / 2), of a value that is already off by the first term:
|y - exact| <= 2^-8 |exact| + (1 + 2^-8) K 2^-23 S."""
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu


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
    """The values MXFP8 holds of v (blocks along the last dimension), in 64 bits."""
    q, s = O.mxfp8_quantize(v.contiguous())
    return O.mxfp8_dequantize(q, s).double()


def close(got, want, mag, k):
    assert got.dtype is torch.bfloat16 and got.shape == want.shape
    off = (got.double().cpu() - want).abs()
    bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * k * 2.0 ** -23 * mag
    assert (off <= bound).all(), (off - bound).max().item()


def forward(x, w, offsets):
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(y)
    for g, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        if b > a:
            xa, wa = mx(x[a:b]), mx(w[g])
            y[a:b], mag[a:b] = xa @ wa.T, xa.abs() @ wa.abs().T
    return y, mag


def backward(dy, x, w, offsets):
    dx, dw = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(w.shape, dtype=torch.float64)
    dx_mag, dw_mag = torch.zeros_like(dx), torch.zeros_like(dw)
    for g, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        if b > a:
            d, wt = mx(dy[a:b]), mx(w[g].T)
            dx[a:b], dx_mag[a:b] = d @ wt.T, d.abs() @ wt.abs().T
            dt, xt = mx(dy[a:b].T), mx(x[a:b].T)
            dw[g], dw_mag[g] = dt @ xt.T, dt.abs() @ xt.abs().T
    return dx, dw, dx_mag, dw_mag


def inputs(rows, groups, n, k, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen)
    x = torch.where(torch.rand(rows, k, generator=gen) < 0.01, 50 * x, x).bfloat16()
    w = (torch.randn(groups, n, k, generator=gen) / k ** 0.5).bfloat16()
    dy = (0.1 * torch.randn(rows, n, generator=gen)).bfloat16()
    return x, w, dy


def offs(*sizes, head=0):
    out = [head]
    for s in sizes:
        out.append(out[-1] + s)
    return out


def on(dev, offsets):
    return torch.tensor(offsets, dtype=torch.int32, device=dev)


SIZES = [
    (1,), (0, 1, 0), (31, 1, 32, 33), (127, 0, 128, 129), (255, 256, 257), (0, 0, 0), (5, 300, 0, 2), (600,),
]
WIDTHS = [(128, 128), (256, 256), (8, 32), (1, 1), (33, 65), (200, 72), (520, 136), (384, 300)]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("n,k", [(256, 256), (200, 72)])
def test_forward_group_sizes(dev, sizes, n, k):
    import rtx_b200

    offsets = offs(*sizes, head=3)
    x, w, _ = inputs(offsets[-1] + 7, len(sizes), n, k)
    y = rtx_b200.mxfp8_grouped_linear(x.to(dev), w.to(dev), on(dev, offsets))
    close(y, *forward(x, w, offsets), k)


@pytest.mark.parametrize("n,k", WIDTHS)
def test_forward_widths(dev, n, k):
    import rtx_b200

    offsets = offs(40, 0, 129, 3)
    x, w, _ = inputs(offsets[-1], 4, n, k, seed=1)
    y = rtx_b200.mxfp8_grouped_linear(x.to(dev), w.to(dev), on(dev, offsets))
    close(y, *forward(x, w, offsets), k)


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("n,k", [(256, 256), (200, 72)])
def test_backward_group_sizes(dev, sizes, n, k):
    import rtx_b200

    offsets = offs(*sizes, head=3)
    x, w, dy = inputs(offsets[-1] + 7, len(sizes), n, k)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dy.to(dev), x.to(dev), w.to(dev), on(dev, offsets))
    want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
    close(dx, want_dx, dx_mag, n)
    close(dw, want_dw, dw_mag, max(sizes))


@pytest.mark.parametrize("n,k", WIDTHS)
def test_backward_widths(dev, n, k):
    import rtx_b200

    offsets = offs(40, 0, 129, 3)
    x, w, dy = inputs(offsets[-1], 4, n, k, seed=1)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dy.to(dev), x.to(dev), w.to(dev), on(dev, offsets))
    want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
    close(dx, want_dx, dx_mag, n)
    close(dw, want_dw, dw_mag, 129)


@pytest.mark.parametrize("groups", [1, 17, 512])
def test_many_groups_and_larger_operands(dev, groups):
    """More tiles than resident CTAs: the persistent loop, the accumulator windows and the ring wrap around."""
    import rtx_b200

    gen = torch.Generator().manual_seed(5)
    sizes = torch.randint(0, 2 * (3000 // groups) + 2, (groups,), generator=gen).tolist()
    n, k = (1024, 512) if groups < 512 else (128, 128)
    offsets = offs(*sizes)
    x, w, dy = inputs(offsets[-1] + 1, groups, n, k, seed=2)
    xd, wd, dyd, od = x.to(dev), w.to(dev), dy.to(dev), on(dev, offsets)
    close(rtx_b200.mxfp8_grouped_linear(xd, wd, od), *forward(x, w, offsets), k)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dyd, xd, wd, od)
    want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
    close(dx, want_dx, dx_mag, n)
    close(dw, want_dw, dw_mag, max(sizes))


@pytest.mark.parametrize("groups", [30, 31, 32, 33])
def test_list_lengths_around_a_warp(dev, groups):
    """Lists shorter and longer than a warp are read by different code: same results, and the same for a bad list."""
    import rtx_b200
    from rtx_b200 import ops

    gen = torch.Generator().manual_seed(groups)
    sizes = torch.randint(0, 20, (groups,), generator=gen).tolist()
    sizes[0], sizes[-1] = 300, 130
    offsets = offs(*sizes, head=3)
    n, k = 64, 96
    x, w, dy = inputs(offsets[-1] + 5, groups, n, k, seed=4)
    xd, wd, dyd = x.to(dev), w.to(dev), dy.to(dev)
    close(rtx_b200.mxfp8_grouped_linear(xd, wd, on(dev, offsets)), *forward(x, w, offsets), k)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dyd, xd, wd, on(dev, offsets))
    want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
    close(dx, want_dx, dx_mag, n)
    close(dw, want_dw, dw_mag, max(sizes))

    bad = list(offsets)
    bad[groups // 2], bad[-1] = -7, 2 ** 31 - 1
    held = [0] * len(bad)
    for i, v in enumerate(bad):
        held[i] = max(min(max(v, 0), x.shape[0]), held[i - 1] if i else 0)
    y = rtx_b200.mxfp8_grouped_linear(xd, wd, on(dev, bad))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="offsets"):
        ops.check_device_status(dev)
    close(y, *forward(x, w, held), k)


@pytest.mark.parametrize("rows", [1, 4, 48, 400])
def test_packed_weight_gives_the_same_bits_as_the_bf16_weight(dev, rows):
    import rtx_b200

    x, w, _ = inputs(rows, 5, 256, 320, seed=3)
    offsets = offs(0, rows // 2, 0, rows - rows // 2, 0)
    xd, wd, od = x.to(dev), w.to(dev), on(dev, offsets)
    y = rtx_b200.mxfp8_grouped_linear(xd, wd, od)
    assert torch.equal(rtx_b200.mxfp8_grouped_linear(xd, rtx_b200.quantize_mxfp8(wd), od), y)
    close(y, *forward(x, w, offsets), 320)


def test_a_group_gets_the_bits_of_the_dense_linear(dev):
    import rtx_b200

    offsets = offs(130, 7, 300)
    x, w, dy = inputs(437, 3, 256, 384, seed=4)
    xd, wd, dyd, od = x.to(dev), w.to(dev), dy.to(dev), on(dev, offsets)
    y = rtx_b200.mxfp8_grouped_linear(xd, wd, od)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dyd, xd, wd, od)
    for g, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        assert torch.equal(y[a:b], rtx_b200.mxfp8_linear(xd[a:b], wd[g]))
        want_dx, want_dw = rtx_b200.mxfp8_linear_backward(dyd[a:b].contiguous(), xd[a:b].contiguous(), wd[g])
        assert torch.equal(dx[a:b], want_dx) and torch.equal(dw[g], want_dw)


def test_pitches_views_and_unaligned_rows(dev):
    import rtx_b200

    offsets = offs(50, 90, head=2)
    x, w, dy = inputs(150, 2, 128, 96, seed=6)
    want, mag = forward(x, w, offsets)
    wd, od = w.to(dev), on(dev, offsets)
    for pad, lead in ((24, 0), (13, 0), (13, 1), (7, 3)):
        wide = torch.full((150, 96 + pad + lead), float("nan"), dtype=torch.bfloat16, device=dev)
        xs = wide[:, lead:lead + 96]
        xs.copy_(x)
        close(rtx_b200.mxfp8_grouped_linear(xs, wd, od), want, mag, 96)
        wide_dy = torch.full((150, 128 + pad + lead), float("nan"), dtype=torch.bfloat16, device=dev)
        dys = wide_dy[:, lead:lead + 128]
        dys.copy_(dy)
        dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dys, xs, wd, od)
        want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
        close(dx, want_dx, dx_mag, 128)
        close(dw, want_dw, dw_mag, 90)
    # transposed activation, weight view: copied, same result
    close(rtx_b200.mxfp8_grouped_linear(x.T.contiguous().to(dev).T, w.transpose(1, 2).contiguous().to(dev).transpose(1, 2), od),
          want, mag, 96)


@pytest.mark.parametrize("n,k", [(64, 63), (65, 130), (191, 97), (136, 264), (33, 192)])
def test_every_alignment_gives_the_same_bits(dev, n, k):
    """Operands in wider tensors of NaN: pitches odd and even, starts at every two-byte place, groups that begin on odd rows.
    All of them against the contiguous operands' bits, and those against the definition."""
    import rtx_b200

    offsets = offs(45, 1, 140, 66, head=3)
    rows = offsets[-1] + 2
    x, w, dy = inputs(rows, 4, n, k, seed=21)
    xd, wd, dyd, od = x.to(dev), w.to(dev), dy.to(dev), on(dev, offsets)
    y = rtx_b200.mxfp8_grouped_linear(xd, wd, od)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dyd, xd, wd, od)
    close(y, *forward(x, w, offsets), k)
    want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
    close(dx, want_dx, dx_mag, n)
    close(dw, want_dw, dw_mag, 140)

    def moved(t, pad, lead):
        flat = torch.full((t.shape[0] * (t.shape[1] + pad) + lead + 8,), float("nan"), dtype=torch.bfloat16, device=dev)
        view = flat.as_strided(t.shape, (t.shape[1] + pad, 1), lead)
        view.copy_(t)
        return view

    for pad, lead in ((0, 1), (0, 2), (1, 0), (1, 4), (1, 3), (2, 0), (2, 6), (7, 5), (8, 8)):
        xv, dyv = moved(xd, pad, lead), moved(dyd, pad, lead)
        wv = moved(wd.view(-1, k), 0, lead).view(4, n, k)
        assert wv.data_ptr() % 16 == 2 * lead % 16
        assert torch.equal(rtx_b200.mxfp8_grouped_linear(xv, wv, od), y), (pad, lead)
        got_dx, got_dw = rtx_b200.mxfp8_grouped_linear_backward(dyv, xv, wv, od)
        assert torch.equal(got_dx, dx) and torch.equal(got_dw, dw), (pad, lead)


def test_out_argument_with_a_pitch_keeps_what_is_beside_it(dev):
    from rtx_b200 import ops

    offsets = offs(33, 65, head=1)
    x, w, _ = inputs(104, 2, 200, 64, seed=7)
    want, mag = forward(x, w, offsets)
    for pad, lead in ((8, 0), (5, 0), (8, 1)):
        wide = torch.full((104, 200 + pad + lead), 7.0, dtype=torch.bfloat16, device=dev)
        out = wide[:, lead:lead + 200]
        ops.mxfp8_grouped_linear_fwd(x.to(dev), w.to(dev), on(dev, offsets), out=out)
        close(out, want, mag, 64)
        assert (wide[:, :lead] == 7).all() and (wide[:, lead + 200:] == 7).all()


def test_rows_of_no_group_are_not_read(dev):
    """NaN and infinity in rows of no group reach no result: zero there, and the groups' rows unchanged."""
    import rtx_b200

    offsets = offs(40, 60, head=5)
    x, w, dy = inputs(120, 2, 128, 128, seed=8)
    want, mag = forward(x, w, offsets)
    want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
    bad_x, bad_dy = x.clone(), dy.clone()
    for t in (bad_x, bad_dy):
        t[:5] = float("nan")
        t[105:] = float("inf")
    args = (bad_x.to(dev), w.to(dev), on(dev, offsets))
    y = rtx_b200.mxfp8_grouped_linear(*args)
    close(y, want, mag, 128)
    assert (y[:5] == 0).all() and (y[105:] == 0).all()
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(bad_dy.to(dev), *args)
    close(dx, want_dx, dx_mag, 128)
    close(dw, want_dw, dw_mag, 60)


def test_a_nan_stays_in_its_row(dev):
    """A NaN activation (its block's scale becomes NaN) makes its own result row NaN and no other."""
    import rtx_b200

    x, w, _ = inputs(100, 2, 128, 128, seed=9)
    offsets = offs(37, 63)
    want, mag = forward(x, w, offsets)
    x[36, 5] = float("nan")
    y = rtx_b200.mxfp8_grouped_linear(x.to(dev), w.to(dev), on(dev, offsets))
    assert y[36].isnan().all()
    keep = [i for i in range(100) if i != 36]
    close(y[keep], want[keep], mag[keep], 128)


def test_gradients_through_autograd_and_against_differences(dev):
    """Autograd returns the backward's gradients; and the backward is the gradient: on operands that MXFP8 holds
    exactly (small whole numbers) and whose products BF16 holds exactly, the loss is linear in each of x and w, so a
    difference of two losses equals the gradient times the step without any rounding."""
    import rtx_b200

    gen = torch.Generator().manual_seed(10)
    offsets = offs(3, 0, 5)
    x = torch.randint(-1, 2, (8, 32), generator=gen).bfloat16()
    w = torch.randint(-1, 2, (3, 32, 32), generator=gen).bfloat16()
    c = torch.randint(-1, 2, (8, 32), generator=gen).bfloat16()
    od = on(dev, offsets)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = rtx_b200.mxfp8_grouped_linear(xd, wd, od)
    gx, gw = torch.autograd.grad(y, (xd, wd), c.to(dev))
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(c.to(dev), xd.detach(), wd.detach(), od)
    assert torch.equal(gx, dx) and torch.equal(gw, dw)

    def loss(a, b):
        return (rtx_b200.mxfp8_grouped_linear(a.to(dev), b.to(dev), od).double() * c.to(dev).double()).sum().item()

    step_x = torch.randint(-1, 2, x.shape, generator=gen).bfloat16()
    step_w = torch.randint(-1, 2, w.shape, generator=gen).bfloat16()
    assert loss(x + step_x, w) - loss(x - step_x, w) == 2 * (gx.double().cpu() * step_x.double()).sum().item()
    assert loss(x, w + step_w) - loss(x, w - step_w) == 2 * (gw.double().cpu() * step_w.double()).sum().item()


def test_one_gradient_at_a_time(dev):
    import rtx_b200

    offsets = offs(20, 50)
    x, w, dy = inputs(72, 2, 96, 160, seed=11)
    xd, wd, dyd, od = x.to(dev), w.to(dev), dy.to(dev), on(dev, offsets)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dyd, xd, wd, od)
    a = xd.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(rtx_b200.mxfp8_grouped_linear(a, wd, od), a, dyd)[0], dx)
    b = wd.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(rtx_b200.mxfp8_grouped_linear(xd, b, od), b, dyd)[0], dw)
    # an expanded gradient (sum().backward()) is read like any other
    c = xd.clone().requires_grad_(True)
    rtx_b200.mxfp8_grouped_linear(c, wd, od).sum().backward()
    ones = torch.ones(72, 96, dtype=torch.bfloat16, device=dev)
    assert torch.equal(c.grad, rtx_b200.mxfp8_grouped_linear_backward(ones, xd, wd, od)[0])


def test_captured_graph_replays_with_other_offsets_and_inputs(dev):
    import rtx_b200

    x, w, dy = inputs(300, 3, 256, 128, seed=12)
    xd, wd, dyd, od = x.to(dev), w.to(dev), dy.to(dev), on(dev, offs(100, 100, 100))
    rtx_b200.mxfp8_grouped_linear(xd, wd, od)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):     # two graphs on one capture stream: their scratch must not be shared
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = rtx_b200.mxfp8_grouped_linear(xd, wd, od)
            dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dyd, xd, wd, od)
        graphs.append((graph, y, dx, dw))
    for offsets in (offs(300, 0, 0), offs(1, 2, 3, head=290), offs(0, 257, 43)):
        od.copy_(on(dev, offsets))
        x = x.flip(0).contiguous()
        xd.copy_(x)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, *_), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want, mag = forward(x, w, offsets)
        want_dx, want_dw, dx_mag, dw_mag = backward(dy, x, w, offsets)
        for _, y, dx, dw in graphs:
            close(y, want, mag, 128)
            close(dx, want_dx, dx_mag, 256)
            close(dw, want_dw, dw_mag, 300)


def test_two_streams_at_once(dev):
    import rtx_b200

    cases = []
    for seed in range(4):
        x, w, _ = inputs(700, 4, 512, 256, seed=20 + seed)
        offsets = offs(100 * seed, 30, 250, 5)
        cases.append((x.to(dev), w.to(dev), on(dev, offsets), *forward(x, w, offsets)))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for (xd, wd, od, *_), stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                outs.append(rtx_b200.mxfp8_grouped_linear(xd, wd, od))
    torch.cuda.synchronize()
    for i, y in enumerate(outs):
        close(y, *cases[i % 4][3:], 256)


def test_offsets_that_are_no_list_are_held_inside_and_reported(dev):
    """Decreasing or too large offsets: the kernels use the nearest list inside [0, rows] and set the status word."""
    import rtx_b200
    from rtx_b200 import ops

    x, w, _ = inputs(64, 3, 128, 64, seed=13)
    for offsets, held in (([0, 40, 20, 64], [0, 40, 40, 64]), ([0, 10, 20, 500], [0, 10, 20, 64]),
                          ([-5, 10, 20, 30], [0, 10, 20, 30])):
        y = rtx_b200.mxfp8_grouped_linear(x.to(dev), w.to(dev), on(dev, offsets))
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="offsets"):
            ops.check_device_status(dev)
        close(y, *forward(x, w, held), 64)


def test_module_dynamic_packed_and_state_dict(dev):
    import rtx_b200

    torch.manual_seed(0)
    m = rtx_b200.MXFP8GroupedLinear(3, 96, 128, device=dev)
    x = torch.randn(50, 96, device=dev).bfloat16()
    od = on(dev, offs(10, 0, 30, head=4))
    y = m(x, od)
    close(y, *forward(x.cpu(), m.weight.detach().cpu(), offs(10, 0, 30, head=4)), 96)
    y.sum().backward()
    assert m.weight.grad.shape == m.weight.shape and (m.weight.grad[1] == 0).all()
    packed = m.to_quantized_weight()
    assert torch.equal(packed(x, od), y)
    other = rtx_b200.MXFP8GroupedLinear(3, 96, 128, device=dev)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x, od), y)
    assert torch.equal(rtx_b200.mxfp8_grouped_linear(x, packed.packed_weight(), od), y)


def test_compiled_graph_gives_the_same_bits(dev):
    import rtx_b200

    x, w, dy = inputs(60, 2, 128, 64, seed=14)
    xd, wd, od = x.to(dev), w.to(dev).requires_grad_(True), on(dev, offs(20, 30))
    fn = torch.compile(lambda a, b, o: rtx_b200.mxfp8_grouped_linear(a, b, o) * 2, fullgraph=True)
    y = fn(xd, wd, od)
    assert torch.equal(y, rtx_b200.mxfp8_grouped_linear(xd, wd, od) * 2)
    got = torch.autograd.grad(y, wd, dy.to(dev))[0]
    assert torch.equal(got, torch.autograd.grad(rtx_b200.mxfp8_grouped_linear(xd, wd, od) * 2, wd, dy.to(dev))[0])


def test_packed_weight_under_compile(dev):
    import rtx_b200

    x, w, _ = inputs(60, 2, 128, 64, seed=15)
    xd, od = x.to(dev), on(dev, offs(20, 30))
    m = rtx_b200.MXFP8GroupedLinear(2, 64, 128, packed_weight=rtx_b200.quantize_mxfp8(w.to(dev)))
    y = m(xd, od)
    assert torch.equal(torch.compile(lambda a, o: m(a, o), fullgraph=True)(xd, od), y)
    close(y, *forward(x, w, offs(20, 30)), 64)


def test_replaced_packed_storage_is_used(dev):
    """A packed weight whose storage is exchanged (a reload in place) is read where it now is."""
    import rtx_b200

    x, w, _ = inputs(60, 2, 128, 64, seed=17)
    xd, wd, od = x.to(dev), w.to(dev), on(dev, offs(20, 30))
    packed, other = rtx_b200.quantize_mxfp8(wd), rtx_b200.quantize_mxfp8(2 * wd.flip(1))
    first, want = rtx_b200.mxfp8_grouped_linear(xd, packed, od), rtx_b200.mxfp8_grouped_linear(xd, other, od)
    packed.qdata.data, packed.scale.data = other.qdata.data, other.scale.data
    got = rtx_b200.mxfp8_grouped_linear(xd, packed, od)
    assert torch.equal(got, want) and not torch.equal(got, first)


def test_forward_mode_is_refused(dev):
    import rtx_b200
    from torch.autograd import forward_ad

    x, w, _ = inputs(60, 2, 128, 64, seed=18)
    xd, wd, od = x.to(dev), w.to(dev), on(dev, offs(20, 30))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(xd, torch.ones_like(xd))
        for args in ((dual, wd), (xd, forward_ad.make_dual(wd, torch.ones_like(wd))), (dual, rtx_b200.quantize_mxfp8(wd))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                rtx_b200.mxfp8_grouped_linear(*args, od)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rtx_b200.mxfp8_grouped_linear_backward(torch.ones(60, 128, device=dev).bfloat16(), dual, wd, od)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: rtx_b200.mxfp8_grouped_linear(t, wd, od), (xd,), (torch.ones_like(xd),))


def test_vmap_runs_one_call_after_the_other(dev):
    import rtx_b200

    x, w, _ = inputs(60, 2, 128, 64, seed=19)
    xd, wd, od = x.to(dev), w.to(dev), on(dev, offs(10, 15, head=2))
    got = torch.func.vmap(lambda t: rtx_b200.mxfp8_grouped_linear(t, wd, od))(xd.view(2, 30, 64))
    assert torch.equal(got, torch.stack([rtx_b200.mxfp8_grouped_linear(t, wd, od) for t in xd.view(2, 30, 64)]))


def test_second_derivatives_are_refused(dev):
    import rtx_b200

    x, w, dy = inputs(40, 2, 64, 64, seed=16)
    xd = x.to(dev).requires_grad_(True)
    y = rtx_b200.mxfp8_grouped_linear(xd, w.to(dev), on(dev, offs(10, 30)))
    g = torch.autograd.grad(y, xd, dy.to(dev).requires_grad_(True), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_offsets_changed_between_forward_and_backward_are_refused(dev):
    """The backward needs the forward's offsets: writing into them in between is caught by autograd's version count."""
    import rtx_b200

    x, w, dy = inputs(40, 2, 64, 64, seed=17)
    xd, od = x.to(dev).requires_grad_(True), on(dev, offs(10, 30))
    y = rtx_b200.mxfp8_grouped_linear(xd, w.to(dev), od)
    od.copy_(on(dev, offs(20, 20)))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy.to(dev))


def test_empty_batch(dev):
    import rtx_b200

    w = torch.randn(2, 64, 32, device=dev).bfloat16().requires_grad_(True)
    x = torch.empty(0, 32, dtype=torch.bfloat16, device=dev, requires_grad=True)
    y = rtx_b200.mxfp8_grouped_linear(x, w, on(dev, offs(0, 0)))
    assert y.shape == (0, 64)
    y.sum().backward()
    assert x.grad.shape == (0, 32) and (w.grad == 0).all()


def test_shared_weights_and_expanded_inputs(dev):
    """One weight expanded over the groups, one row expanded over the batch: copied on the way in, gradients summed."""
    import rtx_b200

    gen = torch.Generator().manual_seed(18)
    w1 = torch.randint(-1, 2, (1, 32, 32), generator=gen).bfloat16().to(dev).requires_grad_(True)
    row = torch.randint(-1, 2, (1, 32), generator=gen).bfloat16().to(dev).requires_grad_(True)
    od = on(dev, offs(3, 2))
    y = rtx_b200.mxfp8_grouped_linear(row.expand(5, 32), w1.expand(2, 32, 32), od)
    want = row.detach().double() @ w1.detach()[0].double().T
    assert torch.equal(y.double(), want.expand(5, 32))        # small whole numbers: exact throughout
    y.sum().backward()
    assert torch.equal(row.grad.double(), 5 * w1.detach()[0].double().sum(0, keepdim=True))
    assert torch.equal(w1.grad[0].double(), 5 * row.detach().double().expand(32, 32))


@pytest.mark.parametrize("rows,n,k", [(140_000, 64, 16_384), (70_000, 32_768, 32)])
def test_operands_beyond_32_bit_offsets(dev, rows, n, k):
    """More than 2^31 values in x, respectively in the result: the last group's rows, and its gradients, have the bits of
    a call on those rows alone."""
    import rtx_b200

    last = 300
    x = torch.randn(rows, k, device=dev, dtype=torch.bfloat16)
    w = torch.randn(2, n, k, device=dev, dtype=torch.bfloat16)
    od, alone = on(dev, offs(rows - last - 5, last)), on(dev, offs(last))
    assert max(rows * k, rows * n) > 2 ** 31
    y = rtx_b200.mxfp8_grouped_linear(x, w, od)
    tail = slice(rows - last - 5, rows - 5)
    assert torch.equal(y[tail], rtx_b200.mxfp8_grouped_linear(x[tail], w[1:], alone))
    assert (y[-5:] == 0).all()
    dy = y.mul_(2.0 ** -8)
    dx, dw = rtx_b200.mxfp8_grouped_linear_backward(dy, x, w, od)
    want_dx, want_dw = rtx_b200.mxfp8_grouped_linear_backward(dy[tail], x[tail], w[1:], alone)
    assert torch.equal(dx[tail], want_dx) and torch.equal(dw[1], want_dw[0]) and (dx[-5:] == 0).all()
