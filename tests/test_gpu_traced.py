"""The grouped linear and the linear with an epilogue where something else has to see their ops: `make_fx`,
`torch.jit.trace`, a dispatch mode.  What they record is replayed on other inputs and has to give the eager call's bits."""
import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev(native_lib):
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device")
    torch.cuda.set_device(0)
    return torch.device("cuda", 0)


def calls(dev):
    """{name: (function of tensors alone, its inputs, others of the same shapes, the op that a graph of it holds)}"""
    import rtx_b200 as r

    gen = torch.Generator(device=dev).manual_seed(5)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev).bfloat16()

    offsets = [torch.tensor(o, dtype=torch.int32, device=dev) for o in ((0, 20, 20, 66), (3, 5, 40, 70))]
    wp, gp = r.quantize_mxfp8(normal(72, 96)), r.quantize_mxfp8(normal(3, 128, 96))

    def two(make):
        return make(0), make(1)

    x2 = lambda i: (normal(70, 96),)
    return {
        "grouped": (r.mxfp8_grouped_linear, *two(lambda i: (*x2(i), normal(3, 72, 96), offsets[i])), "mxfp8_grouped_linear"),
        "grouped packed": (lambda x, o: r.mxfp8_grouped_linear(x, gp, o), *two(lambda i: (*x2(i), offsets[i])),
                           "mxfp8_grouped_linear_prequant_w"),
        "grouped backward": (r.mxfp8_grouped_linear_backward,
                             *two(lambda i: (normal(70, 72), *x2(i), normal(3, 72, 96), offsets[i])), "mxfp8_grouped_linear_bwd"),
        "epilogue": (lambda x, w, b, res: r.mxfp8_linear_epilogue(x, w, b, res, activation="gelu"),
                     *two(lambda i: (*x2(i), normal(72, 96), normal(72), normal(70, 72))), "mxfp8_linear_epilogue"),
        "epilogue packed": (lambda x, b: r.mxfp8_linear_epilogue(x, wp, b, activation="silu"),
                            *two(lambda i: (*x2(i), normal(72))), "mxfp8_linear_epilogue_prequant_w"),
        "epilogue backward": (lambda dy, z, x, w: r.mxfp8_linear_epilogue_backward(dy, z, x, w, activation="gelu_tanh"),
                              *two(lambda i: (normal(70, 72), normal(70, 72), *x2(i), normal(72, 96))),
                              "mxfp8_linear_epilogue_bwd"),
    }


NAMES = ["grouped", "grouped packed", "grouped backward", "epilogue", "epilogue packed", "epilogue backward"]


def same(got, want):
    got, want = (v if isinstance(v, (tuple, list)) else [v] for v in (got, want))
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.dtype is b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("mode", ["real", "fake"])
def test_make_fx_graph(dev, name, mode):
    f, first, other, op = calls(dev)[name]
    graph = make_fx(f, tracing_mode=mode, _allow_non_fake_inputs=True)(*first)   # packed weights are the graph's own
    assert [n for n in graph.graph.nodes if str(n.target) == f"rtx.{op}.default"], graph.graph
    same(graph(*other), f(*other))


@pytest.mark.parametrize("name", NAMES)
def test_jit_trace_graph(dev, name):
    f, first, other, op = calls(dev)[name]
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        graph = torch.jit.trace(f, first, check_trace=False)
    assert f"rtx::{op}(" in str(graph.graph)
    same(graph(*other), f(*other))


@pytest.mark.parametrize("name", NAMES)
def test_a_dispatch_mode_sees_the_op(dev, name):
    f, first, _, op = calls(dev)[name]
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    want = f(*first)
    with Watch():
        got = f(*first)
    assert f"rtx.{op}.default" in seen
    same(got, want)


@pytest.mark.parametrize("name", ["grouped", "epilogue"])
def test_traced_graphs_of_trainable_weights_are_differentiable(dev, name):
    """The recorded op carries its gradient: a replayed graph's gradients are the eager call's."""
    f, first, other, _ = calls(dev)[name]
    leaves = [t.requires_grad_(True) for t in other if t.is_floating_point()]
    traced = tuple(t.requires_grad_(True) if t.is_floating_point() else t for t in first)
    y = f(*other)
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, leaves, dy)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        graphs = [make_fx(f)(*traced), torch.jit.trace(f, traced, check_trace=False)]
    for graph in graphs:
        out = graph(*other)
        same(out, y)
        same(torch.autograd.grad(out, leaves, dy), want)

    # a whole step, its backward inside the graph
    def step(*args):
        args = [a.detach().requires_grad_(a.is_floating_point()) for a in args]
        return torch.autograd.grad(f(*args), [a for a in args if a.requires_grad], dy)

    same(make_fx(step)(*first)(*other), want)


@pytest.mark.parametrize("name", ["grouped", "epilogue"])
def test_vmap_over_trainable_weights(dev, name):
    """One call after the other, with the gradients of both in the shared operands."""
    f, first, other, _ = calls(dev)[name]
    rest = tuple(t.requires_grad_(True) if t.is_floating_point() else t for t in first[1:])
    leaves = [t for t in rest if t.is_floating_point()]
    x = torch.stack([first[0], other[0]]).requires_grad_(True)
    y = torch.func.vmap(f, (0, *[None] * len(rest)))(x, *rest)
    want = torch.stack([f(a, *rest) for a in x])
    same(y, want)
    dy = torch.randn_like(want)
    same(torch.autograd.grad(y, [x, *leaves], dy, retain_graph=True), torch.autograd.grad(want, [x, *leaves], dy))


@pytest.mark.parametrize("name", ["grouped", "epilogue"])
def test_func_transforms(dev, name):
    """grad, vjp and jacrev, alone and around or inside vmap, give autograd's gradients."""
    f, first, other, _ = calls(dev)[name]
    rest = first[1:]
    leaves = [t.requires_grad_(True) for t in first if t.is_floating_point()]
    numbers = tuple(i for i, t in enumerate(first) if t.is_floating_point())
    dy = torch.randn_like(f(*first))
    want = torch.autograd.grad(f(*first), leaves, dy)
    loss = lambda *args: (f(*args) * dy).sum()
    same(torch.func.grad(loss, argnums=numbers)(*first), want)
    same(torch.func.grad(loss, argnums=numbers)(*(t.detach() for t in first)), want)
    y, pull = torch.func.vjp(lambda *args: f(*args, *first[len(numbers):]), *leaves)
    same(y, f(*first))
    same(pull(dy), want)
    xs = torch.stack([first[0], other[0]]).detach()
    each = [torch.autograd.grad(loss(x, *rest), leaves[1:]) for x in xs]
    over = (0, *[None] * len(rest))
    got = torch.func.vmap(torch.func.grad(loss, argnums=numbers[1:]), over)(xs, *rest)   # a gradient per sample
    same(got, [torch.stack(g) for g in zip(*each)])
    around = torch.func.grad(lambda *args: (torch.func.vmap(f, over)(xs, *args) * dy).sum(), argnums=tuple(range(len(leaves) - 1)))
    same(around(*rest), [a + b for a, b in zip(*each)])
    some = torch.func.jacrev(lambda x: f(x, *rest)[4, :3])(first[0])
    for i in range(3):
        pick = torch.zeros_like(dy)
        pick[4, i] = 1
        same(some[i], torch.autograd.grad(f(*first), first[0], pick)[0])
    assert torch.equal(torch.func.functionalize(f)(*(t.detach() for t in first)), y)
    scaled = torch.func.jvp(lambda s: f(*first) * s, (torch.ones((), device=dev),), (torch.ones((), device=dev),))
    assert torch.equal(scaled[1].bfloat16(), y)                 # constants of a forward-mode call


@pytest.mark.parametrize("name", ["grouped", "epilogue"])
def test_no_form_drops_a_second_derivative(dev, name):
    """Each path refuses it; none gives zeros."""
    f, first, _, _ = calls(dev)[name]
    x, *rest = first
    x.requires_grad_(True)
    loss = lambda x: f(x, *rest).square().sum()

    class Pass(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Pass():                                                # the registered op
        g = torch.autograd.grad(loss(x), x, create_graph=True)[0]
        with pytest.raises(NotImplementedError, match="no derivative of its own"):
            g.sum().backward()
    with pytest.raises(NotImplementedError, match="no derivative of its own"):
        torch.func.grad(lambda x: torch.func.grad(loss)(x).sum())(x)
    g = torch.autograd.grad(loss(x), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("name", ["grouped packed", "grouped backward", "epilogue packed", "epilogue backward"])
def test_transforms_of_what_has_no_derivative_are_refused(dev, name):
    f, first, _, _ = calls(dev)[name]

    def total(*args):
        out = f(*args)
        return sum(t.float().sum() for t in (out if isinstance(out, tuple) else (out,)))

    with pytest.raises(RuntimeError, match="inference-only|no derivative of its own"):
        torch.func.grad(total)(*first)
    over = (None,) * (len(first) - 1)
    with pytest.raises(RuntimeError, match="inference-only|no derivative of its own"):   # the batched operand hides the tracked one
        torch.func.grad(lambda t: torch.func.vmap(total, (0, *over))(torch.stack([t, t]), *first[1:]).sum())(first[0])
    batch = torch.func.vmap(f, (0, *over))(torch.stack([first[0]] * 2), *first[1:])
    same([b[1] for b in batch] if isinstance(batch, tuple) else batch[1], f(*first))


def test_offsets_that_are_no_tensor_are_named(dev):
    import rtx_b200 as r

    x, w = torch.zeros(8, 64, device=dev).bfloat16(), torch.zeros(2, 128, 64, device=dev).bfloat16()
    for weight in (w, r.quantize_mxfp8(w)):
        with pytest.raises(TypeError, match="offsets must be a torch.Tensor"):
            r.mxfp8_grouped_linear(x, weight, [0, 4, 8])


@pytest.mark.parametrize("act", ["none", "relu2"])
def test_func_transforms_without_bias_and_residual(dev, act):
    """What is left out is no operand of a transform; activation "none" keeps no z."""
    import rtx_b200 as r

    x, w, b, res = calls(dev)["epilogue"][1]
    xs = torch.stack([x, x.flip(0)])
    for bias, residual in ((None, None), (b, None), (None, res)):
        f = lambda x, w: r.mxfp8_linear_epilogue(x, w, bias, residual, activation=act)
        same(torch.func.vmap(f, (0, None))(xs, w), torch.stack([f(t, w) for t in xs]))
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        loss = lambda x, w: f(x, w).float().sum()
        want = torch.autograd.grad(loss(*leaves), leaves)
        same(torch.func.grad(loss, argnums=(0, 1))(x, w), want)
        each = torch.func.vmap(torch.func.grad(loss), (0, None))(xs, w)
        same(each[0], want[0])


@pytest.mark.parametrize("name", NAMES)
def test_no_form_drops_a_tangent(dev, name):
    """Forward-mode calls are refused, also where vmap hides the tangent from the function."""
    f, first, _, _ = calls(dev)[name]
    rest = first[1:]

    def total(t):
        out = f(t, *rest)
        return sum(v.float().sum() for v in (out if isinstance(out, tuple) else (out,)))

    x, t = first[0], torch.ones_like(first[0])
    batched = lambda v: torch.func.vmap(total)(torch.stack([v, v])).sum()
    for g in (total, batched):
        with pytest.raises(NotImplementedError):
            torch.func.jvp(g, (x,), (t,))
    # constants of the transform, batched below it, have no tangent to drop
    one = torch.ones((), device=dev)
    part = lambda v: out[0] if isinstance(out := f(v, *rest), tuple) else out
    got = torch.func.jvp(lambda s: torch.func.vmap(part)(torch.stack([x, x])) * s, (one,), (one,))
    same(got[1][1], part(x))
    if name in ("grouped", "epilogue"):
        few = lambda v: f(v.bfloat16(), *rest).float().square().sum()
        with pytest.raises(NotImplementedError):
            torch.func.jvp(torch.func.grad(few), (x,), (t,))                 # forward over reverse


@pytest.mark.parametrize("name", ["grouped", "epilogue"])
def test_checkpointed_training(dev, name):
    """Activation checkpointing, plain and by a policy that names the op, gives the bits of the plain step."""
    import functools

    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

    f, first, _, _ = calls(dev)[name]
    leaves = [t.requires_grad_(True) for t in first if t.is_floating_point()]
    dy = torch.randn_like(f(*first))
    want = torch.autograd.grad(f(*first) * 2, leaves, dy)
    op = torch.ops.rtx.mxfp8_grouped_linear_train if name == "grouped" else torch.ops.rtx.mxfp8_linear_epilogue_train
    named = []

    def policy(ctx, func, *args, **kwargs):
        if func is op.default:
            named.append(func)
            return CheckpointPolicy.MUST_SAVE
        return CheckpointPolicy.PREFER_RECOMPUTE

    run = lambda *args: f(*args) * 2
    for kwargs in ({}, {"context_fn": functools.partial(create_selective_checkpoint_contexts, policy)}):
        y = checkpoint(run, *first, use_reentrant=False, **kwargs)
        same(torch.autograd.grad(y, leaves, dy), want)
    assert named


@pytest.mark.parametrize("name", ["grouped backward", "epilogue backward"])
def test_backward_functions_carry_no_gradient(dev, name):
    """With operands that require one, too: eager, compiled and recorded alike."""
    f, first, other, _ = calls(dev)[name]
    first, other = (tuple(t.requires_grad_(True) if t.is_floating_point() else t for t in v) for v in (first, other))
    want = f(*other)
    compiled = torch.compile(f, fullgraph=True)
    for g in (f, compiled, make_fx(f)(*first), torch.jit.trace(f, first, check_trace=False)):
        got = g(*other)
        same(got, want)
        assert not any(t.requires_grad for t in got)
