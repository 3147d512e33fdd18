"""When the package may call a launcher past the dispatcher (no GPU)."""
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode


def test_whatever_has_to_see_an_op_is_noticed():
    from rtx_b200._oplib import interposed

    seen = {}

    def probe(name):
        def f(t):
            seen[name] = interposed()
            return t * 2
        return f

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    t = torch.ones(3)
    probe("plain")(t)
    for mode in ("real", "fake", "symbolic"):
        make_fx(probe("make_fx " + mode), tracing_mode=mode)(t)
    torch.jit.trace(probe("jit.trace"), t, check_trace=False)
    with Watch():
        probe("dispatch mode")(t)
    torch.func.vmap(probe("vmap"))(t)
    torch.func.grad(lambda v: probe("grad")(v).sum())(t)
    torch.func.functionalize(probe("functionalize"))(t)
    torch.compile(lambda v: v * 2 if interposed() else v * 3, backend="eager", fullgraph=True)
    assert seen.pop("plain") is False
    assert len(seen) == 8 and all(seen.values()), seen
    assert interposed() is False
    assert torch.equal(torch.compile(lambda v: v * 2 if interposed() else v * 3, backend="eager", fullgraph=True)(t), 2 * t)


def test_operands_that_are_not_plain_cuda_tensors_go_through_the_dispatcher():
    from rtx_b200._oplib import eager

    class Wrapped(torch.Tensor):
        pass

    class OnCuda:          # what `eager` asks of its first operand, without a device
        is_cuda = True

    t = torch.ones(3)
    assert not eager(t) and not eager(torch.nn.Parameter(t)) and not eager(OnCuda(), t)
    assert not eager(t, t.as_subclass(Wrapped))
