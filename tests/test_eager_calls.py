"""When an entry may call the library directly (`_lib.eager`): not while something traces, transforms,
observes or fakes the call, which then goes through the dispatcher."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.flop_counter import FlopCounterMode

import unifiedlm_c_b200._lib as L


class Seen(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class Own(torch.Tensor):
    pass


def run_mode(mode):
    def run(f):
        with mode():
            f(torch.ones(3))
    return run


def dual(f):
    with forward_ad.dual_level():
        f(forward_ad.make_dual(torch.ones(3), torch.ones(3)))


ways = dict(
    make_fx=lambda f: make_fx(f)(torch.ones(3)),
    make_fx_pre_dispatch=lambda f: make_fx(f, pre_dispatch=True)(torch.ones(3)),
    make_fx_symbolic=lambda f: make_fx(f, tracing_mode="symbolic")(torch.ones(3)),
    jit_trace=lambda f: torch.jit.trace(f, (torch.ones(3),), check_trace=False),
    grad=lambda f: torch.func.grad(lambda x: f(x).sum())(torch.ones(3)),
    vmap=lambda f: torch.func.vmap(f)(torch.ones(3, 2)),
    jvp=lambda f: torch.func.jvp(f, (torch.ones(3),), (torch.ones(3),)),
    functionalize=lambda f: torch.func.functionalize(f)(torch.ones(3)),
    dual=dual,
    mode=run_mode(Seen),
    flops=run_mode(lambda: FlopCounterMode(display=False)),
    fake=run_mode(FakeTensorMode),
    subclass=lambda f: f(torch.ones(3).as_subclass(Own)),
    compiled=lambda f: torch.compile(f, backend="eager", fullgraph=True)(torch.ones(3)),
)


@pytest.mark.parametrize("way", sorted(ways))
def test_not_eager(way):
    seen = []

    def f(x):
        if way == "compiled":  # (a list of the outside is not traced: the answer comes back in the value)
            return x + (1 if L.eager(x) else 0)
        seen.append(L.eager(x))
        return x * 2

    got = ways[way](f)
    if way == "compiled":
        assert torch.equal(got, torch.ones(3))
    else:
        assert seen and not any(seen)


def test_eager():
    assert L.eager(torch.ones(3), torch.nn.Parameter(torch.ones(2)))
    with torch.no_grad():
        assert L.eager(torch.ones(3))
    with torch.inference_mode():
        assert L.eager(torch.ones(3))
    seen = []
    x = torch.ones(3, requires_grad=True)
    y = x * 2
    y.register_hook(lambda g: seen.append(L.eager(g)))
    torch.utils.checkpoint.checkpoint(lambda z: seen.append(L.eager(z)) or z * 3, y, use_reentrant=False).sum().backward()
    assert seen and all(seen)
