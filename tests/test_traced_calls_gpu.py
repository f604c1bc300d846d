"""The log-probability and embedding entries under tracers, dispatch modes and differentiation of other
kinds: the call is recorded and runs with new inputs, or is refused."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from unifiedlm_c_b200.clip import clip_grads, grad_norm
from unifiedlm_c_b200.embed import embedding
from unifiedlm_c_b200.logprobs import lm_head_logprobs, token_logprobs

pytestmark = pytest.mark.gpu


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


def inputs():
    gen = torch.Generator().manual_seed(0)
    w = torch.randn(50, 16, generator=gen).cuda()
    t = torch.randint(0, 16, (6,), generator=gen).cuda()
    return w, t, torch.randn(20, 16, generator=gen).cuda(), torch.randn(20, 16, generator=gen).cuda()


def calls(w, t):
    return dict(lm_head_logprobs=lambda x: tuple(lm_head_logprobs(x[:6], w, t, top_k=2)),
                token_logprobs=lambda x: tuple(token_logprobs(x[:6], t, top_k=2)),
                embedding=lambda x: (embedding(t, x, scale=2.0),))


NAMES = ["lm_head_logprobs", "token_logprobs", "embedding"]


@pytest.mark.parametrize("name", NAMES)
def test_traced_programs_make_the_call(name):
    w, t, a, b = inputs()
    f = calls(w, t)[name]
    want = f(b)
    for g in (make_fx(f)(a), make_fx(f, pre_dispatch=True)(a), torch.jit.trace(f, (a,))):
        assert all(torch.equal(x, y) for x, y in zip(g(b), want))


@pytest.mark.parametrize("name", NAMES)
def test_dispatch_modes_see_the_call(name):
    w, t, a, _ = inputs()
    f = calls(w, t)[name]
    with Seen() as seen:
        got = f(a)
    assert f"ulm.{name}_fwd.default" in seen.names
    assert all(torch.equal(x, y) for x, y in zip(got, f(a)))
    x = a.clone().requires_grad_()
    with Seen() as seen:
        f(x)[0].sum().backward()
    assert f"ulm.{name}_bwd.default" in seen.names
    y = a.clone().requires_grad_()
    f(y)[0].sum().backward()
    assert torch.equal(x.grad, y.grad)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    w, t, a, b = inputs()
    f = calls(w, t)[name]
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(a, b))
        assert all(torch.equal(x, y) for x, y in zip(f(a), f(a)))  # without a tangent as ever
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (a,), (b,))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: f(x)[0].sum())(a)


def test_clipping_is_not_traced():
    w, _, a, b = inputs()
    calls = (lambda x: grad_norm([x]), lambda x: clip_grads([x], 1.0, out=[w[:20]]), lambda x: clip_grads([x], 1.0))
    for f in calls:
        before = a.clone()
        for way in (lambda: make_fx(f)(a), lambda: make_fx(f, pre_dispatch=True)(a), lambda: torch.jit.trace(f, (a,)),
                    lambda: torch.func.vmap(f)(torch.stack([a, b]))):
            with pytest.raises(RuntimeError, match="traced"):
                way()
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(forward_ad.make_dual(a, b))
        assert torch.equal(a, before)


def test_clipping_where_something_looks_on():
    """A dispatch mode that records nothing, and torch.compile, which breaks its graph at the call."""
    _, _, a, _ = inputs()
    want = clip_grads([a], 1.0, out=[torch.empty_like(a)])
    with Seen():
        assert torch.equal(clip_grads([a], 1.0, out=[torch.empty_like(a)]), want)
    f = torch.compile(lambda x: clip_grads([x * 1.0], 1.0), backend="eager")
    assert torch.equal(f(a), want)
