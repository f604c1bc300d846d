"""The token embedding and its gradient (embed.embedding) against the definition in float64: types,
odd widths, strides, scales, padding, one hot token, and positions in every order. y is one product
rounded once; the gradient adds at most c rows per token one after another in fp32 (c the token's
count), each step off by 2^-24 of the sum of magnitudes, then rounds once to its type."""
import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.embed import embedding

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def check(tokens, V, D, dtype, scale=1.0, out_dtype=None, weight=None, gen=None):
    gen = gen or torch.Generator().manual_seed(V + D)
    w = (torch.randn(V, D, generator=gen).to(dtype).cuda() if weight is None else weight).requires_grad_()
    y = embedding(tokens, w, scale=scale, out_dtype=out_dtype)
    assert y.shape == (*tokens.shape, D) and y.dtype == (out_dtype or dtype)
    t = tokens.reshape(-1)
    keep = (t >= 0).double()[:, None]
    want = w.detach().double()[t.clamp(min=0)] * scale * keep
    err = (y.detach().double().view(-1, D) - want).abs()
    assert bool((err <= (HALF[y.dtype] + 2 * U) * want.abs()).all())
    dy = torch.randn(y.shape, generator=gen).to(y.dtype).cuda()
    dw, = torch.autograd.grad(y, w, dy)
    assert dw.dtype == dtype and dw.shape == w.shape
    g = dy.double().view(-1, D) * scale * keep
    want = torch.zeros(V, D, dtype=torch.float64).cuda().index_add_(0, t.clamp(min=0), g)
    mag = torch.zeros(V, D, dtype=torch.float64).cuda().index_add_(0, t.clamp(min=0), g.abs())
    count = torch.zeros(V, dtype=torch.float64).cuda().index_add_(0, t.clamp(min=0), keep[:, 0])
    tol = mag * (count[:, None] + 2) * U + HALF[dtype] * want.abs()
    assert bool(((dw.double() - want).abs() <= tol).all())
    assert L.device_error() == 0
    return y, dw


def zipf(n, V, gen):
    p = torch.arange(1, V + 1).double() ** -1.1
    t = torch.multinomial(p / p.sum(), n, replacement=True, generator=gen)
    t[torch.rand(n, generator=gen) < 0.05] = -1
    return t.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 32000, 768), (5, 3, 7), (77, 4099, 288), (1000, 300, 33), (4096, 32000, 96),
                                   (9000, 50, 1030), (33000, 70000, 16), (70000, 1000, 24)])
def test_embedding(dtype, N, V, D):
    gen = torch.Generator().manual_seed(N + D)
    check(zipf(N, V, gen), V, D, dtype, gen=gen)


@pytest.mark.parametrize("scale", [0.0, -1.5, 768.0 ** 0.5])
def test_scale_and_types(scale):
    gen = torch.Generator().manual_seed(1)
    check(zipf(300, 100, gen).view(3, 100), 100, 64, torch.bfloat16, scale=scale, gen=gen)
    check(zipf(300, 100, gen).view(3, 4, 25), 100, 60, torch.float32, scale=scale, out_dtype=torch.bfloat16, gen=gen)


@pytest.mark.parametrize("N", [1, 31, 1024, 5000, 20001])
def test_one_token_everywhere_and_none(N):
    check(torch.full((N,), 6).cuda(), 9, 40, torch.float32)
    _, dw = check(torch.full((N,), -1).cuda(), 9, 40, torch.float32)
    assert bool((dw == 0).all())


def test_rows_in_order_reversed_and_shuffled():
    V = 3000
    gen = torch.Generator().manual_seed(2)
    for t in (torch.arange(V), torch.arange(V).flip(0), torch.randperm(V, generator=gen), torch.arange(2 * V) // 2,
              torch.arange(V).repeat(3), torch.cat([torch.full((500,), V - 1), torch.zeros(500, dtype=torch.long)])):
        check(t.cuda(), V, 20, torch.float32, gen=gen)


def test_int32_strided_tokens_and_weight():
    gen = torch.Generator().manual_seed(4)
    t = torch.randint(0, 50, (8, 12), generator=gen, dtype=torch.int32).cuda()[:, ::2]
    big = torch.randn(50, 100, generator=gen).cuda()
    for w in (big[:, :64], big[:, 1:66], big.t()[:, :50]):
        y = embedding(t % w.shape[0], w)
        assert torch.equal(y, w[(t % w.shape[0]).long()])
    check(t.long(), 50, 30, torch.float32)
    assert embedding(t[:0], big).shape == (0, 6, 100)
    w = big.clone().requires_grad_()
    assert bool((torch.autograd.grad(embedding(t[:0], w).sum(), w)[0] == 0).all())


def test_tokens_out_of_range():
    w = torch.randn(10, 12).cuda().requires_grad_()
    t = torch.tensor([3, 10, -2, -1, 3, 2 ** 40]).cuda()
    y = embedding(t, w)
    assert y.isnan().all(1).tolist() == [False, True, True, False, False, True] and bool((y[3] == 0).all())
    dw, = torch.autograd.grad(y, w, torch.ones_like(y))
    want = torch.zeros(10, 12).cuda()
    want[3] = 2
    assert torch.equal(dw, want)


def test_gradient_is_the_slope():
    """The gradient of sum(c * y) against differences of the definition in float64 (linear: exact up to
    rounding)."""
    gen = torch.Generator().manual_seed(5)
    t = zipf(500, 40, gen)
    w = torch.randn(40, 16, generator=gen).cuda().requires_grad_()
    c = torch.randn(500, 16, generator=gen).cuda()
    dw, = torch.autograd.grad(embedding(t, w, scale=2.5), w, c)
    way = torch.randn(40, 16, generator=gen, dtype=torch.float64).cuda()
    f = lambda z: (c.double() * torch.where((t >= 0)[:, None], z[t.clamp(min=0)], 0.0) * 2.5).sum()  # noqa: E731
    slope = f(w.detach().double() + way) - f(w.detach().double())
    got = (dw.double() * way).sum()
    assert abs(float(got - slope)) <= 502 * U * 2.5 * float((c.double().abs().sum() * way.abs().max())) + 1e-9


def test_the_same_bits_in_every_run_and_stream():
    gen = torch.Generator().manual_seed(6)
    t = zipf(20000, 32000, gen)
    w = torch.randn(32000, 64, generator=gen).cuda().requires_grad_()
    dy = torch.randn(20000, 64, generator=gen).cuda()
    once = lambda: torch.autograd.grad(embedding(t, w), w, dy)[0]  # noqa: E731
    want = once().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = [once() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want) for o in other)


def test_captured_forward_and_backward():
    """A training step captured while no eager graph of the same leaf lives; two graphs share nothing."""
    gen = torch.Generator().manual_seed(7)
    done = []
    for V, N in ((500, 900), (32000, 64)):
        w = torch.randn(V, 32, generator=gen).cuda().requires_grad_()
        t, dy = zipf(N, V, gen), torch.randn(N, 32, generator=gen).cuda()
        torch.autograd.grad(embedding(t, w), w, dy)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = embedding(t, w)
            dw, = torch.autograd.grad(y, w, dy)
        done.append((g, w, t, dy, y, dw))
    for i in range(3):
        for g, w, t, dy, y, dw in done:
            t.copy_(t.roll(i + 1)), dy.normal_()
            g.replay()
        for g, w, t, dy, y, dw in done:
            y2 = embedding(t, w)
            assert torch.equal(y, y2) and torch.equal(dw, torch.autograd.grad(y2, w, dy)[0])


def test_torch_compile_fullgraph():
    w = torch.randn(40, 16, device="cuda").requires_grad_()
    t = torch.randint(-1, 40, (6, 7), device="cuda")
    f = lambda w: (embedding(t, w, scale=3.0) ** 2).sum()  # noqa: E731
    want, = torch.autograd.grad(f(w), w)
    got, = torch.autograd.grad(torch.compile(f, fullgraph=True, backend="aot_eager")(w), w)
    assert torch.equal(got, want)


def test_refusals():
    w, t = torch.randn(5, 4).cuda(), torch.zeros(3, dtype=torch.long).cuda()
    for a, kw in (((t, w[0]), {}), ((t.cpu(), w), {}), ((t, w[:0]), {}), ((t, w.bfloat16()), dict(out_dtype=torch.float32))):
        with pytest.raises(ValueError):
            embedding(*a, **kw)
    for a in ((t.float(), w), (t, w.half()), (t.bool(), w)):
        with pytest.raises(TypeError):
            embedding(*a)


def test_second_derivatives_are_refused():
    w = torch.randn(5, 4, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(embedding(torch.zeros(3, dtype=torch.long, device="cuda"), w).sum(), w, create_graph=True)
