"""The global gradient norm and clipping (clip.py) against the definition in float64. The norm is a sum
of squares in fp64, rounded to fp32: off by 2^-24, and its square root's rounding. A clipped value has
three roundings in fp32 (the norm, the factor, the product) and one to its type."""
import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.clip import clip_grad_norm_, clip_grads, grad_norm
from unifiedlm_c_b200.dp import GradBucket

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def norm64(grads):
    return float(torch.cat([g.reshape(-1).double() for g in grads]).norm())


def check(grads, max_norm, out=None):
    before = [g.clone() for g in grads]
    n = norm64(grads)
    got = clip_grads(grads, max_norm, out=out)
    assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - n) <= 4 * U * n
    f = min(1.0, max_norm / (n + 1e-6))
    for b, g, o in zip(before, grads, grads if out is None else out):
        want = b.double() * f
        assert bool(((o.double() - want).abs() <= want.abs() * (HALF[o.dtype] + 8 * U) + 1e-45).all())
        assert out is None or torch.equal(g, b)  # the gradients stay
        if f == 1.0 and o.dtype == b.dtype:
            assert torch.equal(o, b)
    assert L.device_error() == 0


def model_like(gen, dtypes, D=72, M=130, layers=3, V=611):
    shapes = ([(D,), (D, 1, 4), (M, D), (M,), (D, M), (), (D, D), (), (M,)] * layers) + [(D,), (V, D)]
    return [torch.randn(s, generator=gen).to(dtypes[i % len(dtypes)]).cuda() for i, s in enumerate(shapes)]


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("max_norm", [0.0, 1.0, 1e6, float("inf")])
def test_in_place(dtypes, max_norm):
    check(model_like(torch.Generator().manual_seed(1), dtypes), max_norm)


@pytest.mark.parametrize("src", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dst", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm", [1.0, 1e6])
def test_into_a_bucket(src, dst, max_norm):
    """Outputs packed one after another: their starts have every alignment."""
    grads = model_like(torch.Generator().manual_seed(2), [src])
    bucket = GradBucket([g.shape for g in grads], device="cuda", dtype=dst)
    check(grads, max_norm, out=bucket.views())
    again = GradBucket([g.shape for g in grads], device="cuda", dtype=dst)
    n = again.pack_clipped(grads, max_norm)
    assert torch.equal(again.flat, bucket.flat) and abs(float(n) - norm64(grads)) <= 4 * U * float(n)


@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [3] * 700, [8192], [8193, 1, 8191], [1 << 21, 7], [40_000_003]])
def test_sizes(sizes):
    gen = torch.Generator(device="cuda").manual_seed(len(sizes))
    check([torch.randn(n, device="cuda", generator=gen) for n in sizes], 1.0)
    check([torch.randn(n, device="cuda", generator=gen).bfloat16() for n in sizes], 1.0)


def test_odd_starts():
    buf = torch.randn(5000).cuda()
    b16 = torch.randn(5000).cuda().bfloat16()
    check([buf[1:1000], buf[1003:2001], b16[1:900], b16[905:4000]], 0.5)
    check([buf[1:1000], b16[3:900]], 0.5, out=[torch.empty(1000).cuda()[1:], torch.empty(898).cuda().bfloat16()[1:]])


def test_strided_gradients():
    a = torch.randn(40, 30).cuda()
    check([a.t(), torch.randn(8, 9, 10).cuda()[:, ::2], torch.randn(6).cuda().expand(3, 6)[0]], 1.0)
    out = torch.empty(30, 40).cuda()
    check([a.t()], 1.0, out=[out]), check([out], 1.0, out=[a.t()])


def test_large_and_small_values():
    """Squares past fp32's range, and below it."""
    check([torch.full((1000,), 3e30).cuda(), torch.ones(5).cuda()], 1.0)
    check([torch.full((1000,), 1e-30).cuda()], 1e-32)
    x = torch.zeros(100).cuda()
    assert float(clip_grads([x], 1.0)) == 0 and bool((x == 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_finite_as_torch(bad):
    for max_norm in (1.0, float("inf")):
        ps = [torch.nn.Parameter(torch.ones(50).cuda()) for _ in range(3)]
        qs = [torch.nn.Parameter(torch.ones(50).cuda()) for _ in range(3)]
        for p, q in zip(ps, qs):
            p.grad, q.grad = torch.ones(50).cuda(), torch.ones(50).cuda()
        ps[1].grad[7] = qs[1].grad[7] = bad
        got, want = clip_grad_norm_(ps, max_norm), torch.nn.utils.clip_grad_norm_(qs, max_norm)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        for p, q in zip(ps, qs):
            assert torch.equal(p.grad.isnan(), q.grad.isnan()) and torch.equal(p.grad.nan_to_num(), q.grad.nan_to_num())


def test_parameters_and_norm():
    lin = torch.nn.Linear(64, 32).cuda()
    assert float(clip_grad_norm_(lin.parameters(), 1.0)) == 0.0  # no gradients
    lin.weight.grad = torch.randn(32, 64).cuda()
    n = norm64([lin.weight.grad])
    v = lin.weight.grad._version
    assert abs(float(grad_norm([lin.weight.grad, None])) - n) <= 4 * U * n
    assert float(grad_norm([lin.weight.grad] * 2)) == pytest.approx(n * 2 ** 0.5, rel=1e-6)
    assert abs(float(clip_grad_norm_(lin.weight, 0.5)) - n) <= 4 * U * n
    assert norm64([lin.weight.grad]) <= 0.5 * (1 + 8 * U) and lin.weight.grad._version > v
    bucket = GradBucket([(32, 64)], device="cuda")
    bucket.pack([torch.randn(32, 64).cuda()])
    bucket.clip_norm_(0.25)
    assert abs(norm64([bucket.flat]) - 0.25) < 1e-6


def test_runs_repeat_and_replay():
    gen = torch.Generator().manual_seed(8)
    grads = model_like(gen, [torch.float32, torch.bfloat16])
    out = [torch.empty_like(g) for g in grads]
    norms = {float(clip_grads(grads, 1.0, out=out)) for _ in range(5)}
    assert len(norms) == 1
    want = [o.clone() for o in out]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n = clip_grads(grads, 1.0, out=out)
    for _ in range(2):
        [o.zero_() for o in out]
        g.replay()
        assert float(n) in norms and all(torch.equal(o, w) for o, w in zip(out, want))


def test_refusals():
    x, y = torch.ones(10).cuda(), torch.ones(10).cuda()
    for bad in (float("nan"), -1.0):
        with pytest.raises(ValueError):
            clip_grads([x], bad)
    for a, kw in ((([x, y], 1.0), dict(out=[x])), (([x], 1.0), dict(out=[y[:9]])), (([x], 1.0), dict(out=[y.cpu()])),
                  (([x, y.cpu()], 1.0), {})):
        with pytest.raises((ValueError, RuntimeError)):
            clip_grads(*a, **kw)
    for grads, out in (([x, x], None), ([x[:6], x[5:]], None), ([x, y], [y, x]), ([x[1:]], [x[:-1]]), ([x, y], [torch.empty(10).cuda()] * 2)):
        with pytest.raises(L.UlmError, match="overlap"):
            clip_grads(grads, 1.0, out=out)
    with pytest.raises(L.UlmError, match="type"):
        clip_grads([x.half()], 1.0)
    assert bool((x == 1).all()) and bool((y == 1).all())
