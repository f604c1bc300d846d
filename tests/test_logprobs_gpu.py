"""Log probabilities of given tokens (logprobs.token_logprobs, logprobs.lm_head_logprobs) against the
definition in float64: values, entropies, alternatives and gradients, over types, odd sizes, strides,
masks and ties.

Tolerances, from the arithmetic (u = 2^-24, fp32's half step; bf16's is 2^-8):
* s = sum exp(x - m) is a sum of V positive terms in at most V / 32 + 32 steps one after another, each
  off by u; an exp is off by 2^-22 (the hardware's exp2) plus the rounding of its argument,
  |x - m| log2(e) u: rel_s below. logp = (x_t - m) - log s adds two roundings.
* H = log s - u1 / s with u1 = sum exp(x - m)(x - m): the same relative error in u1 and s.
* a logit of a product over D is off by the accumulation, at most (D / 16 + 16) steps of 2u (a tensor
  core may truncate) of sum_d |h_d w_d|: its logp by twice that.
"""
import math

import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.logprobs import lm_head_logprobs, token_logprobs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}


def plain(x, tokens, k=0):
    """float64: (logprobs, entropy, top ids, log softmax)."""
    x = x.double()
    logp = x - x.amax(-1, keepdim=True)  # first: a common -3e38 leaves no digits for log s otherwise
    logp = logp - logp.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    ent = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(-1)
    V = x.shape[-1]
    ok = (tokens >= 0) & (tokens < V)
    lp = logp.gather(-1, torch.where(ok, tokens, 0)[..., None])[..., 0]
    lp = torch.where(ok, lp, torch.where(tokens == -1, 0.0, math.nan).double())
    # stable sorts: equal logits in id order, then NaN above all, +inf too
    ids = torch.sort(torch.where(x.isnan(), math.inf, x) + 0.0, dim=-1, descending=True, stable=True).indices
    nan = torch.sort(x.isnan().gather(-1, ids).int(), dim=-1, descending=True, stable=True).indices
    ids = ids.gather(-1, nan)[..., :k]
    return lp, ent, ids, logp


def plain_dx(logp, ent, tokens, a, b):
    p = logp.exp()
    a = torch.where(tokens >= 0, a.double(), 0.0)
    d = -p * (a[:, None] + b.double()[:, None] * (logp + ent[:, None]))
    return d.scatter_add(1, tokens.clamp(min=0)[:, None], a[:, None])


def tol_s(V, spread):
    return (V / 32 + 32) * U + 2.0 ** -22 + 2 * spread * U


def assert_close(got, want, tol):
    want = want.to(got.device)
    assert torch.equal(got.isnan(), want.isnan())
    fin = want.isfinite()
    assert torch.equal(got.double()[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    err = (got.double() - want).abs()[fin]
    tol = tol.expand_as(want)[fin] if torch.is_tensor(tol) else tol
    assert bool((err <= tol).all()), float((err / tol).max() if torch.is_tensor(tol) else err.max())


def check_stats(out, x, tokens, k, extra=0.0):
    lp, ent, ids, logp = plain(x, tokens, k)
    spread = float((x.double().amax(-1) - torch.where(x.isfinite(), x.double(), math.inf).amin(-1)).nan_to_num(0, 0, 0).max())
    rs = tol_s(x.shape[-1], min(spread, 40.0)) + 2 * extra
    assert_close(out.logprobs, lp, rs + 4 * U * lp.abs().nan_to_num(0, 0, 0) + 2 * U * math.log(x.shape[-1]))
    big = ent.nan_to_num(0).abs() + math.log(x.shape[-1])
    assert_close(out.entropy, ent, 3 * rs * (1 + big) + 4 * U * big)
    if k:
        if not extra:
            assert torch.equal(out.top_ids, ids)
        got = logp.gather(-1, out.top_ids)
        assert_close(out.top_logprobs, got, rs + 4 * U * got.abs().nan_to_num(0, 0, 0) + 2 * U * math.log(x.shape[-1]))
    return lp, ent, logp, rs


def given(N, V, gen):
    t = torch.randint(0, V, (N,), generator=gen)
    t[::5] = -1
    return t.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (3, 2, 2), (2, 7, 0), (1, 32000, 5), (5, 513, 32), (64, 4099, 20),
                                   (300, 97, 8), (7, 70001, 31), (9, 32000, 1)])
def test_rows(dtype, N, V, k):
    gen = torch.Generator().manual_seed(N * V + k)
    x = (torch.randn(N, V, generator=gen) * 3).to(dtype).cuda()
    t = given(N, V, gen)
    check_stats(token_logprobs(x, t, top_k=k), x, t, k)
    assert L.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("stride", [1000, 1001, 1003, 1008])
def test_row_strides_and_offsets(dtype, stride):
    gen = torch.Generator().manual_seed(stride)
    buf = torch.randn(13 * stride + 16, generator=gen).to(dtype).cuda()
    for off in (0, 1, 3):
        x = buf[off:off + 13 * stride].view(13, stride)[:, :997]
        t = given(13, 997, gen)
        check_stats(token_logprobs(x, t, top_k=7), x, t, 7)
    xt = buf[:990 * 13].view(990, 13).t()  # the vocabulary is the outer dimension
    t = given(13, 990, gen)
    check_stats(token_logprobs(xt, t, top_k=7), xt, t, 7)


def test_leading_shapes_and_int32():
    x = torch.randn(2, 3, 50, device="cuda")
    t = torch.randint(0, 50, (2, 3), device="cuda", dtype=torch.int32)
    r = token_logprobs(x, t, top_k=4)
    assert r.logprobs.shape == (2, 3) and r.entropy.shape == (2, 3) and r.top_ids.shape == (2, 3, 4)
    check_stats(type(r)(r.logprobs.view(6), r.entropy.view(6), r.top_ids.view(6, 4), r.top_logprobs.view(6, 4)),
                x.view(6, 50), t.view(6).long(), 4)
    empty = token_logprobs(x[:0], t[:0], top_k=4)
    assert empty.logprobs.shape == (0, 3) and empty.top_ids.shape == (0, 3, 4)


@pytest.mark.parametrize("V", [64, 1000, 32000])
def test_masked_rows(V):
    """Rows of which one, three, or no tokens are left; the type's lowest value as the mask; all equal;
    every second one equal."""
    inf, low = float("inf"), torch.finfo(torch.float32).min
    x = torch.full((8, V), -inf)
    x[0, V - 1] = 2.0
    x[1, [3, 17, V // 2]] = torch.tensor([1.0, -1.0, 1.0])
    x[3] = low
    x[4] = low
    x[4, V // 3] = 5.0
    x[5] = 0.25
    x[6, ::2] = 1e30
    x[7] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0)
    x, t = x.cuda(), torch.tensor([V - 1, 0, 1, 2, V // 3, 4, 0, 9]).cuda()
    r = token_logprobs(x, t, top_k=20)
    check_stats(r, x, t, 20)
    assert r.logprobs[0] == 0 and r.entropy[0] == 0 and r.logprobs[1] == -inf and bool(r.logprobs[2].isnan())
    assert r.top_ids[2].tolist() == list(range(20)) and r.top_ids[7].tolist() == list(range(20))


def test_nan_inf_and_tokens_out_of_range():
    V = 3000
    x = torch.randn(6, V)
    x[1, 100] = float("nan")
    x[2, 7] = float("inf")
    x[3, :] = float("nan")
    x, t = x.cuda(), torch.tensor([5, 5, 5, 5, V, -7]).cuda()
    r = token_logprobs(x, t, top_k=3)
    want = plain(x, t)[0]
    assert torch.equal(r.logprobs.isnan(), want.isnan()) and torch.equal(r.logprobs.isnan().cpu(), torch.tensor([0, 1, 1, 1, 1, 1]).bool())
    assert torch.equal(r.entropy.isnan().cpu(), torch.tensor([0, 1, 1, 1, 0, 0]).bool())
    assert r.top_ids[1, 0] == 100 and r.top_ids[2, 0] == 7 and r.top_ids[3].tolist() == [0, 1, 2]


def test_many_equal_best():
    """More equal logits than any list of candidates holds: the lowest ids win."""
    V = 20000
    x = torch.randn(3, V).clamp(max=-0.5)
    x[0, 5000:7000] = 3.0
    x[1, ::3] = 1.0
    x[2, V - 40:] = 2.0
    x[2, 11] = 4.0
    x, t = x.cuda(), torch.zeros(3, dtype=torch.long).cuda()
    for k in (1, 17, 32):
        check_stats(token_logprobs(x, t, top_k=k), x, t, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(1, 1), (4, 3), (33, 1001), (5, 32000)])
def test_rows_backward(dtype, N, V):
    gen = torch.Generator().manual_seed(N + V)
    x = (torch.randn(N, V, generator=gen) * 2).to(dtype).cuda().requires_grad_()
    t = given(N, V, gen)
    a, b = torch.randn(N, generator=gen).cuda(), torch.randn(N, generator=gen).cuda()
    r = token_logprobs(x, t)
    lp, ent, _, logp = plain(x.detach(), t)
    rs = tol_s(V, 20.0)
    for ga, gb in ((a, b), (a, None), (None, b)):
        outs = [o for o, g in ((r.logprobs, ga), (r.entropy, gb)) if g is not None]
        d, = torch.autograd.grad(outs, x, [g for g in (ga, gb) if g is not None], retain_graph=True)
        za, zb = (g if g is not None else torch.zeros(N).cuda() for g in (ga, gb))
        want = plain_dx(logp, ent, t, za, zb)
        size = logp.exp() * (za.abs()[:, None] + zb.abs()[:, None] * (logp.abs() + ent[:, None]))
        # the statistics are sums of 2^(x log2 e - fl(m log2 e)): the exponent's two roundings, of a number up
        # to 2 |m|, leave log p and H an absolute error of 4 u (1 + |m|), also where both are zero (V = 1)
        base = 4 * U * (1 + x.detach().double().abs().amax(-1, keepdim=True))
        size = size + logp.exp() * zb.abs()[:, None] * base
        assert d.dtype == dtype
        assert_close(d, want, size * (4 * rs + 8 * U * (1 + logp.abs())) + logp.exp() * zb.abs()[:, None] * base +
                     2 * HALF[dtype] * want.abs() + 1e-37)
    assert L.device_error() == 0


def test_rows_backward_is_the_slope():
    """Against differences of the definition in float64, in a direction of its own for each row."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, 700, generator=gen).cuda().requires_grad_()
    t = given(6, 700, gen)
    r = token_logprobs(x, t)
    d, = torch.autograd.grad(r.logprobs.sum() + 0.7 * r.entropy.sum(), x)
    way = torch.randn(6, 700, generator=gen, dtype=torch.float64).cuda()
    f = lambda z: sum(w * v for w, v in zip((1.0, 0.7), plain(z, t)[:2]))  # noqa: E731
    e = 1e-5
    slope = (f(x.detach().double() + e * way) - f(x.detach().double() - e * way)) / (2 * e)
    # differences: O(e^2) and 1e-16 / e; the sum over 700 products of fp32 gradients: their relative error
    size = (d.double() * way).abs().sum(-1)
    assert bool(((d.double() * way).sum(-1) - slope).abs().le(1e-8 + 1e-5 * size).all())


def test_masked_backward():
    x = torch.randn(4, 50)
    x[0, 10:] = -float("inf")
    x[1, :] = -float("inf")
    x = x.cuda().requires_grad_()
    t = torch.tensor([3, 3, 99, 5]).cuda()
    r = token_logprobs(x, t)
    d, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), x)
    assert bool((d[0, 10:] == 0).all()) and bool(d[0].isfinite().all()) and bool(d[3].isfinite().all())
    assert bool(d[1].isnan().all()) and bool(d[2].isnan().all())


def test_rows_at_the_ends_of_the_range():
    """Rows that hold nothing but the type's lowest value, or logits near its largest: values and
    gradients as of any other row."""
    big = 3e38
    x = torch.full((5, 300), torch.finfo(torch.float32).min)
    x[1, 7], x[1, 8] = big, big
    x[2] = torch.linspace(-big, big, 300)  # (its step overflows: a row with NaN and +inf)
    x[3] = 1e35 + torch.arange(300) * 0.0
    x[4] = torch.linspace(-1, 1, 300) * big
    x = x.cuda().requires_grad_()
    t = torch.tensor([5, 7, 299, 0, 299]).cuda()
    r = token_logprobs(x, t, top_k=2)
    lp, ent, logp, rs = check_stats(r, x.detach(), t, 2)
    a, b = torch.ones(5).cuda(), torch.full((5,), 0.5).cuda()
    d, = torch.autograd.grad([r.logprobs, r.entropy], x, [a, b])
    assert_close(d, plain_dx(logp, ent, t, a, b), 20 * rs + 1e-37)


# ---- from hidden states -------------------------------------------------------------------------------

def head_inputs(N, V, D, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    h = torch.randn(N, D, generator=gen).to(dtype).cuda()
    w = (torch.randn(V, D, generator=gen) * 1.5 / D ** 0.5).to(dtype).cuda()
    return h, w, given(N, V, gen), gen


def head_extra(h, w, D):
    big = max(float((h[i:i + 256].double().abs() @ w.double().abs().t()).max()) for i in range(0, h.shape[0], 256))
    return (D / 16 + 16) * 2 * U * big


HEAD = [(1, 1, 1, 1), (1, 32000, 768, 5), (3, 17, 33, 9), (130, 300, 40, 20), (257, 1000, 288, 3), (300, 513, 100, 0),
        (700, 2100, 64, 32), (2, 40000, 96, 8)]


@pytest.mark.parametrize("precision,dtype", [("bf16", torch.bfloat16), ("fp32", torch.float32)])
@pytest.mark.parametrize("N,V,D,k", HEAD)
def test_head(precision, dtype, N, V, D, k):
    h, w, t, _ = head_inputs(N, V, D, dtype, N + V)
    r = lm_head_logprobs(h, w, t, top_k=k, precision=precision)
    x = h.double() @ w.double().t()
    extra = head_extra(h, w, D)
    check_stats(r, x, t, k, extra=extra)
    if k:  # any two alternatives in another order are nearer than the logits' error
        best = x.gather(1, r.top_ids)
        assert bool((best[:, :-1] - best[:, 1:] >= -2 * extra).all())
        assert bool((x.sort(-1, descending=True).values[:, :k] - best).abs().le(2 * extra).all())
        assert all(len(set(row)) == k for row in r.top_ids.tolist())
    assert L.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_head_alternatives_on_a_grid(dtype):
    """Operands in whole steps, so that each logit is exact whatever the order of its sum: the
    alternatives are then the definition's, equal logits in the order of their ids."""
    gen = torch.Generator().manual_seed(0)
    for N, V, D, k in ((65, 5000, 96, 20), (600, 1500, 64, 32), (3, 32000, 200, 5)):
        h = (torch.randn(N, D, generator=gen) * 4).round().clamp(-15, 15).cuda() / 8
        w = (torch.randn(V, D, generator=gen) * 3).round().clamp(-15, 15).cuda() / 64
        t = given(N, V, gen)
        r = lm_head_logprobs(h.to(dtype), w.to(dtype), t, top_k=k, precision="bf16" if dtype == torch.bfloat16 else "fp32")
        x = h.double() @ w.double().t()
        check_stats(r, x, t, k)


@pytest.mark.parametrize("precision,dtype", [("bf16", torch.bfloat16), ("fp32", torch.float32)])
@pytest.mark.parametrize("N,V,D", [(1, 5, 8), (37, 300, 40), (300, 1000, 288), (513, 257, 129), (16, 9000, 64)])
def test_head_backward(precision, dtype, N, V, D):
    h, w, t, gen = head_inputs(N, V, D, dtype, N * V)
    h, w = h.requires_grad_(), w.requires_grad_()
    a, b = torch.randn(N, generator=gen).cuda(), torch.randn(N, generator=gen).cuda()
    r = lm_head_logprobs(h, w, t, precision=precision)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [h, w], [a, b], retain_graph=True)
    h64, w64 = h.detach().double(), w.detach().double()
    lp, ent, _, logp = plain(h64 @ w64.t(), t)
    d = plain_dx(logp, ent, t, a, b)
    # dlogits: their own error, and their rounding to the operand type; then two sums of products
    rs = tol_s(V, 20.0) + 2 * head_extra(h64, w64, D)
    size = logp.exp() * (a.abs().double()[:, None] + b.abs().double()[:, None] * (logp.abs() + ent[:, None]))
    d_err = size * 8 * rs + (d.abs() + size) * (HALF[dtype] + 8 * U)
    assert dh.dtype == dtype and dw.dtype == dtype
    sums = lambda n: (n / 16 + 16) * 2 * U  # noqa: E731
    for got, want, err, mag, n in ((dh, d @ w64, d_err @ w64.abs(), d.abs() @ w64.abs(), V),
                                   (dw, d.t() @ h64, d_err.t() @ h64.abs(), d.abs().t() @ h64.abs(), N)):
        assert_close(got, want, err + sums(n) * mag + 2 * HALF[dtype] * want.abs() + 1e-30)
    only_h, = torch.autograd.grad(r.logprobs, h, a, retain_graph=True)
    only_w, = torch.autograd.grad(r.entropy, w, b)
    assert only_h.shape == h.shape and only_w.shape == w.shape
    assert L.device_error() == 0


@pytest.mark.parametrize("N,V,D", [(1, 700, 64), (7, 9000, 288), (256, 3000, 96)])
def test_head_backward_of_few_rows_rounds_once(N, V, D):
    """bf16 operands, up to 256 rows: the logits' gradient goes into the products in two bf16 parts (16
    digits), so that dh and dW are off by their own rounding alone: each value by half a step, and by the
    fp32 sums and 2^-17 of the terms' magnitudes before it."""
    h, w, t, gen = head_inputs(N, V, D, torch.bfloat16, N)
    h, w = h.requires_grad_(), w.requires_grad_()
    a, b = torch.randn(N, generator=gen).cuda(), torch.randn(N, generator=gen).cuda()
    r = lm_head_logprobs(h, w, t)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [h, w], [a, b])
    h64, w64 = h.detach().double(), w.detach().double()
    lp, ent, _, logp = plain(h64 @ w64.t(), t)
    d = plain_dx(logp, ent, t, a, b)
    rs = tol_s(V, 20.0) + 2 * head_extra(h64, w64, D)
    size = logp.exp() * (a.abs().double()[:, None] + b.abs().double()[:, None] * (logp.abs() + ent[:, None]))
    d_err = size * 8 * rs + (d.abs() + size) * 2.0 ** -17
    for got, want, err, mag, n in ((dh, d @ w64, d_err @ w64.abs(), d.abs() @ w64.abs(), V),
                                   (dw, d.t() @ h64, d_err.t() @ h64.abs(), d.abs().t() @ h64.abs(), N)):
        assert_close(got, want, err + (n / 16 + 16) * 4 * U * mag + HALF[torch.bfloat16] * want.abs() + 1e-30)


def test_head_mixed_types_strides_and_empty():
    h = torch.randn(6, 4, 70, device="cuda")[..., :64].requires_grad_()  # rows of stride 70
    w = torch.randn(200, 64, device="cuda").bfloat16().requires_grad_()
    t = torch.randint(0, 200, (6, 4), device="cuda")
    r = lm_head_logprobs(h, w, t, top_k=2)
    x = h.detach().reshape(24, 64).bfloat16().double() @ w.detach().double().t()
    flat = type(r)(r.logprobs.reshape(24), r.entropy.reshape(24), r.top_ids.reshape(24, 2), r.top_logprobs.reshape(24, 2))
    check_stats(flat, x, t.view(24), 2, extra=head_extra(h.detach().reshape(24, 64), w.detach(), 64))
    dh, dw = torch.autograd.grad(r.logprobs.sum(), [h, w])
    assert dh.dtype == torch.float32 and dh.shape == h.shape and dw.dtype == torch.bfloat16
    e = lm_head_logprobs(h[:0], w, t[:0], top_k=2)
    dw0, = torch.autograd.grad(e.logprobs.sum(), w)
    assert e.logprobs.shape == (0, 4) and bool((dw0 == 0).all())


def test_runs_repeat_bit_for_bit_and_on_other_streams():
    h, w, t, _ = head_inputs(700, 3000, 128, torch.bfloat16, 1)
    h, w = h.requires_grad_(), w.requires_grad_()

    def once():
        r = lm_head_logprobs(h, w, t, top_k=8)
        return [r.logprobs, r.entropy, r.top_ids, r.top_logprobs, *torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), [h, w])]

    want = [o.clone() for o in once()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = once()
    torch.cuda.current_stream().wait_stream(s)
    for got in (once(), other):
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_captured_graphs_replayed_in_turn():
    """Two graphs of different sizes, replayed alternately on one stream with new inputs in place."""
    cases = []
    for N, V, D in ((40, 900, 64), (3, 5000, 96)):
        h, w, t, _ = head_inputs(N, V, D, torch.bfloat16, N)
        x = torch.randn(N, V, device="cuda")
        lm_head_logprobs(h, w, t, top_k=4), token_logprobs(x, t, top_k=4)  # first-call set-up
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = lm_head_logprobs(h, w, t, top_k=4), token_logprobs(x, t, top_k=4)
        cases.append((g, h, w, t, x, out))
    for rnd in range(3):
        for g, h, w, t, x, out in cases:
            h.normal_(), x.normal_()
            g.replay()
        for g, h, w, t, x, out in cases:
            for got, want in zip(out, (lm_head_logprobs(h, w, t, top_k=4), token_logprobs(x, t, top_k=4))):
                assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_torch_compile_fullgraph():
    h, w, t, _ = head_inputs(20, 300, 32, torch.bfloat16, 5)
    h = h.requires_grad_()

    def f(h):
        r = lm_head_logprobs(h, w, t, top_k=2)
        return r.logprobs.sum() + 0.1 * r.entropy.sum() + token_logprobs(h, t % 32).logprobs.sum()

    want, = torch.autograd.grad(f(h), h)
    got, = torch.autograd.grad(torch.compile(f, fullgraph=True, backend="aot_eager")(h), h)
    assert torch.equal(got, want)


def test_refusals():
    h, w, t = torch.randn(4, 8).cuda(), torch.randn(9, 8).cuda(), torch.zeros(4, dtype=torch.long).cuda()
    x = torch.randn(4, 9).cuda()
    for bad in (dict(tokens=t[:3]), dict(tokens=t.cpu()), dict(top_k=10), dict(top_k=-1), dict(h=h[:, :7]),
                dict(precision="fp16"), dict(weight=w[0]), dict(weight=w.cpu()), dict(weight=w[:0])):
        with pytest.raises(ValueError):
            lm_head_logprobs(**{**dict(h=h, weight=w, tokens=t), **bad})
    for bad in (dict(tokens=t[:3]), dict(tokens=t.cpu()), dict(top_k=10), dict(logits=x[:, :0])):
        with pytest.raises(ValueError):
            token_logprobs(**{**dict(logits=x, tokens=t), **bad})
    with pytest.raises(ValueError):
        token_logprobs(torch.randn(2, 100).cuda(), t[:2], top_k=33)
    for bad in (t.float(), t.bool()):
        with pytest.raises(TypeError):
            token_logprobs(x, bad)


@pytest.mark.parametrize("N,V,k", [(9000, 8000, 8), (9000, 8000, 1), (9001, 30000, 20), (9000, 29999, 32), (2100, 33000, 9)])
def test_head_alternatives_of_many_rows(N, V, k):
    """The forms for many rows (lists kept by the epilogue, rows in several launches), on a grid (above):
    some rows all equal, some ascending (each chunk enters the list), some descending."""
    D = 64
    gen = torch.Generator(device="cuda").manual_seed(N + k)
    h = (torch.randn(N, D, device="cuda", generator=gen) * 4).round().clamp(-15, 15) / 8
    w = (torch.randn(V, D, device="cuda", generator=gen) * 3).round().clamp(-15, 15) / 64
    w[:, 0] = torch.arange(V, device="cuda") // 128 / 2 ** 8
    h[:, 0] = 0
    h[5:1000:100] = 0
    h[7:1000:100] = 0
    h[7:1000:100, 0] = 8
    h[9:1000:100] = 0
    h[9:1000:100, 0] = -8
    t = torch.randint(-1, V, (N,), device="cuda", generator=gen)
    h, w = h.bfloat16(), w.bfloat16()  # (257 / 256 and the like round: the definition takes them rounded)
    r = lm_head_logprobs(h, w, t, top_k=k)
    for a in range(0, N, 1024):
        rows = slice(a, a + 1024)
        x = h[rows].double() @ w.double().t()
        check_stats(type(r)(*(o[rows] for o in r)), x, t[rows], k)
    assert L.device_error() == 0


def test_head_rows_of_nan():
    """A row of hidden states that holds a NaN, in each form: NaN results, ids in range, other rows as they
    are."""
    for N, V, k in ((3, 500, 20), (600, 4000, 9), (9000, 8000, 8)):
        h = torch.randn(N, 64, device="cuda").bfloat16()
        w = torch.randn(V, 64, device="cuda").bfloat16()
        t = torch.randint(0, V, (N,), device="cuda")
        want = lm_head_logprobs(h, w, t, top_k=k)
        h[1, 5] = float("nan")
        r = lm_head_logprobs(h, w, t, top_k=k)
        assert bool(r.logprobs[1].isnan()) and bool(r.entropy[1].isnan()) and bool(r.top_logprobs[1].isnan().all())
        assert r.top_ids[1].tolist() == list(range(k))
        keep = torch.arange(N, device="cuda") != 1
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(r, want))


def test_two_calls_at_once():
    """The same kernels on two streams at the same time, each with its own inputs and workspaces."""
    cases = [head_inputs(N, V, D, torch.bfloat16, N)[:3] for N, V, D in ((900, 4000, 128), (40, 30000, 96))]
    xs = [torch.randn(N, V, device="cuda") for N, V in ((300, 9000), (2, 32000))]

    def one(h, w, t, x):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        r = lm_head_logprobs(h, w, t, top_k=7)
        g = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), [h, w])
        s = token_logprobs(x, torch.arange(x.shape[0], device="cuda"), top_k=7)
        return [*r, *g, *s]

    want = [[o.detach().clone() for o in one(*c, x)] for c, x in zip(cases, xs)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, c, x in zip(streams, cases, xs):
            with torch.cuda.stream(s):
                got.append(one(*c, x))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    assert L.device_error() == 0


def test_captured_training_step():
    """Forward and backward in one graph, captured while no eager graph of the same leaves lives, replayed
    with new inputs in place."""
    for N, V, D, dt in ((70, 900, 64, torch.bfloat16), (300, 700, 40, torch.float32)):
        h, w, t, _ = head_inputs(N, V, D, dt, N)
        h, w = h.requires_grad_(), w.requires_grad_()
        x = torch.randn(N, V, device="cuda").to(dt).requires_grad_()
        prec = "bf16" if dt == torch.bfloat16 else "fp32"

        def step():
            r, s = lm_head_logprobs(h, w, t, precision=prec), token_logprobs(x, t)
            return torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + s.logprobs.sum() + s.entropy.sum(), [h, w, x])

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for _ in range(2):
            with torch.no_grad():
                h.normal_(), x.normal_()
            g.replay()
            got = [o.clone() for o in out]
            assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_second_derivatives_are_refused():
    x = torch.randn(3, 40, device="cuda", requires_grad=True)
    w = torch.randn(50, 40, device="cuda", requires_grad=True)
    t = torch.zeros(3, dtype=torch.long, device="cuda")
    for out in (token_logprobs(x, t).logprobs, lm_head_logprobs(x, w, t).entropy):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(out.sum(), x, create_graph=True)
