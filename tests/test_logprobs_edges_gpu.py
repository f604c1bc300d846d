"""The log-probability entries at their edges: digits of the gradients, alternatives of rows in order,
many small calls one after another, rows with NaN, tokens out of range. Oracles in float64."""
import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.logprobs import lm_head_logprobs, token_logprobs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def on_grid(N, V, D, seed, dtype):
    """Operands in whole steps that bf16 holds, so that each logit is exact in fp32, whatever the order
    of its sum: products are multiples of 2^-9 below 2^2, a thousand of them below 2^12."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    h = (torch.randn(N, D, device="cuda", generator=gen) * 4).round().clamp(-15, 15) / 8
    w = (torch.randn(V, D, device="cuda", generator=gen) * 3).round().clamp(-15, 15) / 64
    t = torch.randint(-1, V, (N,), device="cuda", generator=gen)
    return h.to(dtype), w.to(dtype), t, gen


@pytest.mark.parametrize("N,V,D", [(1, 300, 64), (256, 1000, 64), (257, 1000, 64), (700, 2050, 96), (2049, 515, 40)])
def test_head_backward_holds_the_logits_gradient_in_16_digits(N, V, D):
    """bf16 operands held in fp32 tensors: dh and dw come in fp32, and with the logits exact their only
    errors are those of the statistics, of the logits' gradient in two bf16 parts (each value off by 2^-17)
    and of the fp32 sums. One bf16 part (2^-8 a value) is a hundred times past the bound."""
    h, w, t, gen = on_grid(N, V, D, N, torch.float32)
    h, w = h.requires_grad_(), w.requires_grad_()
    a = torch.randn(N, device="cuda", generator=gen)
    b = torch.randn(N, device="cuda", generator=gen)
    r = lm_head_logprobs(h, w, t, precision="bf16")
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [h, w], [a, b])
    assert dh.dtype == torch.float32 and dw.dtype == torch.float32
    h64, w64, a, b = h.detach().double(), w.detach().double(), a.double(), b.double()
    logp = torch.log_softmax(h64 @ w64.t(), -1)
    p = logp.exp()
    ent = -(p * logp).sum(-1)
    a = torch.where(t >= 0, a, 0.0)
    d = -p * (a[:, None] + b[:, None] * (logp + ent[:, None]))
    size = p * (a.abs()[:, None] + b.abs()[:, None] * (logp.abs() + ent[:, None]))
    d = d.scatter_add(1, t.clamp(min=0)[:, None], a[:, None])
    # the statistics: sums of V powers, each of them off by 2^-22 and by its argument's rounding (up to 40 log2 e)
    rs = (V / 32 + 32) * U + 2.0 ** -22 + 80 * U
    d_err = size * 8 * rs + (d.abs() + size) * 2.0 ** -17
    for got, want, err, mag, n in ((dh, d @ w64, d_err @ w64.abs(), d.abs() @ w64.abs(), V),
                                   (dw, d.t() @ h64, d_err.t() @ h64.abs(), d.abs().t() @ h64.abs(), N)):
        # sums of n products of two parts, in steps of 16 that may each cut off 2u
        tol = err + (n / 16 + 16) * 4 * U * mag + 1e-30
        assert bool(((got.double() - want).abs() <= tol).all())
    assert L.device_error() == 0


@pytest.mark.parametrize("k", [1, 2, 8, 9, 20])
def test_alternatives_of_rows_whose_every_chunk_enters_the_list(k):
    """Rows ascending from chunk to chunk of 32 logits: each chunk takes the place of the one that leaves,
    with one alternative always the same place. Logits are exact (whole 1/1024s below 2^10): the
    alternatives are the last ids, in the reverse order in descending rows."""
    N, V, D = 9000, 32000, 64
    v = torch.arange(V, device="cuda")
    w = torch.zeros(V, D, device="cuda")
    w[:, 0], w[:, 1], w[:, 2] = (v // 1024) * 4, (v // 32) % 32 / 8, (v % 32) / 1024
    h = torch.zeros(N, D, device="cuda")
    h[:, :3] = 1
    h[1::3, :3] = -1
    h[2::3, :3] = 0.5
    t = torch.arange(N, device="cuda") % V
    w, h = w.bfloat16(), h.bfloat16()
    x = h[:3, :3].double() @ w[:, :3].double().t()
    logp = torch.log_softmax(x, -1)
    for _ in range(3):
        r = lm_head_logprobs(h, w, t, top_k=k)
        for i in range(3):
            ids = torch.arange(k, device="cuda") if i == 1 else V - 1 - torch.arange(k, device="cuda")
            assert bool((r.top_ids[i::3] == ids).all())
            want = logp[i, ids]
            # log s of 32000 powers: each off by 2^-22 and by its argument's rounding (up to 160 log2 e)
            tol = (V / 32 + 32) * U + 2.0 ** -22 + 320 * U + 4 * U * 160
            assert bool(((r.top_logprobs[i::3].double() - want).abs() <= tol).all())
    assert L.device_error() == 0


@pytest.mark.parametrize("N,V", [(1, 32000), (3, 16384), (37, 33001), (80, 20000)])
def test_rows_split_over_a_cluster_again_and_again(N, V):
    """Few rows: a row's CTAs store their results into the first one's shared memory. Many calls one after
    another, on two streams beside a product that keeps the GPU full: the same bits each time."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(N, V, device="cuda", generator=gen) * 3
    t = torch.randint(0, V, (N,), device="cuda", generator=gen)
    big = torch.randn(4096, 4096, device="cuda", generator=gen).bfloat16()
    want = [o.clone() for o in token_logprobs(x, t, top_k=9)]
    logp = torch.log_softmax(x.double(), -1)
    assert torch.equal(want[2], torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :9])
    rs = (V / 32 + 32) * U + 2.0 ** -22 + 80 * U
    assert bool(((want[0] - logp.gather(1, t[:, None])[:, 0]).abs() <= rs + 4 * U * 40).all())
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(60):
        with torch.cuda.stream(streams[i % 2]):
            if i % 10 == 0:
                big @ big
            got.append(token_logprobs(x, t, top_k=9))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    assert L.device_error() == 0


@pytest.mark.parametrize("N,V,k,bad", [(3, 40, 32, 20), (3, 40, 32, 39), (300, 500, 20, 7), (9000, 8000, 8, 300), (9000, 8000, 1, 2)])
def test_alternatives_of_rows_with_some_nan(N, V, k, bad):
    """Weight rows of NaN: every row of logits holds some. NaN results, and k different tokens as
    alternatives."""
    h, w, t, gen = on_grid(N, V, 64, N, torch.bfloat16)
    w[torch.randperm(V, device="cuda", generator=gen)[:bad]] = float("nan")
    r = lm_head_logprobs(h, w, t, top_k=k)
    assert bool(r.logprobs[t >= 0].isnan().all()) and bool((r.logprobs[t < 0] == 0).all())
    assert bool(r.entropy.isnan().all()) and bool(r.top_logprobs.isnan().all())
    assert bool((r.top_ids >= 0).all()) and bool((r.top_ids < V).all())
    ids = r.top_ids.sort(-1).values
    assert bool((ids[:, 1:] != ids[:, :-1]).all())
    assert L.device_error() == 0


@pytest.mark.parametrize("N,V,k", [(5, 300, 4), (9000, 8000, 8)])
def test_head_rows_past_the_range(N, V, k):
    """Products below -1e30 throughout, or beyond 2.3e38: NaN, not an infinite or a finite answer; other rows
    as they are."""
    h, w, t, _ = on_grid(N, V, 64, 1, torch.bfloat16)
    t = t.clamp(min=0)
    h[:, 0], w[:, 0] = 0, 2.0 ** 60
    want = lm_head_logprobs(h, w, t, top_k=k)
    h[1, 0], h[3, 0] = -(2.0 ** 50), 2.0 ** 67 * 1.75  # -1.3e33 and 3e38
    r = lm_head_logprobs(h, w, t, top_k=k)
    for i in (1, 3):
        assert bool(r.logprobs[i].isnan()) and bool(r.entropy[i].isnan()) and bool(r.top_logprobs[i].isnan().all())
        ids = r.top_ids[i].sort().values
        assert bool((ids[1:] != ids[:-1]).all()) and 0 <= int(ids[0]) and int(ids[-1]) < V
    keep = (torch.arange(N, device="cuda") != 1) & (torch.arange(N, device="cuda") != 3)
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(r, want))
    hh, ww = h.requires_grad_(), w.requires_grad_()
    r = lm_head_logprobs(hh, ww, t)
    dh, = torch.autograd.grad(r.logprobs.sum(), hh)
    assert bool(dh[1].isnan().all()) and bool(dh[3].isnan().all()) and bool(dh[keep].isfinite().all())


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_the_entropys_gradient_does_not_see_the_token(precision):
    """A token out of range makes its logprob NaN, and the gradients through it; the entropy and its
    gradient have nothing of it."""
    dtype = torch.bfloat16 if precision == "bf16" else torch.float32
    h, w, t, _ = on_grid(7, 300, 64, 2, dtype)
    h, w = h.requires_grad_(), w.requires_grad_()
    x = (torch.randn(7, 300, device="cuda") * 2).to(dtype).requires_grad_()
    bad = t.clone()
    bad[1], bad[4] = 300, -5
    for call, leaves in ((lambda t: lm_head_logprobs(h, w, t, precision=precision), [h, w]), (lambda t: token_logprobs(x, t), [x])):
        want = torch.autograd.grad(call(t).entropy.sum(), leaves)
        got = torch.autograd.grad(call(bad).entropy.sum(), leaves)
        assert all(torch.equal(a, b) and bool(a.isfinite().all()) for a, b in zip(got, want))
        through = torch.autograd.grad(call(bad).logprobs.sum(), leaves)
        assert all(bool(g.isnan().any()) for g in through)
