"""The operators at the two ends of UnifiedLM's training and serving loop, as cases to measure.

head    log probabilities of given tokens from the final hidden states and the output weight, with
        the entropy and the best alternatives (`logprobs.lm_head_logprobs`), and its gradients
logits  the same from logits that exist already, as after a decode step (`logprobs.token_logprobs`)
embed   token embedding lookup with a scale, and the weight's gradient (`embed.embedding`)
clip    the global gradient norm over many tensors, and clipping by it (`clip.clip_grads`)

`run` computes a case by elementary torch operations, or with `own` by the framework's entry points;
`exact` computes it in 64 bits.
"""
import functools
import math

import torch

own = False

# Widths, vocabulary and batch shapes are those of the 15M (dim 288, 6 layers, M 768), 42M (dim 512,
# M 1024) and 110M (dim 768, 12 layers, M 2048) UnifiedLM shapes with the 32000-token vocabulary.


def listed():
    return [
        # a server scores the one token that it has just emitted, with the five best alternatives
        dict(name="head_score_1", kind="head", N=1, V=32000, D=768, dtype="bf16", k=5, train=False),
        # a ragged prompt of an evaluation set on the 15M model, with the twenty best alternatives
        dict(name="head_score_333", kind="head", N=333, V=32000, D=288, dtype="bf16", k=20, train=False),
        # a whole batch of 16 x 1024 prompt tokens on the 110M model, as for distillation data
        dict(name="head_score_16384", kind="head", N=16384, V=32000, D=768, dtype="bf16", k=8, train=False),
        # a policy-gradient step with an entropy bonus: 8 x 1024 tokens of the 110M model
        dict(name="head_train_8192", kind="head", N=8192, V=32000, D=768, dtype="bf16", k=0, train=True),
        # the fp32 parity mode on the 15M width, a 4099-token vocabulary and an odd number of rows
        dict(name="head_train_fp32", kind="head", N=1001, V=4099, D=288, dtype="fp32", k=3, train=True),
        # one sequence's decode step: its logits, some of them masked by a grammar
        dict(name="logits_1", kind="logits", N=1, V=32000, dtype="fp32", k=5, train=False),
        # a decode step of 256 sequences
        dict(name="logits_256", kind="logits", N=256, V=32000, dtype="fp32", k=20, train=False),
        # training on bf16 logits of another head: 4 x 1024 tokens
        dict(name="logits_train_4096", kind="logits", N=4096, V=32000, dtype="bf16", k=0, train=True),
        # the 110M model's embedding over 16 x 1024 tokens, forward and gradient
        dict(name="embed_train_16384", kind="embed", N=16384, V=32000, D=768, dtype="fp32", scale=1.0, train=True),
        # bf16 weights, scaled by sqrt(dim), 97 sequences of 256 tokens
        dict(name="embed_train_bf16", kind="embed", N=24832, V=32000, D=512, dtype="bf16", scale=512.0 ** 0.5, train=True),
        # every gradient of the 110M model, clipped in place before the optimizer step
        dict(name="clip_110m", kind="clip", D=768, M=2048, L=12, V=32000, dtype="fp32", max_norm=1.0, inplace=True),
        # bf16 gradients of a small model, written clipped into an fp32 bucket
        dict(name="clip_small_bf16", kind="clip", D=288, M=712, L=2, V=4099, dtype="bf16", max_norm=1.0, inplace=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["head", "head", "logits", "embed", "clip"])
    V = rng.choice([32000, _log(rng, 300, 50000), _log(rng, 300, 50000)])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "head":
        train = rng.random() < 0.5
        D = rng.choice([288, 512, 768, _log(rng, 32, 1024)])
        # no more products than the largest listed case; the fp32 mode is for smaller work
        top = (4e11 if dtype == "bf16" else 4e10) / (V * D * (3 if train else 1))
        N = max(1, _log(rng, 1, max(2, min(16384, int(top)))))
        return dict(kind=kind, N=N, V=V, D=D, dtype=dtype, k=rng.choice([0, 1, 5, 8, 20, 31]), train=train)
    if kind == "logits":
        train = rng.random() < 0.4
        N = _log(rng, 1, max(2, min(8192, 130_000_000 // V)))
        return dict(kind=kind, N=N, V=V, dtype=dtype, k=0 if train else rng.choice([0, 1, 5, 20, 32]), train=train)
    if kind == "embed":
        D = rng.choice([288, 512, 768, _log(rng, 16, 1024)])
        N = _log(rng, 1, max(2, min(131072, 16384 * 768 // D)))
        return dict(kind=kind, N=N, V=V, D=D, dtype=dtype, scale=rng.choice([1.0, float(D) ** 0.5]), train=rng.random() < 0.7)
    return dict(kind=kind, D=_log(rng, 32, 768), M=_log(rng, 64, 2048), L=rng.randint(1, 12), V=V, dtype=dtype,
                max_norm=rng.choice([0.5, 1.0, 1000.0]), inplace=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


class _State:
    pass


def _on_grid(x, step, most):
    """Values in whole steps. The operands of the products are given as fixed-point numbers with so few
    digits that every sum of their products has an exact value in 32 bits, whatever the order of the
    additions: which token is the 20th best is then one answer and not a matter of rounding."""
    return (x / step).round().clamp(-most, most) * step


def _zipf(n, V, gen):
    """Token ids that fall off as a text's do (Zipf, s = 1.1)."""
    cdf = (torch.arange(1, V + 1, dtype=torch.float64) ** -1.1).cumsum(0)  # on the host: the same each time
    cdf = (cdf / cdf[-1]).float().cuda()
    return torch.searchsorted(cdf, torch.rand(n, device="cuda", generator=gen)).clamp_(max=V - 1)


def _clip_shapes(c):
    """The shapes of a UnifiedLM's parameters: nine tensors a block, the final norm, the embedding."""
    D, M = c["D"], c["M"]
    block = [(D,), (D, 1, 4), (M, D), (M,), (D, M), (), (D, D), (), (M,)]
    return block * c["L"] + [(D,), (c["V"], D)]


def prepare(case, seed):
    s, c = _State(), case
    s.case = c
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    dt = _DT[c["dtype"]]
    if c["kind"] == "head":
        N, V, D = c["N"], c["V"], c["D"]
        s.tokens = _zipf(N, V, gen)
        u = normal(V, D)
        # hidden states lean towards the given token by a share of their own, as a trained model's do;
        # bf16 operands have steps of 2^-5 and 2^-12 (8 digits), fp32 ones of 2^-8 and 2^-12
        lean = torch.rand(N, 1, device="cuda", generator=gen) * 0.5
        h = normal(N, D) + lean * u[s.tokens]
        s.h = (_on_grid(h, 2.0 ** -5, 127) if dt == torch.bfloat16 else _on_grid(h, 2.0 ** -8, 1023)).to(dt)
        s.weight = _on_grid(u * 0.02, 2.0 ** -12, 255).to(dt)
    elif c["kind"] == "logits":
        N, V = c["N"], c["V"]
        s.tokens = _zipf(N, V, gen)
        s.logits = (normal(N, V) * 2.5).to(dt)
        if not c["train"]:  # a grammar leaves about 70% of the tokens open, the given one among them
            shut = torch.rand(N, V, device="cuda", generator=gen) < 0.3
            shut[torch.arange(N, device="cuda"), s.tokens] = False
            s.logits.masked_fill_(shut, float("-inf"))
            del shut
    elif c["kind"] == "embed":
        s.tokens = _zipf(c["N"], c["V"], gen)
        s.weight = (normal(c["V"], c["D"]) * 0.02).to(dt)
        s.dy = normal(c["N"], c["D"]).to(dt)
    else:
        shapes = _clip_shapes(c)
        sizes = [math.prod(x) for x in shapes]
        std = 1e-3
        fresh = normal(sum(sizes)) * std
        if c["inplace"]:  # the step's gradients, as they arrive, and the bucket that they are clipped in
            s.fresh = fresh.to(dt)
            s.flat = torch.empty_like(s.fresh)
            s.grads = [v.view(x) for v, x in zip(s.flat.split(sizes), shapes)]
        else:
            s.grads = [v.to(dt, copy=True).view(x) for v, x in zip(fresh.split(sizes), shapes)]
            s.flat = torch.empty(sum(sizes), device="cuda")
            s.out = [v.view(x) for v, x in zip(s.flat.split(sizes), shapes)]
        return s
    # about one position in twenty is padding
    s.tokens[torch.rand(c["N"], device="cuda", generator=gen) < 0.05] = -1
    if c["kind"] != "embed" and c["train"]:
        s.dlogprobs = normal(c["N"]) / c["N"]  # advantages
        s.dentropy = torch.full((c["N"],), 0.01 / c["N"], device="cuda")  # entropy bonus
    if c["train"]:
        for t in (getattr(s, n, None) for n in ("h", "weight", "logits")):
            if t is not None:
                t.requires_grad_()
    return s


# ---- plain forms -------------------------------------------------------------------------------------

def _plain_stats(x, tokens, k):
    """(log softmax, its entropy, outputs) of fp32 logits x."""
    m = x.amax(-1, keepdim=True)
    logp = x - m
    logp = logp - logp.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    given = logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    out = {"logprobs": torch.where(tokens >= 0, given, 0.0), "entropy": entropy}
    if k:
        # whole numbers in the values' order, the lower index first among equals
        bits = (x + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32
        key = key + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))
        ids = x.shape[1] - 1 - (key.topk(k, dim=-1).values & 0xFFFFFFFF)
        out["top_ids"], out["top_logprobs"] = ids, logp.gather(1, ids)
    return logp, entropy, out


def _plain_dlogits(logp, entropy, s):
    p = logp.exp()
    given = torch.where(s.tokens >= 0, s.dlogprobs, 0.0)
    d = -p * (given[:, None] + s.dentropy[:, None] * (logp + entropy[:, None]))
    return d.scatter_add_(1, s.tokens.clamp(min=0)[:, None], given[:, None])


def _plain_head(s):
    h, w = s.h.detach().float(), s.weight.detach().float()
    logp, entropy, out = _plain_stats(h @ w.t(), s.tokens, s.case["k"])
    if s.case["train"]:
        d = _plain_dlogits(logp, entropy, s)
        out["dh"], out["dweight"] = (d @ w).to(s.h.dtype), (d.t() @ h).to(s.weight.dtype)
    return out


def _plain_logits(s):
    logp, entropy, out = _plain_stats(s.logits.detach().float(), s.tokens, s.case["k"])
    if s.case["train"]:
        out["dlogits"] = _plain_dlogits(logp, entropy, s).to(s.logits.dtype)
    return out


def _plain_embed(s):
    w, pad = s.weight.detach(), (s.tokens < 0)[:, None]
    rows = w[s.tokens.clamp(min=0)].float() * s.case["scale"]
    out = {"y": rows.masked_fill(pad, 0.0).to(w.dtype)}
    if s.case["train"]:
        dy = (s.dy.float() * s.case["scale"]).masked_fill(pad, 0.0)
        dw = torch.zeros(w.shape, device=w.device)
        out["dweight"] = dw.index_add_(0, s.tokens.clamp(min=0), dy).to(w.dtype)
    return out


def _plain_clip(s):
    if s.case["inplace"]:
        s.flat.copy_(s.fresh)
    norm = torch.stack([g.float().square().sum() for g in s.grads]).sum().sqrt()
    factor = (s.case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [o.copy_(g.float() * factor) for g, o in zip(s.grads, s.grads if s.case["inplace"] else s.out)]
    return {"norm": norm, "grads": s.flat}


# ---- the framework's entry points --------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _framework():
    from __graft_entry__ import load_package
    load_package()
    from unifiedlm_c_b200 import clip, embed, logprobs
    return logprobs, embed, clip


def _as_dict(r, k):
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    return dict(out, top_ids=r.top_ids, top_logprobs=r.top_logprobs) if k else out


def _own_head(s):
    c = s.case
    r = _framework()[0].lm_head_logprobs(s.h, s.weight, s.tokens, top_k=c["k"], precision=c["dtype"])
    out = _as_dict(r, c["k"])
    if c["train"]:
        out["dh"], out["dweight"] = torch.autograd.grad([r.logprobs, r.entropy], [s.h, s.weight], [s.dlogprobs, s.dentropy])
    return out


def _own_logits(s):
    c = s.case
    r = _framework()[0].token_logprobs(s.logits, s.tokens, top_k=c["k"])
    out = _as_dict(r, c["k"])
    if c["train"]:
        out["dlogits"], = torch.autograd.grad([r.logprobs, r.entropy], [s.logits], [s.dlogprobs, s.dentropy])
    return out


def _own_embed(s):
    y = _framework()[1].embedding(s.tokens, s.weight, scale=s.case["scale"])
    if not s.case["train"]:
        return {"y": y}
    return {"y": y, "dweight": torch.autograd.grad(y, s.weight, s.dy)[0]}


def _own_clip(s):
    clip = _framework()[2]
    if s.case["inplace"]:
        s.flat.copy_(s.fresh)
        return {"norm": clip.clip_grads(s.grads, s.case["max_norm"]), "grads": s.flat}
    return {"norm": clip.clip_grads(s.grads, s.case["max_norm"], out=s.out), "grads": s.flat}


_PLAIN = {"head": _plain_head, "logits": _plain_logits, "embed": _plain_embed, "clip": _plain_clip}
_OWN = {"head": _own_head, "logits": _own_logits, "embed": _own_embed, "clip": _own_clip}


def run(state):
    return (_OWN if own else _PLAIN)[state.case["kind"]](state)


# ---- work and exact values ---------------------------------------------------------------------------

def work(case):
    c = case
    es = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "head":
        N, V, D = c["N"], c["V"], c["D"]
        operands = (N + V) * D * es
        return {"bytes": operands * (2 if c["train"] else 1) + N * (16 + 12 * c["k"]),
                "flops": 2 * N * V * D * (3 if c["train"] else 1)}
    if c["kind"] == "logits":
        N, V = c["N"], c["V"]
        return {"bytes": N * V * es * (2 if c["train"] else 1) + N * (16 + 12 * c["k"]), "flops": 6 * N * V}
    if c["kind"] == "embed":
        N, V, D = c["N"], c["V"], c["D"]
        there = (min(N, V) + N) * D * es + 8 * N
        return {"bytes": there + ((N + V) * D * es if c["train"] else 0), "flops": N * D * (2 if c["train"] else 1)}
    n = sum(math.prod(x) for x in _clip_shapes(c))
    return {"bytes": n * (es + (es if c["inplace"] else 4)), "flops": 3 * n}


def _exact_rows(x, tokens, k):
    """Outputs and log probabilities of rows of logits in 64 bits."""
    lse = torch.logsumexp(x, -1, keepdim=True)
    logp = x - lse
    p = logp.exp()
    out = {"logprobs": torch.where(tokens < 0, 0.0, logp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]),
           "entropy": -torch.nan_to_num(p * logp, nan=0.0).sum(-1)}
    if k:
        left, ids = x.clone(), []
        place = torch.arange(x.shape[1], device=x.device).expand_as(x)
        for _ in range(k):
            best = left.amax(-1, keepdim=True)
            at = torch.where(left == best, place, x.shape[1]).amin(-1, keepdim=True)
            ids.append(at)
            left.scatter_(1, at, float("nan"))
            left = torch.where(left.isnan(), -math.inf, left)
        out["top_ids"] = torch.cat(ids, 1)
        out["top_logprobs"] = logp.gather(1, out["top_ids"])
    return out, logp, p


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    with torch.no_grad():
        if c["kind"] == "embed":
            keep = (s.tokens >= 0).double()[:, None]
            at = s.tokens.clamp(min=0)
            out = {"y": s.weight.double()[at] * c["scale"] * keep}
            if c["train"]:
                dw = torch.zeros(s.weight.shape, dtype=torch.float64, device="cuda")
                out["dweight"] = dw.index_put_((at,), s.dy.double() * c["scale"] * keep, accumulate=True)
            return out
        if c["kind"] == "clip":
            g = s.fresh.double() if c["inplace"] else torch.cat([x.reshape(-1) for x in s.grads]).double()
            norm = torch.linalg.vector_norm(g)
            return {"norm": norm, "grads": g * min(1.0, c["max_norm"] / (float(norm) + 1e-6))}
        parts, wide = [], max(1, (1 << 26) // c["V"])
        w = s.weight.double() if c["kind"] == "head" else None
        dw = torch.zeros_like(w) if w is not None and c["train"] else None
        for a in range(0, c["N"], wide):
            rows = slice(a, a + wide)
            t = s.tokens[rows]
            x = s.h[rows].double() @ w.t() if w is not None else s.logits[rows].double()
            out, logp, p = _exact_rows(x, t, c["k"])
            if c["train"]:
                dlp, dent = s.dlogprobs[rows].double(), s.dentropy[rows].double()
                hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
                d = (dlp * (t >= 0))[:, None] * (hot - p) - dent[:, None] * p * (logp + out["entropy"][:, None])
                if w is None:
                    out["dlogits"] = d
                else:
                    out["dh"] = d @ w
                    dw += d.t() @ s.h[rows].double()
            parts.append(out)
        whole = {n: torch.cat([q[n] for q in parts]) for n in parts[0]}
        if dw is not None:
            whole["dweight"] = dw
        return whole
