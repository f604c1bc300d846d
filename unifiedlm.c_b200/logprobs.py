"""Log probabilities of given tokens on sm_100a, with the entropy and the best alternatives.

For logits x of a row and its token t (the log_softmax and gather that score a text, a policy's
samples or a decode step; the reference's logits are model.py:153-157):

    logprob = x_t - logsumexp(x),   entropy = - sum_v p_v log p_v,   p = softmax(x)

and the `top_k` best tokens in descending order (the lower id first among equals).

`lm_head_logprobs(h, weight, tokens)` takes the logits h @ weight.T of the output Linear, like
`head.lm_head_loss`; `token_logprobs(logits, tokens)` takes logits that exist already (a decode
step's, `BatchedDecoder.logprobs`). Both are differentiable in logprobs and entropy. Token -1 is
padding: logprob 0, no gradient through it. Any other token outside the vocabulary makes its
logprob, and the gradients that it reaches, NaN. Masked tokens (logits of -inf) of `token_logprobs`
have probability 0; a row that is masked throughout, or holds a NaN or +inf, has NaN results, as
log_softmax has. The products of `lm_head_logprobs` are taken as finite: a row with one that is not has
a NaN entropy (and logprobs, but for -inf), and its alternatives are some top_k different tokens. The
work runs in libulm_b200.so (ulm_lm_head_logprobs_*, ulm_token_logprobs_*) through `torch.library`
ops. No CPU path.
"""
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .kernel import PRECISION, _op_dtype, operand_ld

MAX_TOP_K = 32


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # (...) fp32
    entropy: torch.Tensor       # (...) fp32
    top_ids: torch.Tensor       # (..., top_k) int64
    top_logprobs: torch.Tensor  # (..., top_k) fp32


def _operand(x, opt):
    """(matrix, row stride) of a 2-d operand of a product: x itself where it can be read in place, else
    a padded copy in the operand type."""
    n, d = x.shape
    ld = x.stride(0) if n > 1 else operand_ld(d)
    if (x.dtype == opt and (d == 1 or x.stride(1) == 1) and ld >= d and
            (opt == torch.float32 or (ld % 8 == 0 and x.data_ptr() % 16 == 0))):
        return x, ld
    c = torch.empty(n, operand_ld(d), device=x.device, dtype=opt)
    c[:, :d] = x
    return c, operand_ld(d)


def _outputs(N, top_k, dev, stats=True):
    f32 = dict(device=dev, dtype=torch.float32)
    return (torch.empty(N, **f32), torch.empty(N, **f32), torch.empty(N, 2, **f32) if stats else None,
            torch.empty(N, top_k, device=dev, dtype=torch.int64), torch.empty(N, top_k, **f32))


def _addr(t):
    return None if t is None else t.data_ptr()


_OUT = tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]


# ---- from hidden states -------------------------------------------------------------------------------

def lm_head_logprobs_fwd_raw(h, weight, tokens, top_k, precision, stats=True):
    """ulm_lm_head_logprobs_fwd on fresh buffers: (logprobs, entropy, stats or None, top_ids,
    top_logprobs)."""
    N, D = h.shape
    V = weight.shape[0]
    lib = L.lib()
    out = lp, ent, st, ids, tlp = _outputs(N, top_k, h.device, stats)
    opt = _op_dtype(precision)
    h_op, ld_h = _operand(h, opt)
    w_op, ld_w = _operand(weight, opt)
    with L.on(h.device):
        work = torch.empty(lib.ulm_lm_head_logprobs_work_bytes(N, V, D, top_k, 0, precision), device=h.device,
                           dtype=torch.uint8)
        L.check(lib.ulm_lm_head_logprobs_fwd(h_op.data_ptr(), ld_h, w_op.data_ptr(), ld_w, tokens.data_ptr(),
                                             lp.data_ptr(), ent.data_ptr(), _addr(st), ids.data_ptr(), tlp.data_ptr(),
                                             work.data_ptr(), N, V, D, top_k, precision, L.stream(h.device)))
    return out


def lm_head_logprobs_bwd_raw(dlp, dent, h, weight, tokens, stats, ent, precision, need_dh, need_dw):
    """ulm_lm_head_logprobs_bwd on fresh buffers: (dh, dweight), None for one that is not needed."""
    N, D = h.shape
    V = weight.shape[0]
    lib = L.lib()
    dh = torch.empty(N, D, device=h.device, dtype=h.dtype) if need_dh else None
    dw = torch.empty(V, D, device=h.device, dtype=weight.dtype) if need_dw else None
    opt = _op_dtype(precision)
    h_op, ld_h = _operand(h, opt)
    w_op, ld_w = _operand(weight, opt)
    with L.on(h.device):
        work = torch.empty(lib.ulm_lm_head_logprobs_work_bytes(N, V, D, 0, 1, precision), device=h.device,
                           dtype=torch.uint8)
        L.check(lib.ulm_lm_head_logprobs_bwd(
            _addr(dlp), _addr(dent), h_op.data_ptr(), ld_h, w_op.data_ptr(), ld_w, tokens.data_ptr(), stats.data_ptr(),
            ent.data_ptr(), _addr(dh), L.dtype_code(h.dtype), _addr(dw), L.dtype_code(weight.dtype), work.data_ptr(),
            N, V, D, precision, L.stream(h.device)))
    return dh, dw


def _grad_in(g):
    return None if g is None else g.float().contiguous()


class _HeadLogprobs(torch.autograd.Function):
    """The eager form of the two ops below."""

    @staticmethod
    def forward(ctx, h, weight, tokens, top_k, precision):
        lp, ent, stats, ids, tlp = lm_head_logprobs_fwd_raw(h, weight, tokens, top_k, precision)
        ctx.save_for_backward(h, weight, tokens, stats, ent)
        ctx.precision = precision
        ctx.mark_non_differentiable(ids, tlp)
        ctx.set_materialize_grads(False)
        return lp, ent, ids, tlp

    @staticmethod
    def backward(ctx, dlp, dent, *unused):
        if dlp is None and dent is None:
            return None, None, None, None, None
        L.first_order("lm_head_logprobs")
        dh, dw = lm_head_logprobs_bwd_raw(_grad_in(dlp), _grad_in(dent), *ctx.saved_tensors, ctx.precision,
                                          *ctx.needs_input_grad[:2])
        return dh, dw, None, None, None


@torch.library.custom_op("ulm::lm_head_logprobs_fwd", mutates_args=())
def lm_head_logprobs_fwd(h: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor, top_k: int, precision: int) -> _OUT:
    """h (N, D), weight (V, D), tokens (N,) int64. Returns (logprobs, entropy, stats, top_ids,
    top_logprobs); stats (N, 2) is saved for the backward."""
    return lm_head_logprobs_fwd_raw(h, weight, tokens, top_k, precision)


@lm_head_logprobs_fwd.register_fake
def _lm_head_logprobs_fwd_fake(h, weight, tokens, top_k, precision):
    return _outputs(h.shape[0], top_k, h.device)


@torch.library.custom_op("ulm::lm_head_logprobs_bwd", mutates_args=())
def lm_head_logprobs_bwd(dlp: Optional[torch.Tensor], dent: Optional[torch.Tensor], h: torch.Tensor,
                         weight: torch.Tensor, tokens: torch.Tensor, stats: torch.Tensor, ent: torch.Tensor,
                         precision: int, need_dh: bool, need_dw: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Returns (dh in h's type, dweight in weight's type); one that is not needed is empty."""
    dh, dw = lm_head_logprobs_bwd_raw(dlp, dent, h, weight, tokens, stats, ent, precision, need_dh, need_dw)
    return h.new_empty(0) if dh is None else dh, weight.new_empty(0) if dw is None else dw


@lm_head_logprobs_bwd.register_fake
def _lm_head_logprobs_bwd_fake(dlp, dent, h, weight, tokens, stats, ent, precision, need_dh, need_dw):
    return (torch.empty(h.shape if need_dh else (0,), device=h.device, dtype=h.dtype),
            torch.empty(weight.shape if need_dw else (0,), device=h.device, dtype=weight.dtype))


def _head_setup(ctx, inputs, output):
    h, weight, tokens, top_k, precision = inputs
    _, ent, stats, ids, tlp = output
    ctx.save_for_backward(h, weight, tokens, stats, ent)
    ctx.precision = precision
    ctx.mark_non_differentiable(stats, ids, tlp)
    ctx.set_materialize_grads(False)


def _head_backward(ctx, dlp, dent, *unused):
    if dlp is None and dent is None:
        return (None,) * 5
    h, weight, tokens, stats, ent = ctx.saved_tensors
    need_dh, need_dw = ctx.needs_input_grad[:2]
    dh, dw = lm_head_logprobs_bwd(_grad_in(dlp), _grad_in(dent), h, weight, tokens, stats, ent, ctx.precision,
                                  need_dh, need_dw)
    return dh if need_dh else None, dw if need_dw else None, None, None, None


torch.library.register_autograd("ulm::lm_head_logprobs_fwd", _head_backward, setup_context=_head_setup)


# ---- from logits --------------------------------------------------------------------------------------

def _row_stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def token_logprobs_fwd_raw(logits, tokens, top_k, stats=True):
    """ulm_token_logprobs_fwd on fresh buffers, as lm_head_logprobs_fwd_raw."""
    N, V = logits.shape
    out = lp, ent, st, ids, tlp = _outputs(N, top_k, logits.device, stats)
    with L.on(logits.device):
        L.check(L.lib().ulm_token_logprobs_fwd(logits.data_ptr(), L.dtype_code(logits.dtype), _row_stride(logits),
                                               tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(), _addr(st),
                                               ids.data_ptr(), tlp.data_ptr(), N, V, top_k, L.stream(logits.device)))
    return out


def token_logprobs_bwd_raw(dlp, dent, logits, tokens, stats, ent):
    """ulm_token_logprobs_bwd on a fresh buffer: dlogits (N, V) in logits' type."""
    N, V = logits.shape
    d = torch.empty(N, V, device=logits.device, dtype=logits.dtype)
    with L.on(logits.device):
        L.check(L.lib().ulm_token_logprobs_bwd(_addr(dlp), _addr(dent), logits.data_ptr(), L.dtype_code(logits.dtype),
                                               _row_stride(logits), tokens.data_ptr(), stats.data_ptr(), ent.data_ptr(),
                                               d.data_ptr(), V, N, V, L.stream(logits.device)))
    return d


class _TokenLogprobs(torch.autograd.Function):
    """The eager form of the two ops below."""

    @staticmethod
    def forward(ctx, logits, tokens, top_k):
        lp, ent, stats, ids, tlp = token_logprobs_fwd_raw(logits, tokens, top_k)
        ctx.save_for_backward(logits, tokens, stats, ent)
        ctx.mark_non_differentiable(ids, tlp)
        ctx.set_materialize_grads(False)
        return lp, ent, ids, tlp

    @staticmethod
    def backward(ctx, dlp, dent, *unused):
        if dlp is None and dent is None:
            return None, None, None
        L.first_order("token_logprobs")
        return token_logprobs_bwd_raw(_grad_in(dlp), _grad_in(dent), *ctx.saved_tensors), None, None


@torch.library.custom_op("ulm::token_logprobs_fwd", mutates_args=())
def token_logprobs_fwd(logits: torch.Tensor, tokens: torch.Tensor, top_k: int) -> _OUT:
    """logits (N, V), tokens (N,) int64; the outputs of lm_head_logprobs_fwd."""
    return token_logprobs_fwd_raw(logits, tokens, top_k)


@token_logprobs_fwd.register_fake
def _token_logprobs_fwd_fake(logits, tokens, top_k):
    return _outputs(logits.shape[0], top_k, logits.device)


@torch.library.custom_op("ulm::token_logprobs_bwd", mutates_args=())
def token_logprobs_bwd(dlp: Optional[torch.Tensor], dent: Optional[torch.Tensor], logits: torch.Tensor,
                       tokens: torch.Tensor, stats: torch.Tensor, ent: torch.Tensor) -> torch.Tensor:
    """Returns dlogits (N, V) in logits' type."""
    return token_logprobs_bwd_raw(dlp, dent, logits, tokens, stats, ent)


@token_logprobs_bwd.register_fake
def _token_logprobs_bwd_fake(dlp, dent, logits, tokens, stats, ent):
    return torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)


def _logits_setup(ctx, inputs, output):
    logits, tokens, top_k = inputs
    _, ent, stats, ids, tlp = output
    ctx.save_for_backward(logits, tokens, stats, ent)
    ctx.mark_non_differentiable(stats, ids, tlp)
    ctx.set_materialize_grads(False)


def _logits_backward(ctx, dlp, dent, *unused):
    if dlp is None and dent is None:
        return None, None, None
    logits, tokens, stats, ent = ctx.saved_tensors
    return token_logprobs_bwd(_grad_in(dlp), _grad_in(dent), logits, tokens, stats, ent), None, None


torch.library.register_autograd("ulm::token_logprobs_fwd", _logits_backward, setup_context=_logits_setup)


# ---- entry points -------------------------------------------------------------------------------------

def _check(x, tokens, V, top_k, name):
    if not x.is_cuda:
        raise RuntimeError(f"{name} runs on CUDA tensors only (no CPU path)")
    if x.dim() < 1 or tokens.shape != x.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} do not match the rows of {tuple(x.shape)}")
    if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
        raise TypeError(f"tokens must be integers, got {tokens.dtype}")
    if tokens.device != x.device:
        raise ValueError(f"tokens on {tokens.device}, {x.device} expected")
    if V < 1:
        raise ValueError("empty vocabulary")
    if not 0 <= top_k <= min(V, MAX_TOP_K):
        raise ValueError(f"top_k={top_k} must be in 0 .. min(vocabulary, {MAX_TOP_K})")


def _rows(t):
    """tokens as one int64 row"""
    t = t if t.dim() == 1 else t.reshape(-1)
    return t.to(torch.int64).contiguous()


def _shaped(out, shape, top_k):
    lp, ent, ids, tlp = out[0], out[1], out[-2], out[-1]
    if len(shape) == 1:
        return TokenLogprobs(lp, ent, ids, tlp)
    return TokenLogprobs(lp.view(shape), ent.view(shape), ids.view(*shape, top_k), tlp.view(*shape, top_k))


def lm_head_logprobs(h, weight, tokens, top_k=0, precision="bf16"):
    """TokenLogprobs of `tokens` (...) under the logits h @ weight.T: h (..., D) fp32 or bf16, weight
    (V, D) fp32 or bf16. "bf16" contracts bf16 operands (rounding fp32 ones; the logits' gradient goes
    into its products in two bf16 parts, 16 digits), "fp32" fp32 ones; the statistics are fp32. Gradients of h and weight flow from logprobs and entropy, in the types of h
    and weight; the alternatives are not differentiable."""
    if weight.dim() != 2 or h.dim() < 1 or h.shape[-1] != weight.shape[1]:
        raise ValueError(f"h {tuple(h.shape)} and weight {tuple(weight.shape)} do not match")
    if precision not in PRECISION:
        raise ValueError(f"precision must be one of {sorted(PRECISION)}, got {precision!r}")
    _check(h, tokens, weight.shape[0], top_k, "lm_head_logprobs")
    if weight.device != h.device:
        raise ValueError(f"weight on {weight.device}, {h.device} expected")
    hh = h if h.dim() == 2 else h.reshape(-1, h.shape[-1])
    hh = hh if hh.dtype in (torch.float32, torch.bfloat16) else hh.float()
    ww = weight if weight.dtype in (torch.float32, torch.bfloat16) else weight.float()
    args = hh, ww, _rows(tokens), top_k, PRECISION[precision]
    if not L.eager(hh, ww, tokens):
        L.no_tangents("lm_head_logprobs", hh, ww)
        out = torch.ops.ulm.lm_head_logprobs_fwd(*args)
    elif (hh.requires_grad or ww.requires_grad) and torch.is_grad_enabled():
        out = _HeadLogprobs.apply(*args)
    else:
        out = lm_head_logprobs_fwd_raw(*args, stats=False)
    return _shaped(out, tokens.shape, top_k)


def token_logprobs(logits, tokens, top_k=0):
    """TokenLogprobs of `tokens` (...) under `logits` (..., V) fp32 or bf16."""
    _check(logits, tokens, logits.shape[-1] if logits.dim() else 0, top_k, "token_logprobs")
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    x = x if x.dtype in (torch.float32, torch.bfloat16) else x.float()
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    tk = _rows(tokens)
    if not L.eager(x, tokens):
        L.no_tangents("token_logprobs", x)
        out = torch.ops.ulm.token_logprobs_fwd(x, tk, top_k)
    elif x.requires_grad and torch.is_grad_enabled():
        out = _TokenLogprobs.apply(x, tk, top_k)
    else:
        out = token_logprobs_fwd_raw(x, tk, top_k, stats=False)
    return _shaped(out, tokens.shape, top_k)
