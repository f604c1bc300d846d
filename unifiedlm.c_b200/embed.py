"""Token embedding with a scale, and its weight's gradient, on sm_100a (model.py:149-150).

`embedding(tokens, weight, scale)` = weight[tokens] * scale, as nn.Embedding with a factor. The
gradient adds the rows of dy by token in fp32, in the order of their positions: the same bits in
every run. Token -1 is padding: a zero row, no gradient. Any other token outside the vocabulary gives
a NaN row. The work runs in libulm_b200.so (ulm_embedding_fwd / _bwd) through the `torch.library`
ops `ulm::embedding_fwd` and `ulm::embedding_bwd`. No CPU path.
"""
import functools

import torch

from . import _lib as L


_FLOATS = {torch.float32, torch.bfloat16}
_INTEGERS = {torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8, torch.uint16, torch.uint32, torch.uint64}


def embedding_fwd_raw(tokens, weight, scale, out_bf16):
    """ulm_embedding_fwd on a fresh buffer: y (N, D)."""
    N = tokens.shape[0]
    V, D = weight.shape
    dev, wdt = weight.device, weight.dtype
    dt = torch.bfloat16 if out_bf16 else wdt
    y = torch.empty(N, D, device=dev, dtype=dt)
    with L.on(dev):
        L.check(L.lib().ulm_embedding_fwd(tokens.data_ptr(), weight.data_ptr(), L.dtype_code(wdt),
                                          weight.stride(0) if V > 1 else D, y.data_ptr(), L.dtype_code(dt), N, V, D,
                                          scale, L.stream(dev)))
    return y


@functools.lru_cache(maxsize=1024)
def _work_bytes(N, V, D):
    return L.lib().ulm_embedding_bwd_work_bytes(N, V, D)


def embedding_bwd_raw(tokens, dy, V, scale, dw_bf16):
    """ulm_embedding_bwd on a fresh buffer: dweight (V, D)."""
    N, D = dy.shape
    dt = torch.bfloat16 if dw_bf16 else torch.float32
    dev = dy.device
    dw = torch.empty(V, D, device=dev, dtype=dt)
    work = torch.empty(_work_bytes(N, V, D), device=dev, dtype=torch.uint8)
    with L.on(dev):
        L.check(L.lib().ulm_embedding_bwd(tokens.data_ptr(), dy.data_ptr(), L.dtype_code(dy.dtype), dw.data_ptr(),
                                          L.dtype_code(dt), work.data_ptr(), N, V, D, scale, L.stream(dev)))
    return dw


class _Embedding(torch.autograd.Function):
    """The eager form of the two ops below."""

    @staticmethod
    def forward(ctx, weight, rest):
        tokens, scale, out_bf16 = rest
        ctx.save_for_backward(tokens)
        ctx.meta = (weight.shape[0], scale, weight.dtype == torch.bfloat16)
        ctx.set_materialize_grads(False)
        return embedding_fwd_raw(tokens, weight, scale, out_bf16)

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None
        L.first_order("embedding")
        return embedding_bwd_raw(*ctx.saved_tensors, dy.contiguous(), *ctx.meta), None


@torch.library.custom_op("ulm::embedding_fwd", mutates_args=())
def embedding_fwd(tokens: torch.Tensor, weight: torch.Tensor, scale: float, out_bf16: bool) -> torch.Tensor:
    """tokens (N,) int64, weight (V, D); y (N, D) in weight's type, or bf16 (out_bf16)."""
    return embedding_fwd_raw(tokens, weight, scale, out_bf16)


@embedding_fwd.register_fake
def _embedding_fwd_fake(tokens, weight, scale, out_bf16):
    return torch.empty(tokens.shape[0], weight.shape[1], device=weight.device,
                       dtype=torch.bfloat16 if out_bf16 else weight.dtype)


@torch.library.custom_op("ulm::embedding_bwd", mutates_args=())
def embedding_bwd(tokens: torch.Tensor, dy: torch.Tensor, V: int, scale: float, dw_bf16: bool) -> torch.Tensor:
    """dweight (V, D), fp32 or bf16, of dy (N, D)."""
    return embedding_bwd_raw(tokens, dy, V, scale, dw_bf16)


@embedding_bwd.register_fake
def _embedding_bwd_fake(tokens, dy, V, scale, dw_bf16):
    return torch.empty(V, dy.shape[1], device=dy.device, dtype=torch.bfloat16 if dw_bf16 else torch.float32)


def _setup(ctx, inputs, output):
    tokens, weight, scale, out_bf16 = inputs
    ctx.save_for_backward(tokens)
    ctx.meta = (weight.shape[0], scale, weight.dtype == torch.bfloat16)
    ctx.set_materialize_grads(False)


def _backward(ctx, dy):
    if dy is None:
        return None, None, None, None
    tokens, = ctx.saved_tensors
    V, scale, bf16 = ctx.meta
    return None, embedding_bwd(tokens, dy.contiguous(), V, scale, bf16), None, None


torch.library.register_autograd("ulm::embedding_fwd", _backward, setup_context=_setup)


def embedding(tokens, weight, scale=1.0, out_dtype=None):
    """scale * weight[tokens]: tokens (...) integer, weight (V, D) fp32 or bf16 on the GPU; (..., D) in
    weight's type, or bf16 with out_dtype=torch.bfloat16. The weight's gradient has the weight's type."""
    if not weight.is_cuda:
        raise RuntimeError("embedding runs on CUDA tensors only (no CPU path)")
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be a (V, D) matrix, got {tuple(weight.shape)}")
    dt = weight.dtype
    if dt not in _FLOATS:
        raise TypeError(f"weight must be fp32 or bf16, got {dt}")
    if tokens.dtype not in _INTEGERS:
        raise TypeError(f"tokens must be integers, got {tokens.dtype}")
    if tokens.get_device() != weight.get_device():
        raise ValueError(f"tokens on {tokens.device}, {weight.device} expected")
    if out_dtype is not None and out_dtype not in (dt, torch.bfloat16):
        raise ValueError(f"out_dtype must be the weight's type or bf16, got {out_dtype}")
    w = weight
    if not w.is_contiguous():
        V, D = w.shape
        if D > 1 and w.stride(1) != 1 or V > 1 and w.stride(0) < D:
            w = w.contiguous()
    tk = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    if tk.dtype != torch.int64 or not tk.is_contiguous():
        tk = tk.to(torch.int64).contiguous()
    scale, out_bf16 = float(scale), out_dtype == torch.bfloat16
    if not L.eager(tk, w):
        L.no_tangents("embedding", w)
        y = torch.ops.ulm.embedding_fwd(tk, w, scale, out_bf16)
    elif w.requires_grad and torch.is_grad_enabled():
        y = _Embedding.apply(w, (tk, scale, out_bf16))
    else:
        y = embedding_fwd_raw(tk, w, scale, out_bf16)
    return y if tk is tokens or tokens.dim() == 1 else y.view(*tokens.shape, y.shape[1])
