"""Token embedding with a scale, and its weight's gradient, on sm_100a (model.py:149-150).

`embedding(tokens, weight, scale)` = weight[tokens] * scale, as nn.Embedding with a factor. The
gradient adds the rows of dy by token in fp32, in the order of their positions: the same bits in
every run. Token -1 is padding: a zero row, no gradient. Any other token outside the vocabulary gives
a NaN row. The work runs in libulm_b200.so (ulm_embedding_fwd / _bwd) through the `torch.library`
ops `ulm::embedding_fwd` and `ulm::embedding_bwd`. No CPU path.
"""
import torch

from . import _lib as L


@torch.library.custom_op("ulm::embedding_fwd", mutates_args=())
def embedding_fwd(tokens: torch.Tensor, weight: torch.Tensor, scale: float, out_bf16: bool) -> torch.Tensor:
    """tokens (N,) int64, weight (V, D); y (N, D) in weight's type, or bf16 (out_bf16)."""
    N = tokens.shape[0]
    V, D = weight.shape
    y = _embedding_fwd_fake(tokens, weight, scale, out_bf16)
    ld = weight.stride(0) if V > 1 else D
    with torch.cuda.device(weight.device):
        L.check(L.lib().ulm_embedding_fwd(L.ptr(tokens), L.ptr(weight), L.dtype_code(weight.dtype), ld, L.ptr(y),
                                          L.dtype_code(y.dtype), N, V, D, scale, L.stream_of(weight)))
    return y


@embedding_fwd.register_fake
def _embedding_fwd_fake(tokens, weight, scale, out_bf16):
    return torch.empty(tokens.shape[0], weight.shape[1], device=weight.device,
                       dtype=torch.bfloat16 if out_bf16 else weight.dtype)


@torch.library.custom_op("ulm::embedding_bwd", mutates_args=())
def embedding_bwd(tokens: torch.Tensor, dy: torch.Tensor, V: int, scale: float, dw_bf16: bool) -> torch.Tensor:
    """dweight (V, D), fp32 or bf16, of dy (N, D)."""
    N, D = dy.shape
    dw = _embedding_bwd_fake(tokens, dy, V, scale, dw_bf16)
    work = torch.empty(int(L.lib().ulm_embedding_bwd_work_bytes(N, V, D)), device=dy.device, dtype=torch.uint8)
    with torch.cuda.device(dy.device):
        L.check(L.lib().ulm_embedding_bwd(L.ptr(tokens), L.ptr(dy), L.dtype_code(dy.dtype), L.ptr(dw),
                                          L.dtype_code(dw.dtype), L.ptr(work), N, V, D, scale, L.stream_of(dy)))
    return dw


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
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be a (V, D) matrix, got {tuple(weight.shape)}")
    if weight.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"weight must be fp32 or bf16, got {weight.dtype}")
    if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
        raise TypeError(f"tokens must be integers, got {tokens.dtype}")
    if tokens.device != weight.device:
        raise ValueError(f"tokens on {tokens.device}, {weight.device} expected")
    if out_dtype not in (None, weight.dtype, torch.bfloat16):
        raise ValueError(f"out_dtype must be the weight's type or bf16, got {out_dtype}")
    V, D = weight.shape
    w = weight
    if D > 1 and w.stride(1) != 1 or V > 1 and w.stride(0) < D:
        w = w.contiguous()
    tk = tokens.reshape(-1).to(torch.int64).contiguous()
    y = torch.ops.ulm.embedding_fwd(tk, w, float(scale), out_dtype == torch.bfloat16)
    return y.view(*tokens.shape, D)
