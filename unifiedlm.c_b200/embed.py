"""Token embedding with a scale, and its weight's gradient, on sm_100a (model.py:149-150).

`embedding(tokens, weight, scale)` = weight[tokens] * scale, as nn.Embedding with a factor. The
gradient adds the rows of dy by token in fp32, in the order of their positions: the same bits in
every run. Token -1 is padding: a zero row, no gradient. Any other token outside the vocabulary gives
a NaN row. The work runs in libulm_b200.so (ulm_embedding_fwd / _bwd) through the `torch.library`
ops `ulm::embedding_fwd` and `ulm::embedding_bwd`. No CPU path.
"""
import torch

from . import _lib as L


def embedding_fwd_raw(tokens, weight, scale, out_bf16):
    """ulm_embedding_fwd on a fresh buffer: y (N, D)."""
    N = tokens.shape[0]
    V, D = weight.shape
    dt = torch.bfloat16 if out_bf16 else weight.dtype
    y = torch.empty(N, D, device=weight.device, dtype=dt)
    with L.on(weight.device):
        L.check(L.lib().ulm_embedding_fwd(tokens.data_ptr(), weight.data_ptr(), L.dtype_code(weight.dtype),
                                          weight.stride(0) if V > 1 else D, y.data_ptr(), L.dtype_code(dt), N, V, D,
                                          scale, L.stream(weight.device)))
    return y


def embedding_bwd_raw(tokens, dy, V, scale, dw_bf16):
    """ulm_embedding_bwd on a fresh buffer: dweight (V, D)."""
    N, D = dy.shape
    dt = torch.bfloat16 if dw_bf16 else torch.float32
    lib = L.lib()
    dw = torch.empty(V, D, device=dy.device, dtype=dt)
    work = torch.empty(lib.ulm_embedding_bwd_work_bytes(N, V, D), device=dy.device, dtype=torch.uint8)
    with L.on(dy.device):
        L.check(lib.ulm_embedding_bwd(tokens.data_ptr(), dy.data_ptr(), L.dtype_code(dy.dtype), dw.data_ptr(),
                                      L.dtype_code(dt), work.data_ptr(), N, V, D, scale, L.stream(dy.device)))
    return dw


class _Embedding(torch.autograd.Function):
    """The eager form of the two ops below."""

    @staticmethod
    def forward(ctx, tokens, weight, scale, out_bf16):
        ctx.save_for_backward(tokens)
        ctx.meta = (weight.shape[0], scale, weight.dtype == torch.bfloat16)
        ctx.set_materialize_grads(False)
        return embedding_fwd_raw(tokens, weight, scale, out_bf16)

    @staticmethod
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None
        L.first_order("embedding")
        return None, embedding_bwd_raw(*ctx.saved_tensors, dy.contiguous(), *ctx.meta), None, None


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
    tk = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    tk = tk.to(torch.int64).contiguous()
    args = tk, w, float(scale), out_dtype == torch.bfloat16
    if not L.eager(tk, w):
        L.no_tangents("embedding", w)
        y = torch.ops.ulm.embedding_fwd(*args)
    elif w.requires_grad and torch.is_grad_enabled():
        y = _Embedding.apply(*args)
    else:
        y = embedding_fwd_raw(*args)
    return y if tokens.dim() == 1 else y.view(*tokens.shape, D)
