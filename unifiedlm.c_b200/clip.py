"""The global gradient norm over many tensors, and clipping by it, on sm_100a (train.py:284).

    norm = sqrt(sum over all gradients of g^2),   g <- g * min(1, max_norm / (norm + 1e-6))

as torch.nn.utils.clip_grad_norm_ with the 2-norm, without a host synchronisation: `clip_grad_norm_`
takes parameters, `clip_grads` a list of gradients (in place, or into other tensors and types, such
as `GradBucket`'s views), `grad_norm` only measures. Squares are added in fp64 in a fixed order, so
the norm is the same in every run. A norm that is not finite makes the factor what IEEE division
gives (0 or NaN), as torch's function does. The work runs in libulm_b200.so (ulm_clip_grads) on the
current stream. No CPU path. Tracers (make_fx, torch.jit.trace) and gradients with a tangent are refused;
torch.compile breaks its graph at the call.
"""
import math
from array import array

import torch

from . import _lib as L


_CODE = {torch.float32: L.ULM_F32, torch.bfloat16: L.ULM_BF16}


def _codes(ts):
    try:
        return array("i", [_CODE[t.dtype] for t in ts])
    except KeyError as e:
        raise L.UlmError(f"unsupported element type {e.args[0]}") from None


def _dims(t):
    """{stride: size} of a tensor in bytes, its elements the innermost dimension; None where two of its
    dimensions have the same stride."""
    es = t.element_size()
    dims = {1: es}
    for n, s in zip(t.shape, t.stride()):
        if n > 1 and s > 0:
            if s * es in dims:
                return None
            dims[s * es] = n
    return dims


def _folded(t):
    """Whether elements of a tensor share memory (or may: each stride is to pass what lies within it)."""
    inner = 0
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s <= inner:
            return True
        inner += (n - 1) * s
    return False


def _end(t):
    if t.is_contiguous():
        return t.data_ptr() + t.nbytes
    return t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _apart(a, b):
    """Whether two tensors have no byte in common. Written in the strides of both, every address is one row
    of digits, as long as no digit of either tensor runs over into the next: they are apart where one
    digit's ranges are. Two starts to count from are tried; what cannot be written so is not apart."""
    if _end(a) <= b.data_ptr() or _end(b) <= a.data_ptr():
        return True
    if a.dim() == 2 and a.stride() == b.stride() and a.stride(1) == 1 and a.stride(0) > 0 and a.dtype == b.dtype:
        # blocks of one matrix (slices of a fused gradient): the digits below, its rows and columns
        base, es, pitch = a.untyped_storage().data_ptr(), a.element_size(), a.stride(0)
        (ra, ca), (rb, cb) = (divmod((t.data_ptr() - base) // es, pitch) for t in (a, b))
        (na, wa), (nb, wb) = a.shape, b.shape
        if ca + wa <= pitch and cb + wb <= pitch:
            return ra + na <= rb or rb + nb <= ra or ca + wa <= cb or cb + wb <= ca
    da, db = _dims(a), _dims(b)
    if da is None or db is None:
        return False
    strides = sorted({*da, *db}, reverse=True)
    for base in (min(a.data_ptr(), b.data_ptr()), a.untyped_storage().data_ptr()):
        ranges, exact = [], True
        for t, d in ((a, da), (b, db)):
            at, digits, last = t.data_ptr() - base, [], 0
            for s in strides:
                low, at = divmod(at, s)
                digits.append((low, low + d.get(s, 1) - 1))
            for s, outer, (_, high) in zip(strides[:0:-1], strides[-2::-1], digits[:0:-1]):
                last += high * s
                exact = exact and last < outer
            ranges.append(digits)
        if exact:
            return any(x[1] < y[0] or y[1] < x[0] for x, y in zip(*ranges))
    return False


def _check_strided(grads, outs):
    """The library's refusals of overlaps, for lists with tensors that it gets as copies."""
    if any(not o.is_contiguous() and _folded(o) for o in outs):
        raise ValueError("an output whose elements share memory")
    items = [(o.data_ptr(), _end(o), i, True, o) for i, o in enumerate(outs) if o.numel()]
    if outs is not grads:
        items += [(g.data_ptr(), _end(g), i, False, g) for i, (g, o) in enumerate(zip(grads, outs)) if g.numel() and g is not o]
    items.sort(key=lambda x: x[:2])
    reach = []  # those that go on past the one at hand
    for x in items:
        reach = [y for y in reach if y[1] > x[0]]
        for y in reach:
            if (x[3] or y[3]) and x[2] != y[2] and not _apart(x[4], y[4]):
                raise L.UlmError(f"gradient {x[2]} overlaps another one's output (the same tensor twice?)")
        reach.append(x)


def _run(grads, outs, max_norm):
    if not torch.compiler.is_compiling():
        L.not_traced("gradient clipping", grads)
    at = grads[0].get_device()
    for g in grads:
        if g.get_device() != at or at < 0:
            if not g.is_cuda:
                raise RuntimeError("gradient clipping runs on CUDA tensors only (no CPU path)")
            raise ValueError("gradients on several GPUs: one device expected")
        if g.layout is not torch.strided:
            raise ValueError("sparse gradients are not supported")
    n = len(grads)
    plain = [g.is_contiguous() for g in grads]
    src = grads if all(plain) else [g if c else g.contiguous() for g, c in zip(grads, plain)]
    dst = None
    if outs is grads:
        dst = src
        if src is not grads:
            _check_strided(grads, outs)
    elif outs is not None:
        plain_out = [o.is_contiguous() for o in outs]
        if src is not grads or not all(plain_out):
            _check_strided(grads, outs)
        dst = [s if o is g else o if c else torch.empty_like(o, memory_format=torch.contiguous_format)
               for g, s, o, c in zip(grads, src, outs, plain_out)]
    lib, dev = L.lib(), grads[0].device
    norm = torch.empty((), device=dev, dtype=torch.float32)
    work = torch.empty(lib.ulm_clip_grads_work_bytes(n), device=dev, dtype=torch.uint8)
    ptrs, counts, codes = array("Q", [t.data_ptr() for t in src]), array("q", [t.numel() for t in src]), _codes(src)
    optrs, ocodes = (ptrs, codes) if dst is src else (array("Q", [t.data_ptr() for t in dst]), _codes(dst)) if dst else (None, None)
    addr = lambda a: None if a is None else a.buffer_info()[0]  # noqa: E731
    with L.on(dev):
        L.check(lib.ulm_clip_grads(addr(ptrs), addr(optrs), addr(counts), addr(codes), addr(ocodes), n, max_norm,
                                   norm.data_ptr(), work.data_ptr(), L.stream(norm.device)))
    if dst is not None:
        for o, d in zip(outs, dst):
            if d is not o:
                o.copy_(d)
        torch.autograd.graph.increment_version(outs)
    return norm


def grad_norm(grads):
    """The 2-norm over all tensors of `grads` (fp32 or bf16, one GPU), a 0-d fp32 tensor."""
    grads = [g for g in grads if g is not None]
    if not grads:
        return torch.tensor(0.0)
    with torch.no_grad():
        return _run(grads, None, 0.0)


def clip_grads(grads, max_norm, out=None):
    """Scales `grads` (fp32 or bf16 tensors of one GPU) to a 2-norm of at most `max_norm`, in place, or
    into the tensors `out` of the same shapes (fp32 or bf16 each). Returns the norm that they had, a 0-d
    fp32 tensor. A tensor may stand in the list once: one that is there twice, or overlaps another, is
    refused, before anything is written."""
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    grads = list(grads)
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"{len(grads)} gradients and {len(outs)} outputs")
    for g, o in zip(grads, outs) if outs is not grads else ():
        if o.shape != g.shape or o.get_device() != g.get_device():
            raise ValueError(f"output {tuple(o.shape)} on {o.device} for a gradient {tuple(g.shape)} on {g.device}")
    if not grads:
        return torch.tensor(0.0)
    with torch.no_grad():
        return _run(grads, outs, max_norm)


def clip_grad_norm_(parameters, max_norm):
    """Clips the gradients of `parameters` (a tensor or an iterable of them; those without a gradient are
    passed over) in place. Returns the norm that they had."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_grads([p.grad for p in parameters if p.grad is not None], max_norm)
