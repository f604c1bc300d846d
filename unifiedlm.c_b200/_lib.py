"""ctypes binding of the C ABI in include/ulm_b200.h (libulm_b200.so, built in-tree).

There is no fallback: if the library is missing or a call fails, the caller gets an exception.
"""
import ctypes
import os

import torch
from torch.autograd import forward_ad

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libulm_b200.so")

ULM_OK, ULM_ERR_INVALID, ULM_ERR_CUDA, ULM_ERR_UNSUPPORTED, ULM_ERR_DEVICE = range(5)
ULM_F32, ULM_BF16 = 0, 1
ULM_PREC_BF16, ULM_PREC_FP32 = 0, 1

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_I = ctypes.c_int

# name -> (restype, argtypes); kept in the order of include/ulm_b200.h
SIGNATURES = {
    "ulm_last_error": (ctypes.c_char_p, []),
    "ulm_version": (_I, []),
    "ulm_device_error": (_I, [ctypes.POINTER(_I)]),
    "ulm_memory_stats_fwd": (_I, [_P, _P, _P, _P, _P, _P, _P, _I, _I64, _I64, _I64, _I64, _P]),
    "ulm_memory_stats_bwd": (_I, [_P] * 12 + [_I64, _I64, _I64, _P]),
    "ulm_memory_stats_bwd_scratch": (_I64, [_I64, _I64, _I64]),
    "ulm_memory_stats_bwd_noalloc": (_I, [_P] * 11 + [_I64, _I64, _I64, _P]),
    "ulm_memory_needs_c": (_I, [_I64, _I64]),
    "ulm_block_scalars_fwd": (_I, [_P] * 6 + [_I64, _P]),
    "ulm_block_scalars_bwd": (_I, [_P] * 11 + [_I64, _P]),
    "ulm_decayed_scores": (_I, [_P, _I64, _P, _I64, _P, _I64, _P, _I64, _I64, _I64, _I, _P]),
    "ulm_causal_apply": (_I, [_P, _I64, _P, _I64, _P, _I64, _I, _I, _I64, _I64, _I64, _I, _P]),
    "ulm_operand_ld": (_I64, [_I64]),
    "ulm_set_gemm_pairs": (_I, [_I]),
    "ulm_set_epilogue_mode": (_I, [_I]),
    "ulm_set_scan_mode": (_I, [_I]),
    "ulm_set_pdl": (_I, [_I]),
    "ulm_set_chunk_mode": (_I, [_I]),
    "ulm_memory_chunk_len": (_I, [_I64, _I64, _I64, _I]),
    "ulm_memory_saved_bytes": (_I64, [_I64, _I64, _I64, _I64, _I]),
    "ulm_memory_bwd_work_bytes": (_I64, [_I64, _I64, _I64, _I64, _I]),
    "ulm_memory_fwd": (_I, [_P, _P, _P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I, _P]),
    "ulm_memory_bwd": (_I, [_P, _P, _I] + [_P] * 19 + [_I64, _I64, _I64, _I64, _I, _P]),
    "ulm_memory_combine_fwd": (_I, [_P, _P, _P, _I, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _P, _P, _P,
                                    _I64, _I64, _I64, _I64, _I, _P]),
    "ulm_memory_combine_bwd": (_I, [_P, _I] + [_P] * 20 + [_I, _P, _P, _P, _I64, _I64, _I64, _I64, _I, _P]),
    "ulm_combine_grad_scratch": (_I64, [_I64, _I64, _I64, _I64]),
    "ulm_address_fwd": (_I, [_P, _I, _P, _I64, _P, _I64, _P, _P, _P, _P, _I, _P, _P, _I64, _I64, _I64, _I64, _I64,
                             _I, _P]),
    "ulm_address_fwd_work_bytes": (_I64, [_I64, _I64, _I64]),
    "ulm_address_bwd": (_I, [_P, _P, _P, _I, _P, _I64, _P, _I, _P, _I64, _P, _I64, _P, _P, _P, _P, _P, _P,
                             _I64, _I64, _I64, _I64, _I, _P]),
    "ulm_address_bwd_work_bytes": (_I64, [_I64, _I64, _I64, _I64, _I]),
    "ulm_addressed_memory_bwd": (_I, [_P, _P, _I] + [_P] * 19 + [_P, _I64, _P, _I, _P, _I64, _P, _I64] + [_P] * 6 +
                                 [_I64] * 4 + [_I, _P]),
    "ulm_mixer_bwd": (_I, [_P, _I] + [_P] * 20 + [_I, _P, _P, _P] + [_P, _I64, _P, _I, _P, _I64, _P, _I64] +
                      [_P] * 6 + [_I64] * 4 + [_I, _P]),
    "ulm_rms_norm_fwd": (_I, [_P, _I, _P, _P, _I, _P, _I64, _I64, ctypes.c_float, _P]),
    "ulm_rms_norm_bwd": (_I, [_P, _I, _P, _I, _P, _P, _P, _P, _P, _P, _I64, _I64, _P]),
    "ulm_rms_norm_bwd_work_bytes": (_I64, [_I64, _I64]),
    "ulm_linear_fwd": (_I, [_P, _I, _P, _P, _P, _P, _I, _I64, _I64, _I64, _I, _P]),
    "ulm_linear_bwd": (_I, [_P, _I, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I, _P]),
    "ulm_linear_bwd_work_bytes": (_I64, [_I64, _I64, _I64, _I]),
    "ulm_lm_head_loss_fwd": (_I, [_P, _I64, _P, _I64, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I, _P]),
    "ulm_lm_head_loss_bwd": (_I, [_P, _P, _P, _I64, _P, _I64, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I, _P]),
    "ulm_lm_head_work_bytes": (_I64, [_I64, _I64, _I64, _I]),
    "ulm_decode_prepare_block": (_I, [_P, _P, _P, _P, _I, _I64, _I64, _P]),
    "ulm_decode_reset_block": (_I, [_P] * 6 + [_I64] * 4 + [_P]),
    "ulm_decode_block_step": (_I, [_P] * 7 + [_I] + [_P] * 8 + [_I64] * 4 + [ctypes.c_float, _P]),
    "ulm_decode_block_work_bytes": (_I64, [_I64, _I64, _I64]),
    "ulm_decode_embed": (_I, [_P, _P, _I, _P, _I64, _I64, _P]),
    "ulm_decode_head": (_I, [_P, _P, _P, _P, _I, _P, _P, _P, _I64, _I64, _I64, ctypes.c_float, _P]),
    "ulm_decode_sample": (_I, [_P, _I64, _I64, ctypes.c_float, ctypes.c_float, _P, _P, _P, _I, _P, _I64, _P]),
    "ulm_decode_head_work_bytes": (_I64, [_I64, _I64]),
    "ulm_decode_prefill_block": (_I, [_P] * 7 + [_I] + [_P] * 7 + [_I64] * 5 + [_I, _P]),
    "ulm_decode_prefill_work_bytes": (_I64, [_I64, _I64, _I64, _I]),
    "ulm_token_logprobs_fwd": (_I, [_P, _I, _I64] + [_P] * 6 + [_I64, _I64, _I, _P]),
    "ulm_token_logprobs_bwd": (_I, [_P, _P, _P, _I, _I64, _P, _P, _P, _P, _I64, _I64, _I64, _P]),
    "ulm_lm_head_logprobs_fwd": (_I, [_P, _I64, _P, _I64] + [_P] * 7 + [_I64, _I64, _I64, _I, _I, _P]),
    "ulm_lm_head_logprobs_bwd": (_I, [_P, _P, _P, _I64, _P, _I64, _P, _P, _P, _P, _I, _P, _I, _P,
                                      _I64, _I64, _I64, _I, _P]),
    "ulm_lm_head_logprobs_work_bytes": (_I64, [_I64, _I64, _I64, _I, _I, _I]),
    "ulm_embedding_fwd": (_I, [_P, _P, _I, _I64, _P, _I, _I64, _I64, _I64, ctypes.c_float, _P]),
    "ulm_embedding_bwd": (_I, [_P, _P, _I, _P, _I, _P, _I64, _I64, _I64, ctypes.c_float, _P]),
    "ulm_embedding_bwd_work_bytes": (_I64, [_I64, _I64, _I64]),
    "ulm_clip_grads": (_I, [_P, _P, _P, _P, _P, _I64, ctypes.c_float, _P, _P, _P]),
    "ulm_clip_grads_work_bytes": (_I64, [_I64]),
}

_lib = None


def lib():
    """The loaded library with argument types declared. Raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; "
                               f"g.build()'` (nvcc, sm_100a)")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


class UlmError(RuntimeError):
    pass


def check(rc):
    if rc != ULM_OK:
        msg = lib().ulm_last_error().decode(errors="replace")
        raise UlmError(f"libulm_b200 status {rc}: {msg}")


def ptr(t):
    """Device (or host) address of a tensor, or NULL for None."""
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_of(t):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def dtype_code(dtype):
    if dtype == torch.float32:
        return ULM_F32
    if dtype == torch.bfloat16:
        return ULM_BF16
    raise UlmError(f"unsupported element type {dtype}")


def device_error():
    """Synchronise and read/clear the device-side error flag (0 = none)."""
    site = _I(0)
    check(lib().ulm_device_error(ctypes.byref(site)))
    return site.value


_PLAIN = (torch.Tensor, torch.nn.Parameter)


_C = torch._C
_PRE_DISPATCH = _C.DispatchKey.PreDispatch


def _observed():
    """Whether something looks on at the dispatcher's calls or transforms them: a dispatch mode (make_fx, a
    FLOP counter, selective checkpointing), torch.jit.trace, a torch.func transform, an open level of
    forward-mode differentiation."""
    return (_C._len_torch_dispatch_stack() > 0 or _C._get_tracing_state() is not None or
            _C._are_functorch_transforms_active() or forward_ad._current_level >= 0 or
            _C._dispatch_tls_is_dispatch_key_included(_PRE_DISPATCH))


def eager(*ts):
    """Whether the tensors hold data that a call can read now and nobody else is to see the call (nothing is
    traced, compiled, faked, transformed or observed): the entries then call the library directly, without
    the dispatcher's cost of a custom op."""
    if torch.compiler.is_compiling() or _observed():
        return False
    for t in ts:
        if type(t) not in _PLAIN:
            return False
    return True


def no_tangents(name, *ts):
    """Refuses inputs that carry a tangent (forward-mode differentiation), which the call would drop."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError(f"{name} has no forward-mode derivative")


_PROXY = _C._TorchDispatchModeKey.PROXY


def not_traced(name, ts):
    """Refuses a call that is no op of the dispatcher where something would record it, or transform its
    inputs: the record would lack it."""
    if not _observed():
        return
    if (_C._get_tracing_state() is not None or _C._get_dispatch_mode(_PROXY) is not None or
            _C._dispatch_tls_is_dispatch_key_included(_PRE_DISPATCH) or _C._are_functorch_transforms_active()):
        raise RuntimeError(f"{name} cannot be traced or transformed")
    no_tangents(name, *ts)


def first_order(name):
    """Called in a backward: refuses the one that is to be differentiated again (create_graph)."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{name} has no second derivative (create_graph)")


def stream(device):
    """The current stream of a device as a plain address (`stream_of` without its wrapper objects)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


class _Here:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on(device):
    """`torch.cuda.device(device)`, or nothing where it is the current one already."""
    return _HERE if _C._cuda_getDevice() == device.index else torch.cuda.device(device)
