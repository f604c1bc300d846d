"""Refusals of the log-probability, embedding and clipping entries without a GPU: CPU tensors, and the
C ABI's checks, which come before any device work."""
import ctypes

import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.clip import clip_grad_norm_, clip_grads, grad_norm
from unifiedlm_c_b200.dp import GradBucket
from unifiedlm_c_b200.embed import embedding
from unifiedlm_c_b200.logprobs import lm_head_logprobs, token_logprobs

P = ctypes.c_void_p(256)


def refused(rc, word):
    assert rc == L.ULM_ERR_INVALID and word in L.lib().ulm_last_error().decode(), (rc, L.lib().ulm_last_error())


def test_cpu_tensors_are_refused():
    t, x = torch.zeros(2, dtype=torch.long), torch.randn(2, 4)
    for call in (lambda: lm_head_logprobs(x, x, t), lambda: token_logprobs(x, t), lambda: embedding(t, x),
                 lambda: clip_grads([x], 1.0), lambda: grad_norm([x]), lambda: GradBucket([(2, 4)], "cpu").clip_norm_(1.0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(grad_norm([None])) == 0.0


def test_token_logprobs_arguments():
    f = L.lib().ulm_token_logprobs_fwd

    def call(x=P, dt=0, ld=8, t=P, lp=P, ids=P, N=2, V=8, k=3):
        return f(x, dt, ld, t, lp, P, P, ids, P, N, V, k, None)

    refused(call(dt=7), "dtype")
    refused(call(ld=7), "stride")
    refused(call(k=33, V=100, ld=100), "top_k")
    refused(call(k=9), "top_k")
    refused(call(k=-1), "top_k")
    refused(call(ids=None), "top_k")
    refused(call(t=None), "null")
    refused(call(x=None), "null")
    refused(call(lp=None), "null")
    refused(call(V=0), "extent")
    refused(call(N=-1), "extent")
    refused(call(N=1 << 31), "extent")
    assert call(N=0, x=None, t=None) == L.ULM_OK
    refused(L.lib().ulm_token_logprobs_bwd(P, P, P, 0, 8, P, P, P, P, 7, 2, 8, None), "stride")
    refused(L.lib().ulm_token_logprobs_bwd(P, P, P, 0, 8, P, None, P, P, 8, 2, 8, None), "null")


def test_head_logprobs_arguments():
    lib = L.lib()

    def fwd(h=P, ld_h=16, ld_w=16, work=P, N=2, V=8, D=16, k=3, prec=0):
        return lib.ulm_lm_head_logprobs_fwd(h, ld_h, P, ld_w, P, P, P, P, P, P, work, N, V, D, k, prec, None)

    refused(fwd(prec=3), "prec")
    refused(fwd(ld_h=15), "stride")
    refused(fwd(ld_w=15), "stride")
    refused(fwd(work=None), "null")
    refused(fwd(work=ctypes.c_void_p(264)), "aligned")
    refused(fwd(h=None), "null")
    refused(fwd(D=0), "extent")
    refused(fwd(k=9), "top_k")
    assert fwd(N=0) == L.ULM_OK
    bwd = lib.ulm_lm_head_logprobs_bwd
    refused(bwd(P, P, P, 16, P, 16, P, P, P, P, 5, P, 0, P, 2, 8, 16, 0, None), "dtype")
    refused(bwd(P, P, P, 16, P, 16, P, None, P, P, 0, P, 0, P, 2, 8, 16, 0, None), "null")
    assert bwd(P, P, P, 16, P, 16, P, P, P, None, 0, None, 0, P, 2, 8, 16, 0, None) == L.ULM_OK  # nothing wanted
    assert lib.ulm_lm_head_logprobs_work_bytes(-1, 8, 16, 0, 0, 0) == -1
    for n, v in ((1, 1), (7, 32000), (16384, 32000)):
        assert 0 < lib.ulm_lm_head_logprobs_work_bytes(n, v, 64, 0, 0, 0) < lib.ulm_lm_head_logprobs_work_bytes(n, v, 64, 32, 0, 0)


def test_embedding_arguments():
    lib = L.lib()

    def fwd(t=P, w=P, wd=0, ld=8, yd=0, N=2, V=4, D=8):
        return lib.ulm_embedding_fwd(t, w, wd, ld, P, yd, N, V, D, 1.0, None)

    refused(fwd(wd=4), "dtype")
    refused(fwd(yd=4), "dtype")
    refused(fwd(ld=7), "stride")
    refused(fwd(t=None), "null")
    refused(fwd(w=None), "null")
    refused(fwd(V=0), "extent")
    refused(fwd(N=1 << 31), "extent")
    assert fwd(N=0) == L.ULM_OK
    refused(lib.ulm_embedding_bwd(P, P, 4, P, 0, P, 2, 4, 8, 1.0, None), "dtype")
    refused(lib.ulm_embedding_bwd(P, P, 0, None, 0, P, 2, 4, 8, 1.0, None), "null")
    refused(lib.ulm_embedding_bwd(P, P, 0, P, 0, None, 2, 4, 8, 1.0, None), "null")
    refused(lib.ulm_embedding_bwd(P, P, 0, P, 0, ctypes.c_void_p(264), 2, 4, 8, 1.0, None), "aligned")
    assert lib.ulm_embedding_bwd_work_bytes(1, -1, 8) == -1


def test_clip_arguments():
    lib = L.lib()

    def call(ptrs, outs=None, counts=None, dts=None, odts=None, max_norm=1.0, norm=P, work=P):
        n = len(ptrs)
        vp, i64, i32 = ctypes.c_void_p * n, ctypes.c_int64 * n, ctypes.c_int * n
        return lib.ulm_clip_grads(vp(*ptrs), vp(*outs) if outs else None, i64(*(counts or [10] * n)), i32(*(dts or [0] * n)),
                                  i32(*(odts or [0] * n)) if outs else None, n, max_norm, norm, work, None)

    refused(call([4096], [4096], max_norm=-1.0), "max_norm")
    refused(call([4096], [4096], max_norm=float("nan")), "max_norm")
    refused(call([4096], [4096], dts=[9]), "dtype")
    refused(call([4096], [4096], odts=[9]), "dtype")
    refused(call([4096], [None]), "null")
    refused(call([None], [4096]), "null")
    refused(call([4096], [4096], counts=[-1]), "count")
    refused(call([4096], [4096], norm=None), "null")
    refused(call([4096], [4096], work=None), "null")
    refused(call([4096], [4096], work=ctypes.c_void_p(260)), "aligned")
    refused(call([4096, 4096], [4096, 4096]), "overlap")           # the same tensor twice
    refused(call([4096, 4100], [4096, 4100]), "overlap")           # a view of another one
    refused(call([4096, 8192], [8192, 4096]), "overlap")           # swapped
    refused(call([4096], [4096], odts=[1]), "overlap")             # in place, but another type
    refused(call([4096], [4116]), "overlap")
    assert lib.ulm_clip_grads_work_bytes(-1) == -1 and lib.ulm_clip_grads_work_bytes(0) > 0
