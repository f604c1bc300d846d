"""Calls from a thread that has done nothing on the GPU yet and whose buffers all come from the
allocator's cache, as in autograd's own threads: no CUDA context is current there."""
import threading

import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.kernel import unified_memory
from unifiedlm_c_b200.logprobs import lm_head_logprobs, lm_head_logprobs_bwd_raw, lm_head_logprobs_fwd_raw
from unifiedlm_c_b200.norm import linear

pytestmark = pytest.mark.gpu


def in_a_new_thread(f):
    got = []

    def run():
        try:
            got.append(f())
        except Exception as e:
            got.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


def cases():
    gen = torch.Generator().manual_seed(0)
    h = torch.randn(300, 128, generator=gen).cuda().bfloat16()
    w = torch.randn(1000, 128, generator=gen).cuda().bfloat16()
    t = torch.randint(0, 1000, (300,), generator=gen).cuda()
    a = torch.randn(300, generator=gen).cuda()
    _, ent, stats, _, _ = lm_head_logprobs_fwd_raw(h, w, t, 0, L.ULM_PREC_BF16)
    r = torch.rand(2, 64, 96, generator=gen).cuda()
    v = torch.randn(2, 64, 128, generator=gen).cuda().bfloat16()
    g, ww = torch.tensor(-0.1).cuda(), torch.rand(96, generator=gen).cuda() + 0.5
    return [lambda: lm_head_logprobs(h, w, t, top_k=3),
            lambda: lm_head_logprobs_bwd_raw(a, a, h, w, t, stats, ent, L.ULM_PREC_BF16, True, True),
            lambda: (linear(h, w, "bf16"),),
            lambda: unified_memory(r, v, g, ww)]


@pytest.mark.parametrize("i", range(4))
def test_first_call_of_a_thread(i):
    f = cases()[i]
    want = [o.clone() for o in f()]
    f()  # its buffers go back to the cache
    torch.cuda.synchronize()
    got = in_a_new_thread(f)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert L.device_error() == 0


def test_first_backward_of_a_process():
    """The same where it was met: in autograd's thread, which a child process has not used before."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from __graft_entry__ import load_package
load_package()
from unifiedlm_c_b200.logprobs import lm_head_logprobs
big = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
h = torch.randn(300, 128, device="cuda").bfloat16().requires_grad_()
w = torch.randn(1000, 128, device="cuda").bfloat16().requires_grad_()
del big  # blocks for all that follows
r = lm_head_logprobs(h, w, torch.arange(300, device="cuda"))
dh, dw = torch.autograd.grad([r.logprobs], [h, w], [torch.ones(300, device="cuda")])
print(float(dh.float().norm()), bool(dw.isfinite().all()))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split()[1] == "True", r.stderr[-2000:]
