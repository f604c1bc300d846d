"""The head's work buffers are sized where the launch happens: the library sizes them by the SMs of the
current device, which is the operands' own only inside `_lib.on`. A fake library stands in for the GPU."""
import contextlib

import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.logprobs import lm_head_logprobs_bwd_raw, lm_head_logprobs_fwd_raw


class Lib:
    def __init__(self):
        self.inside, self.seen = False, []

    def __getattr__(self, name):
        def call(*args):
            self.seen.append((name, self.inside))
            return 64 if name.endswith("work_bytes") else L.ULM_OK
        return call


@pytest.mark.parametrize("backward", [False, True])
def test_work_buffer_is_sized_on_the_operands_device(monkeypatch, backward):
    lib = Lib()

    @contextlib.contextmanager
    def on(device):
        lib.inside = True
        yield
        lib.inside = False

    monkeypatch.setattr(L, "lib", lambda: lib)
    monkeypatch.setattr(L, "on", on)
    monkeypatch.setattr(L, "stream", lambda device: 0)
    h, w, t = torch.randn(3, 8).bfloat16(), torch.randn(5, 8).bfloat16(), torch.zeros(3, dtype=torch.long)
    if backward:
        lm_head_logprobs_bwd_raw(None, torch.ones(3), h, w, t, torch.zeros(3, 2), torch.zeros(3), L.ULM_PREC_BF16, True, True)
    else:
        lm_head_logprobs_fwd_raw(h, w, t, 2, L.ULM_PREC_BF16)
    assert len(lib.seen) == 2 and all(inside for _, inside in lib.seen)
