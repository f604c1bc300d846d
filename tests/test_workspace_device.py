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


def test_work_buffer_holds_what_the_backward_writes():
    """Two bf16 parts of the logits' gradient, and partial sums only where a product is split; in fp32
    precision the gradient, its three parts, the operands' parts and 64 MB for sums."""
    size = L.lib().ulm_lm_head_logprobs_work_bytes
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    for N, V, D in ((1, 64, 32), (256, 512, 1024), (300, 505, 200)):
        ldv, ldd = (V + 7) // 8 * 8, (D + 7) // 8 * 8
        assert size(N, V, D, 0, 1, L.ULM_PREC_BF16) == up(N * ldv * 4)
        f32 = size(N, V, D, 0, 1, L.ULM_PREC_FP32)
        least = up(N * ldv * 4) + up(N * ldv * 6) + up(N * ldd * 6) + up(V * ldd * 6)
        assert least <= f32 <= least + (64 << 20)
    N, V, D = 8192, 32000, 768  # dh in three ranges of the vocabulary, dW whole
    assert size(N, V, D, 0, 1, L.ULM_PREC_BF16) == N * V * 4 + 3 * N * D * 4
