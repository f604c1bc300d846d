"""Clipping lists with strided tensors: slices of one parent are clipped as any others, overlaps are
refused before anything is written."""
import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.clip import clip_grads

pytestmark = pytest.mark.gpu


def test_slices_of_one_parent():
    gen = torch.Generator().manual_seed(0)
    qkv = torch.randn(40, 96, generator=gen).cuda()
    other = torch.randn(7, 5, generator=gen).cuda()
    before, o = qkv.clone(), other.clone()
    n = torch.cat([qkv.reshape(-1), other.reshape(-1)]).double().norm()
    got = clip_grads([qkv[:, :32], qkv[:, 32:64], qkv[:, 64:], other.t()], 1.0)
    assert abs(float(got) - float(n)) <= 4 * 2.0 ** -24 * float(n)
    f = 1.0 / (float(n) + 1e-6)
    for x, y in ((qkv, before), (other, o)):
        assert bool(((x.double() - y.double() * f).abs() <= y.double().abs() * f * 9 * 2.0 ** -24).all())


def test_overlaps_are_refused_before_anything_is_written():
    a = torch.randn(12, 12).cuda()
    b, keep = torch.randn(5).cuda(), a.clone()
    first = b.clone()
    for grads, out in (([b, a, a.t()], None), ([b, a.t(), a.t()], None), ([b, a[:, :7], a[:, 6:]], None),
                       ([a[:, :6], a[:, 6:]], [torch.zeros(12, 12).cuda()[:, :6]] * 2)):
        with pytest.raises(L.UlmError, match="overlap"):
            clip_grads(grads, 0.1, out=out)
    with pytest.raises(ValueError, match="share memory"):
        clip_grads([b, b.clone().expand(3, 5)], 0.1)
    with pytest.raises(ValueError, match="share memory"):
        clip_grads([b, a[:3, :5]], 0.1, out=[torch.zeros(5).cuda(), b.clone().expand(3, 5)])
    torch.cuda.synchronize()
    assert torch.equal(a, keep) and torch.equal(b, first)
