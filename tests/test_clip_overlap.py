"""Which strided tensors clipping takes for overlapping (`clip._apart`, `clip._folded`), against the sets
of their bytes. No GPU: addresses only."""
import itertools
import random

import pytest
import torch

import unifiedlm_c_b200._lib as L
from unifiedlm_c_b200.clip import _apart, _check_strided, _folded


def bytes_of(t):
    es = t.element_size()
    at = {t.data_ptr()}
    for n, s in zip(t.shape, t.stride()):
        at = {a + i * s * es for a in at for i in range(n)}
    return {a + b for a in at for b in range(es)}


def views(a):
    return [a, a.t(), a[:, :5], a[:, 5:], a[1:, :5], a[:-1, 5:], a[::2], a[1::2], a[:, ::2], a[:, 1::2], a[3], a[:, 3], a[2:4],
            a[::2, :4], a[1::2, 2:], a.view(-1)[7:31], a.view(-1)[::3], a.view(2, 4, 12)[:, 1], a.view(2, 4, 12).transpose(0, 2)[3:5],
            a.view(torch.bfloat16)[:, :7], a.view(torch.bfloat16)[:, 10:], a[:, :1], a[-1:, -1:]]


def test_apart_is_never_wrong_and_knows_slices():
    a = torch.zeros(8, 12)
    known = 0
    for x, y in itertools.product(views(a), repeat=2):
        apart = not (bytes_of(x) & bytes_of(y))
        got = _apart(x, y)
        assert not got or apart, (x.shape, x.stride(), y.shape, y.stride())
        known += got == apart
    assert known >= 0.9 * len(views(a)) ** 2
    for x, y in ((a[:, :5], a[:, 5:]), (a[1:, :5], a[:-1, 5:]), (a[:, ::2], a[:, 1::2]), (a[::2], a[1::2]), (a[:, 3], a[:, 4]),
                 (a.t()[:5], a.t()[5:]), (a[:, :5], torch.zeros(8, 12)[:, :5])):
        assert _apart(x, y) and _apart(y, x)


def test_apart_of_random_slices():
    rng = random.Random(0)
    a = torch.zeros(6, 7, 9)

    def one():
        v = a
        for d in range(3):
            lo = rng.randrange(v.shape[d])
            v = v[(slice(None),) * d + (slice(lo, rng.randrange(lo, v.shape[d]) + 1, rng.choice([1, 1, 2, 3])),)]
        return v.permute(*rng.sample(range(3), 3))

    told = 0
    for _ in range(2000):
        x, y = one(), one()
        apart = not (bytes_of(x) & bytes_of(y))
        got = _apart(x, y)
        assert not got or apart
        told += got and apart
    assert told > 200


def test_folded():
    a = torch.zeros(8, 12)
    assert not any(_folded(v) for v in views(a))
    assert _folded(torch.zeros(6).expand(3, 6)) and _folded(torch.zeros(20).as_strided((4, 6), (3, 1)))
    assert not _folded(torch.zeros(6).expand(1, 6)) and not _folded(torch.zeros(()))


def test_lists():
    a, b = torch.zeros(8, 12), torch.zeros(8, 12)
    q, k, v = a[:, :4], a[:, 4:8], a[:, 8:]
    for grads, outs in (([q, k, v], None), ([a.t(), b], None), ([q, k], [b[:, :4], b[:, 4:8]]), ([q, q], [b[:, :4], b[:, 4:8]]),
                        ([a.t()], [a.t()]), ([q, a[:0]], None)):
        _check_strided(grads, grads if outs is None else outs)
    for grads, outs in (([a, a.t()], None), ([a.t(), a.t()], None), ([q, a[:, 3:8]], None), ([q, a[0]], None),
                        ([q, k], [b[:, :4]] * 2), ([q, k], [k, q]), ([a.t(), b], [b.t(), a])):
        with pytest.raises(L.UlmError, match="overlap"):
            _check_strided(grads, grads if outs is None else outs)
    with pytest.raises(ValueError, match="share memory"):
        _check_strided([a, torch.zeros(6).expand(3, 6)], [a, torch.zeros(6).expand(3, 6)])


def test_expanded_gradients_into_other_tensors():
    """An input may be expanded: only its bytes count."""
    a = torch.zeros(8, 12)
    row = a[:1, :4].expand(8, 4)
    _check_strided([row, a[:, 4:8]], [torch.zeros(8, 4), torch.zeros(8, 4)])
    _check_strided([row, a[:, 4:8]], [torch.zeros(8, 4), a[:, 8:]])
    with pytest.raises(L.UlmError, match="overlap"):
        _check_strided([row, a[:, 4:8]], [torch.zeros(8, 4), a[:, :4]])


def test_apart_of_expanded_rows():
    a = torch.zeros(8, 12)
    x, y = a[:1, :4].expand(8, 4), a[:1, 3:7].expand(8, 4)
    assert not _apart(x, y) and _apart(x, a[:1, 4:8].expand(8, 4))
