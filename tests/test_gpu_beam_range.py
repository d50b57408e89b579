"""beam_select over the whole range of finite logits, against a float64 form that keeps log sum exp apart from the maximum:
(x - max) - log sum exp(x - max) + score. Formed as x - (max + log sum exp) the logarithm is lost from 1e16 on.

Scores: the bound of test_gpu_beam, 5e-6 and half a step of fp32; one below fp32's lowest value (a logit of -2.9e38 beside
one of 2.9e38 has -5.8e38, and half a step beyond -3.4028235e38 begins what rounds to -inf) is -inf, of its own beam and token.
No two beams' candidates lie within 1e-6 of each other but those that are equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = math.inf


def _want(logits, scores, k):
    """(scores float64, beams, tokens) [batch, k]."""
    batch, n, vocab = logits.shape
    out = torch.full((batch, k), -INF, dtype=torch.float64)
    frm, token = torch.zeros((batch, k), dtype=torch.int32), torch.zeros((batch, k), dtype=torch.int32)
    for b in range(batch):
        offers = []
        for j in range(n):
            x = logits[b, j].double()
            if x.max() == -INF:
                continue
            x = x - x.max()
            c = x - x.exp().sum().log() + scores[b, j].double()
            order = torch.argsort(c, descending=True, stable=True)[:k]
            offers += [(float(c[v]), j, int(v)) for v in order]
        offers = sorted((o for o in offers if o[0] > -INF), key=lambda o: (-o[0], o[1], o[2]))[:k]
        for i, (c, j, v) in enumerate(offers):
            out[b, i], frm[b, i], token[b, i] = c, j, v
    return out, frm, token


def _select(te, dev, logits, scores, k):
    got = [t.cpu() for t in te.beam_select(logits.to(dev), scores.to(dev), k)]
    want = _want(logits, scores, k)
    some = want[0].float() > -INF
    assert torch.equal(got[0] > -INF, some) and got[0].lt(INF).all()
    off = (got[0].double() - want[0]).abs() - 2.0 ** -24 * want[0].abs()
    assert not some.any() or float(off[some].max()) < 5e-6
    assert torch.equal(got[1], want[1]), "beams"
    assert torch.equal(got[2], want[2]), "tokens"


@pytest.mark.parametrize("k", [1, 5, 40, 64])
@pytest.mark.parametrize("vocab", [1, 9, 50, 3001, 40000])
@pytest.mark.parametrize("dtype,sizes", [(F32, (1e10, 1e17, 1e30, 2.9e38)), (BF16, (1e10, 1e17, 1e30, 2.9e38)), (F16, (6e4,))])
def test_equal_logits_of_any_size(te, gpu_device, dtype, sizes, vocab, k):
    """Each of n equal logits has score - log(n), whatever their size and sign; smaller ones beside them nothing."""
    scores = torch.tensor([[-1.5, -0.25], [-3.0, -9.0]])
    for size in sizes:
        for sign in (1.0, -1.0):
            x = torch.full((2, 2, vocab), sign * size)
            x[1, :, 1::2] = -size
            x[1, 1, ::3] = -INF
            _select(te, gpu_device, x.to(dtype), scores, k)
    # beams of different sizes
    x = torch.stack([torch.full((vocab,), float(s)) for s in (sizes[-1], -sizes[-1], 0.0, sizes[0])])[None]
    _select(te, gpu_device, x.to(dtype), torch.tensor([[-4.0, -1.0, -3.5, -0.75]]), k)


@pytest.mark.parametrize("k", [1, 5, 64])
@pytest.mark.parametrize("vocab", [1, 50, 3001, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_beams_of_the_lowest_value(te, gpu_device, dtype, vocab, k):
    """A mask of the type's lowest value: on a whole beam beside an ordinary one, ahead of it and behind it; on all beams; mixed
    with -inf; in all of a row but one token, far from it."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(vocab + k)
    scores = torch.tensor([[-20.0, -0.25, -30.0], [-1.0, -2.0, -25.0]])
    x = torch.randn((2, 3, vocab), generator=g) * 3
    x = x.to(dtype)
    x[0, 1] = low
    x[1, 2] = low
    _select(te, gpu_device, x, scores, k)
    _select(te, gpu_device, torch.full_like(x, low), scores, k)
    _select(te, gpu_device, torch.full_like(x, low), torch.zeros((2, 3)), k)
    x = torch.full_like(x, low)
    x[0, :, ::2] = -INF
    x[1, 0], x[1, 1, vocab // 2:], x[1, 2, : vocab // 2] = -INF, -INF, -INF
    _select(te, gpu_device, x, scores, k)
    x = torch.full_like(x, low)
    x[0, 0, vocab - 1], x[0, 1, vocab // 2], x[1, 1, 0], x[1, 2, -1] = 0.0, low / 2, torch.finfo(dtype).max, -1.5
    _select(te, gpu_device, x, scores, k)
