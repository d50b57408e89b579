"""beam_select against its float64 restatement (search_ref).

Beams and tokens have to be the restatement's; the inputs leave no two beams' candidates within 1e-6 of each other but those
that are equal. Scores: log sum exp is formed of fp32 exponentials (their arguments rounded twice, weighted with
themselves: 2^-24 of the sum each, and 2^-23 of the function) in runs of up to 64 additions (2^-24 each), joined in 64 bits:
less than 80 x 2^-24 = 5e-6, then one rounding to fp32."""
import math

import pytest
import torch

import search_ref as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")


def _select(te, dev, logits, scores, k, ended=None, end_token=0, on=None):
    """`on`: what the call is given in the place of logits.to(dev)."""
    got = te.beam_select(logits.to(dev) if on is None else on, scores.to(dev), k, ended=None if ended is None else ended.to(dev), end_token=end_token)
    want = ref.beams(logits, scores, k, ended, end_token)
    assert [t.dtype for t in got] == [F32, torch.int32, torch.int32] and all(t.shape == (logits.shape[0], k) for t in got)
    assert torch.equal(got[1].cpu(), want[1]), "beams"
    assert torch.equal(got[2].cpu(), want[2]), "tokens"
    s, w = got[0].double().cpu(), want[0]
    assert torch.equal(s == -INF, w == -INF)
    ok = w > -INF
    assert float(((s - w)[ok].abs() - 2.0 ** -24 * w[ok].abs()).max() if ok.any() else 0.0) < 5e-6
    return got


def _random(batch, beams, vocab, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((batch, beams, vocab), generator=g) * spread).to(dtype), -torch.rand((batch, beams), generator=g) * 20


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 63, 64, 65, 255, 257, 511, 1000, 1001, 2049, 5000, 16385, 49152])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_vocabularies(te, gpu_device, vocab, dtype):
    for batch, beams, k in ((1, 1, 1), (2, 3, 6), (1, 4, 64)):
        x, s = _random(batch, beams, vocab, dtype, vocab + k)
        _select(te, gpu_device, x, s, k)


@pytest.mark.parametrize("beams,k", [(1, 1), (1, 64), (2, 1), (5, 10), (16, 32), (63, 63), (64, 1), (64, 64)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_beams(te, gpu_device, beams, k, dtype):
    x, s = _random(3, beams, 4099, dtype, beams + k)
    ended = torch.rand((3, beams), generator=torch.Generator().manual_seed(k)) < 0.3
    _select(te, gpu_device, x, s, k)
    _select(te, gpu_device, x, s, k, ended, 4098)


def test_a_large_call(te, gpu_device):
    x, s = _random(3, 4, 151936, F16, 0)
    _select(te, gpu_device, x, s, 8)
    x, s = _random(150, 3, 1003, BF16, 1)
    _select(te, gpu_device, x, s, 6)


@pytest.mark.parametrize("k", [1, 5, 64])
@pytest.mark.parametrize("vocab", [50, 3001, 40000])
def test_equal_logits(te, gpu_device, vocab, k):
    """The lowest beams and tokens, where all are equal, in steps, and in two beams alike."""
    x = torch.zeros((2, 3, vocab))
    s = torch.tensor([[0.0, 0.0, 0.0], [-1.0, 0.0, -2.0]])
    for dtype in (F32, F16, BF16):
        _select(te, gpu_device, x.to(dtype), s, k)
        steps = (torch.arange(vocab) // 7 % 5).float().expand(2, 3, -1).contiguous()
        _select(te, gpu_device, steps.to(dtype), s, k)
        y, _ = _random(2, 1, vocab, dtype, k)
        _select(te, gpu_device, y.expand(-1, 3, -1).contiguous(), torch.zeros((2, 3)), k)
        signed = torch.where(torch.arange(vocab) % 2 == 0, -0.0, 0.0).expand(2, 3, -1).contiguous()
        _select(te, gpu_device, signed.to(dtype), s, k)


@pytest.mark.parametrize("vocab", [77, 5000, 60001])
def test_orders(te, gpu_device, vocab):
    """Ascending and descending logits, and the largest ones side by side: every token passes what came before it, the
    largest lie with one lane, one workgroup."""
    ramp = torch.linspace(-30, 30, vocab)
    near = torch.where((torch.arange(vocab) >= vocab // 2) & (torch.arange(vocab) < vocab // 2 + 70), ramp.abs() + 50, ramp)
    apart = torch.where(torch.arange(vocab) % 64 == 3, ramp + 100, ramp)
    for line in (ramp, ramp.flip(0), near, near.flip(0), apart):
        x = torch.stack([line, line.roll(11) - 1])[None]
        for dtype in (F32, F16):
            for k in (1, 9, 64):
                _select(te, gpu_device, x.to(dtype), torch.tensor([[-1.0, -0.6180339]]), k)


def test_banned_tokens(te, gpu_device):
    """Logits of -inf offer nothing, nor do NaN ones, wherever they lie; where fewer than k are left, the rest are none."""
    for vocab in (70, 3000):
        x, s = _random(4, 3, vocab, F32, vocab)
        x[0, :, ::2] = -INF
        x[1, 0], x[1, 2] = -INF, float("nan")
        x[2, :, 5:] = -INF
        x[2, 1, :3] = float("nan")
        x[3] = -INF
        for dtype in (F32, F16, BF16):
            got = _select(te, gpu_device, x.to(dtype), s, 40, end_token=2)
            assert (got[0][3] == -INF).all() and (got[1][3] == 0).all() and (got[2][3] == 2).all()


def test_beams_that_are_not_in_use(te, gpu_device):
    x, s = _random(3, 4, 500, F16, 3)
    s[0, 1:] = -INF
    s[1, 0], s[1, 3] = float("nan"), -INF
    s[2] = -INF
    _select(te, gpu_device, x, torch.where(s.isnan(), -INF, s), 6)
    got = te.beam_select(x.to(gpu_device), s.to(gpu_device), 6)
    want = te.beam_select(x.to(gpu_device), torch.where(s.isnan(), -INF, s).to(gpu_device), 6)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_ended_beams(te, gpu_device):
    """They offer themselves alone, their logits are not looked at; all of them; with fewer candidates than k."""
    x, s = _random(3, 4, 300, F32, 5)
    ended = torch.tensor([[False, True, False, True], [True] * 4, [True, False, False, False]])
    x[ended] = float("nan")
    s[2, 0] = -INF
    for k in (1, 4, 8, 64):
        got = _select(te, gpu_device, x, s, k, ended, 299)
        if k > 4:
            assert (got[0][1, 4:] == -INF).all()


def test_large_logits(te, gpu_device):
    for size in (1e4, 6e4, 1e30):
        x, s = _random(2, 2, 3000, F32, 7)
        _select(te, gpu_device, x * size, s, 4)
    x, s = _random(2, 2, 3000, F16, 8, spread=1e4)
    _select(te, gpu_device, x.clamp(-65504, 65504), s, 8)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_strides(te, gpu_device, dtype):
    """Rows an odd number of elements apart, beams before the batch, every other token, one row for all beams."""
    x, s = _random(3, 4, 1003, dtype, 9)
    wide = torch.zeros((3, 4, 1007), dtype=dtype, device=gpu_device)
    wide[..., 3:1006] = x.to(gpu_device)
    _select(te, gpu_device, x, s, 9, on=wide[..., 3:1006])
    turned = x.transpose(0, 1).contiguous().to(gpu_device).transpose(0, 1)
    _select(te, gpu_device, x, s, 9, on=turned)
    twice = torch.zeros((3, 4, 2006), dtype=dtype, device=gpu_device)
    twice[..., ::2] = x.to(gpu_device)
    _select(te, gpu_device, x, s, 9, on=twice[..., ::2])
    one = x[:, :1].expand(-1, 4, -1)
    _select(te, gpu_device, one.contiguous(), s, 9, on=x[:, :1].to(gpu_device).expand(-1, 4, -1))


def test_repeats_graphs_and_streams(te, gpu_device):
    """The same call twice is bit-identical; every replay of a captured call, with eager calls between, equals an eager
    one; so does a call on another stream."""
    x, s = (t.to(gpu_device) for t in _random(4, 3, 20011, F16, 10))
    eager = te.beam_select(x, s, 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = te.beam_select(x, s, 7)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = te.beam_select(x, s, 7)
    for i in range(4):
        fresh = [t.to(gpu_device) for t in _random(4, 3, 20011, F16, 20 + i)]
        x.copy_(fresh[0])
        s.copy_(fresh[1])
        graph.replay()
        want = te.beam_select(*fresh, 7)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_workspace_of_the_caller(te, gpu_device):
    x, s = (t.to(gpu_device) for t in _random(2, 3, 5000, F32, 11))
    ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device=gpu_device)
    assert all(torch.equal(a, b) for a, b in zip(te.beam_select(x, s, 5, workspace=ws), te.beam_select(x, s, 5)))
    with pytest.raises(te.TrellisError) as e:
        te.beam_select(x, s, 5, workspace=ws[:16])
    assert e.value.status == 10


def test_writes_count(te, gpu_device):
    own = {"x": torch.zeros((1, 2, 50), device=gpu_device), "s": torch.zeros((1, 2), device=gpu_device),
           "e": torch.zeros((1, 2), dtype=torch.bool, device=gpu_device), "ws": torch.zeros(1 << 16, dtype=torch.uint8, device=gpu_device)}
    before = {n: t._version for n, t in own.items()}
    te.beam_select(own["x"], own["s"], 3, ended=own["e"], workspace=own["ws"])
    assert {n for n, t in own.items() if t._version != before[n]} == {"ws"}


def test_infinite_and_missing_scores(te, gpu_device):
    """A score that is not a number is no candidate; a logit of +inf, which is not allowed, ends the call all the same."""
    x, _ = _random(2, 5, 300, F32, 12)
    s = torch.tensor([[math.nan, -math.inf, 1e5, -1e5, 0.0], [math.nan] * 5])
    got = te.beam_select(x.to(gpu_device), s.to(gpu_device), 7)
    want = ref.beams(x, s.nan_to_num(nan=-math.inf), 7)
    assert torch.equal(got[1].cpu(), want[1]) and got[0][1].tolist() == [-math.inf] * 7 and got[1][1].tolist() == [0] * 7
    x[0, 2, 7] = math.inf
    te.beam_select(x.to(gpu_device), s.to(gpu_device), 7)
    torch.cuda.synchronize()


def test_refusals(te, gpu_device):
    dev = gpu_device
    x, s = torch.zeros((2, 3, 50), device=dev), torch.zeros((2, 3), device=dev)
    e = torch.zeros((2, 3), dtype=torch.bool, device=dev)
    call = lambda x=x, s=s, k=2, **kw: te.beam_select(x, s, k, **kw)
    bad = [lambda: call(x[0]), lambda: call(x.double()), lambda: call(x.cpu()), lambda: call(s=s[:1]), lambda: call(s=s.half()),
           lambda: call(s=s.cpu()), lambda: call(k=0), lambda: call(k=65), lambda: call(k=2.5), lambda: call(ended=e.int()),
           lambda: call(ended=e[:1]), lambda: call(end_token=50), lambda: call(end_token=-1), lambda: call(x[..., :0]),
           lambda: call(torch.zeros((1, 65, 9), device=dev), torch.zeros((1, 65), device=dev)), lambda: call(x[:, :0], s[:, :0]),
           lambda: call(x.clone().requires_grad_()), lambda: call(k=-1)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was not refused")
    assert [t.shape for t in call(x[:0], s[:0])] == [(0, 2)] * 3
    assert math.isclose(float(call(k=1)[0][0, 0]), -math.log(50), rel_tol=1e-6)
