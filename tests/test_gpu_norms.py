"""rms_norm and residual_norm against float64 (serve_ref). Tolerances: every fp32 operation rounds by 2^-24;
a row's sum of squares over threads and lanes goes through at most 32 + 10 + 16 roundings of positive terms,
halved by the square root; h has 3 roundings of its terms. 64 x 2^-24 of the row's largest value covers them."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
FP = 64 * 2.0 ** -24


def _inputs(rows, width, x, r, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, width), generator=g).to(x), (torch.randn((rows, width), generator=g) * 3).to(r),
            torch.rand(width, generator=g) + 0.5, torch.rand(width, generator=g) + 0.5, g)


def _bound(t):
    return FP * t.abs().amax(-1, keepdim=True)


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 64), (5, 576), (37, 1531), (1, 4096), (300, 2000), (2, 8192),
                                        (3, 8200), (2, 12288), (2, 16384), (1, 32768), (2, 32767)])
@pytest.mark.parametrize("x,r,y", [(F32, F32, F16), (BF16, BF16, BF16), (F16, F32, F32)])
def test_residual_norm(te, gpu_device, rows, width, x, r, y):
    a, res, w, post, g = _inputs(rows, width, x, r, rows * width)
    dev = gpu_device
    for gate in (None, torch.randn((rows, width), generator=g).to(x)):
        kw = dict(scale=0.37, eps=1e-5)
        for pw in (None, post):
            got_y, got_h = te.residual_norm(a.to(dev), res.to(dev), w.to(dev), out_dtype=y,
                                            post_weight=None if pw is None else pw.to(dev),
                                            gate=None if gate is None else gate.to(dev), **kw)
            want_y, want_h = ref.residual_norm(a, res, w, pw, gate, **kw)
            assert got_y.dtype == y and got_h.dtype == r
            ref.close(got_h, want_h, r, _bound(want_h), "h")
            ref.close(got_y, want_y, y, _bound(want_y) + FP * want_h.abs().amax(-1, keepdim=True) /
                      want_h.pow(2).mean(-1, keepdim=True).add(1e-5).sqrt(), "y")


@pytest.mark.parametrize("x", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(5,), (2, 3, 100), (1, 1, 4096), (0, 64), (7, 136)])
def test_rms_norm_shapes(te, gpu_device, x, shape):
    g = torch.Generator().manual_seed(1)
    a, w = torch.randn(shape, generator=g).to(x), torch.rand(shape[-1], generator=g)
    got = te.rms_norm(a.to(gpu_device), w.to(gpu_device))
    want = ref.rms(a, w)
    assert got.shape == shape and got.dtype == x
    if want.numel():
        ref.close(got, want, x, _bound(want), "y")


def test_many_rows(te, gpu_device):
    a, res, w, _, _ = _inputs(70001, 24, F16, F32, 3)
    want_y, want_h = ref.residual_norm(a, res, w)
    y, h = te.residual_norm(a.to(gpu_device), res.to(gpu_device), w.to(gpu_device), out_dtype=F32)
    ref.close(h, want_h, F32, _bound(want_h), "h")
    ref.close(y, want_y, F32, 2 * _bound(want_y), "y")


def test_gates_and_strides(te, gpu_device):
    """Gates broadcast per row, per column and whole; rows that are strided slices; odd addresses."""
    rows, width = 6, 264
    dev = gpu_device
    a, res, w, _, g = _inputs(rows, 2 * width + 1, F16, F32, 5)
    w = w[:width].clone()
    for cols in (slice(0, width), slice(1, width + 1), slice(width, 2 * width)):
        for gate in (torch.randn((rows, 1), generator=g).half(), torch.randn((1, width), generator=g).half(),
                     torch.randn(width, generator=g).half(), torch.randn((1, 1), generator=g).half()):
            y, h = te.residual_norm(a.to(dev)[:, cols], res.to(dev)[:, cols], w.to(dev), gate=gate.to(dev), out_dtype=F32)
            want_y, want_h = ref.residual_norm(a[:, cols], res[:, cols], w, gate=gate)
            ref.close(h, want_h, F32, _bound(want_h), "h")
            ref.close(y, want_y, F32, 2 * _bound(want_y), "y")
    every = a.to(dev)[:, ::2][:, :width]       # a column stride of 2 is copied
    want = ref.rms(a[:, ::2][:, :width], w)
    ref.close(te.rms_norm(every, w.to(dev)), want, F16, _bound(want), "strided")


def test_in_place_residual_and_stream(te, gpu_device):
    a, res, w, _, _ = _inputs(9, 640, F16, F32, 8)
    want_y, want_h = ref.residual_norm(a, res, w)
    a, r, w = a.to(gpu_device), res.to(gpu_device), w.to(gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, h = te.residual_norm(a, r, w, residual_out=r)
    side.synchronize()
    assert h is r
    ref.close(r, want_h, F32, _bound(want_h), "h")
    ref.close(y, want_y, F16, 2 * _bound(want_y), "y")


def test_extremes(te, gpu_device):
    """Zero rows stay zero; a row of a type's largest values does not overflow on the way; NaN stays in its row."""
    x = torch.zeros((4, 128), dtype=F16)
    x[1] = 65504.0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    w = torch.ones(128)
    y = te.rms_norm(x.to(gpu_device), w.to(gpu_device), out_dtype=F32).cpu()
    assert torch.equal(y[0], torch.zeros(128))
    ref.close(y[1], torch.ones(128), F32, FP)
    assert y[2].isnan().all() and y[3, 7].isnan() and (y[3, :7] == 0).all()


def test_refusals(te, gpu_device):
    x, w = torch.zeros((2, 64), device=gpu_device), torch.ones(64, device=gpu_device)
    bad = [lambda: te.rms_norm(x, w.half()), lambda: te.rms_norm(x, w[:32]), lambda: te.rms_norm(x, w.cpu()),
           lambda: te.rms_norm(x.double(), w), lambda: te.rms_norm(x, w, out_dtype=torch.int32),
           lambda: te.rms_norm(x.clone().requires_grad_(), w), lambda: te.rms_norm(x.cpu(), w),
           lambda: te.residual_norm(x, x[:1], w), lambda: te.residual_norm(x, x.double(), w),
           lambda: te.residual_norm(x, x, w, gate=x.half()), lambda: te.residual_norm(x, x, w, residual_out=x.half()),
           lambda: te.residual_norm(x, x, w, post_weight=w[:1]), lambda: te.residual_norm(x, x, w, gate=x[:, :3])]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(te.TrellisError) as e:
        te.rms_norm(torch.zeros((1, 32769), device=gpu_device), torch.ones(32769, device=gpu_device))
    assert e.value.status == 18
    with torch.no_grad():
        te.rms_norm(x.clone().requires_grad_(), w)
