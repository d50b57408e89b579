"""paged_attention where the logits are so large that fp32 steps over whole units: the softmax of what they are."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = 1 / 1.44269504    # a scale that leaves logits in powers of 2


def _run(te, dev, q, k, v, cache, y, scale):
    """One head: q [d], k and v [n, d]."""
    n, d = k.shape
    pages = -(-n // 16)
    pool = lambda t: torch.cat([t, torch.zeros((pages * 16 - n, d))]).view(pages, 1, 16, d).to(cache).to(dev)
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    return te.paged_attention(q.view(1, 1, d).to(dev), pool(k), pool(v), table, torch.tensor([n], dtype=torch.int32, device=dev),
                              scale=scale, out_dtype=y)[0, 0].double().cpu()


@pytest.mark.parametrize("x,cache,y", [(F16, F16, F16), (F32, F16, F32), (F32, BF16, F32), (BF16, BF16, BF16)])
@pytest.mark.parametrize("size", [2 ** e for e in range(9, 16)])
@pytest.mark.parametrize("n", [1, 40, 300, 700])
def test_large_logits(te, gpu_device, x, cache, y, size, n):
    """Logits up to 2^30 x 16: the token of the largest takes all, and equal ones share. Every one is a power of 2 or
    zero, so that they are exact; up to three weights, so 17 roundings of values below 4 (bf16: 16 bits of a weight)."""
    g = torch.Generator().manual_seed(n)
    d = 16
    v = torch.randn((n, d), generator=g).to(cache).float()
    q = torch.full((d,), float(size)).to(x)
    for order in ("first", "last", "shared"):
        k = torch.zeros((n, d))
        top = {"first": [0], "last": [n - 1], "shared": sorted({0, n // 2, n - 1})}[order]
        k[top] = float(size)
        if order == "last" and n > 1:
            k[:n - 1:5] = float(size) / 2
        got = _run(te, gpu_device, q, k, v, cache, y, UNIT)
        want = v[top].double().mean(0)
        ref.close(got, want, y, 2.0 ** -14 if cache == BF16 and y != F32 else 2.0 ** -18)


@pytest.mark.parametrize("x,y", [(F16, F16), (F32, F32)])
@pytest.mark.parametrize("more", [2, 4, 6, 8])
def test_a_maximum_that_grows_by_rounded_units(te, gpu_device, x, y, more):
    """Logits of 2 x 10^7, where fp32 steps by 2: a later tile's is `more` larger, between where the running maximum
    moves and where it does not."""
    n, d = 200, 8
    q, k = torch.zeros(d), torch.zeros((n, d))
    q[0], q[1] = 512.0, 1.0
    k[0, 0], k[128, 0], k[128, 1] = 39072.0, 39072.0, float(more)
    v = torch.randn((n, d), generator=torch.Generator().manual_seed(more)).half().float()
    got = _run(te, gpu_device, q.to(x), k, v, F16, y, UNIT)
    share = 2.0 ** -more
    want = (v[0].double() * share + v[128].double()) / (1 + share)
    ref.close(got, want, y, 2.0 ** -19 * max(1.0, float(v.abs().max())))


@pytest.mark.parametrize("y", [BF16, F32])
@pytest.mark.parametrize("n", [1, 3, 100, 700])
def test_large_bf16_values(te, gpu_device, y, n):
    """bf16 values up to 2^116 average to what they are: 16-bit (bf16 out) or 24-bit weights and their fp32 sums."""
    g = torch.Generator().manual_seed(n)
    q, k, v = torch.randn(64, generator=g).to(BF16), torch.randn((n, 64), generator=g).to(BF16), torch.rand((n, 64), generator=g)
    v = (v * 2.0 ** 116).to(BF16)
    got = _run(te, gpu_device, q, k.float(), v.float(), BF16, y, 0.125)
    want = torch.softmax(k.double() @ q.double() * 0.125, 0) @ v.double()
    ref.close(got, want, y, 2.0 ** 116 * (2.0 ** -15 if y == BF16 else 2.0 ** -23 * (3 * n + 200)))
