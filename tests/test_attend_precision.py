"""The bound that the attention's GPU tests hold its results to (attend_ref), on the CPU: the kernel's arithmetic keeps
it, and the same arithmetic with any one term lost, or with queries scaled too low for their split, does not."""
import pytest
import torch

import attend_ref as ref

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
LENGTHS = [1, 2, 2, 3, 3, 5, 9, 17, 32, 33, 64, 129, 500]


def _worst(x, cache, d, mistake, **kw):
    """Largest error in units of the bound and fp32's rounding of out."""
    q, kv = ref.inputs(LENGTHS, 2, 3, d, x, cache, d, **kw)
    worst = 0.0
    for b, (k, v) in enumerate(kv):
        for h in range(6):
            one = (q[b, h], k[h // 3].float(), v[h // 3].float(), d ** -0.5)
            want, _, _ = ref.exact(*one)
            err = (ref.kernel(*one, x, cache, F32, mistake).double() - want).abs()
            worst = max(worst, float((err / (ref.bound(*one, x, cache, F32) + ref.U * want.abs()).clamp_min(1e-300)).max()))
    return worst


@pytest.mark.parametrize("d", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("x,cache", [(F32, F16), (F32, BF16), (BF16, F16), (F16, BF16), (F16, F16), (BF16, BF16)])
def test_bound_of_the_attention(x, cache, d):
    assert _worst(x, cache, d, None) < 1
    assert _worst(x, cache, d, None, outlier=1536.0) < 1
    for outlier in (0.0, 1536.0):
        assert _worst(x, cache, d, None, keys="one", outlier=outlier) < 1
        assert _worst(x, cache, d, "p", keys="one", outlier=outlier) > 1
        if x == F32:
            assert _worst(x, cache, d, "q", keys="one", outlier=outlier) > 1
    if cache == F16:
        assert _worst(x, cache, d, "low", keys="one", outlier=1536.0) > 1
