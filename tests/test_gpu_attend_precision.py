"""paged_attention within what its arithmetic may err by, element by element (attend_ref, whose bound the CPU tests show
to fail when a term of a split is lost): queries of the cache's type and of others, plain rows, rows with one large
dim, and keys that make each logit a single product."""
import pytest
import torch

import attend_ref as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
LENGTHS = [1, 2, 0, 2, 3, 3, 5, 9, 17, 32, 33, 64, 129, 500]


def _check(te, dev, lengths, d, x, cache, y, heads=2, group=3, page=16, **kw):
    q, kv = ref.inputs(lengths, heads, group, d, x, cache, d, **kw)
    need = [-(-n // page) for n in lengths]
    g = torch.Generator().manual_seed(d)
    ids = torch.randperm(sum(need), generator=g).int()
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    k_pages, v_pages = (torch.full((sum(need), heads, page, d), float("nan"), dtype=cache) for _ in range(2))
    at = 0
    for b, (n, (k, v)) in enumerate(zip(lengths, kv)):
        table[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
        j = torch.arange(n)
        where = table[b].long()[j // page], slice(None), j % page
        k_pages[where], v_pages[where] = k.transpose(0, 1), v.transpose(0, 1)
    got = te.paged_attention(q.to(dev), k_pages.to(dev), v_pages.to(dev), table.to(dev),
                             torch.tensor(lengths, dtype=torch.int32, device=dev), out_dtype=y).cpu()
    half = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}[y]
    tiny = 2.0 ** -25 if y == F16 else 0.0
    for b, (n, (k, v)) in enumerate(zip(lengths, kv)):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        for h in range(heads * group):
            one = (q[b, h], k[h // group].float(), v[h // group].float(), d ** -0.5)
            want, _, _ = ref.exact(*one)
            bound = ref.bound(*one, x, cache, y)
            over = (got[b, h].double() - want).abs() - bound - half * (want.abs() + bound) - tiny
            assert float(over.max()) <= 0, (b, n, h, float(over.max()), float(bound.max()))


@pytest.mark.parametrize("d", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("x,cache,y", [(F32, F16, F32), (F32, BF16, F32), (BF16, F16, F32), (F16, BF16, F32), (F16, F16, F32),
                                       (BF16, BF16, F32), (F32, F16, F16), (F32, BF16, BF16)])
@pytest.mark.parametrize("keys", ["dense", "one"])
@pytest.mark.parametrize("outlier", [0.0, 1536.0])
def test_attention_within_its_arithmetic(te, gpu_device, x, cache, y, d, keys, outlier):
    _check(te, gpu_device, LENGTHS, d, x, cache, y, keys=keys, outlier=outlier)


@pytest.mark.parametrize("x,cache", [(F32, F16), (F32, BF16), (BF16, BF16)])
def test_attention_within_its_arithmetic_over_chunks(te, gpu_device, x, cache):
    """Rows in several chunks, alone and together."""
    for lengths in ([700], [3000], [0, 1300, 1, 513, 127]):
        for keys in ("dense", "one"):
            _check(te, gpu_device, lengths, 64, x, cache, F32, keys=keys, outlier=1536.0)
