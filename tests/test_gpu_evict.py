"""evict_kv in forms beside test_gpu_kv.py's, against the definition: moves are copies, so everything is
compared bit for bit."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [1 << 20, 2 ** 30])
def test_keep_beyond_every_row(te, gpu_device, keep):
    """Nothing is evicted; into other pages everything is copied. Scratch goes by the rows, not by `keep`."""
    lengths = [70, 0, 33, 16]
    P = ref.Pages(lengths, 2, 16, 64, torch.float16, 1, idle=None)
    need = -(-max(lengths) // 16)
    out = (P.pages + torch.arange(need * len(lengths))).int().view(len(lengths), need)
    grow = lambda t: torch.cat([t, torch.zeros_like(t[:1]).expand(out.numel(), *t.shape[1:])])
    P.k, P.v, P.scores, P.pos = (grow(t) for t in (P.k, P.v, P.scores, P.pos))
    k, v, table, lens, scores, pos = P.to(gpu_device)
    new = te.evict_kv(k, v, scores, pos, table, lens, keep, 5, out_table=out.to(gpu_device))
    assert new.tolist() == lengths
    for b, n in enumerate(lengths):
        page, slot = P.slots(b, n)
        to = out[b].long()[torch.arange(n) // 16]
        for got, old in ((k, P.k), (v, P.v), (scores, P.scores), (pos, P.pos)):
            assert torch.equal(got.cpu()[to, :, slot], old[page, :, slot])
    before = [t.clone() for t in (k, v, scores, pos)]
    assert te.evict_kv(k, v, scores, pos, table, lens, keep, 5).tolist() == lengths
    assert all(torch.equal(a, b) for a, b in zip(before, (k, v, scores, pos)))
