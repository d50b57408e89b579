"""paged_attention under a max_len that is a bound and not the rows' own: rows far below it, empty ones, and a captured
call whose rows grow under it. Tolerances as in test_gpu_kv.py."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def _pages(lengths, bound, heads, page, d, seed):
    """Rows whose tables reach as far as the bound, beyond their own pages with ids that are none."""
    P = ref.Pages(lengths, heads, page, d, F16, seed)
    table = torch.full((len(lengths), -(-bound // page)), -1, dtype=torch.int32)
    table[:, :P.width] = P.table
    P.table, P.width = table, table.shape[1]
    return P


@pytest.mark.parametrize("bound", [600, 4000, 32768, 131072])
@pytest.mark.parametrize("lengths", [[0], [1], [127], [513], [0, 0, 0], [1, 0, 300], [20, 1025, 0, 511]])
@pytest.mark.parametrize("heads,group,d", [(2, 4, 64), (1, 18, 256)])
def test_rows_far_below_the_bound(te, gpu_device, bound, lengths, heads, group, d):
    lengths = [min(n, bound) for n in lengths]
    P = _pages(lengths, bound, heads, 16, d, seed=bound + len(lengths))
    q = torch.randn((len(lengths), heads * group, d), generator=P.g).half()
    k, v, table, lens, scores, _ = P.to(gpu_device)
    want, want_scores = ref.attend(q, P)
    for y, acc in ((F16, None), (F32, scores)):
        got = te.paged_attention(q.to(gpu_device), k, v, table, lens, max_len=bound, scores=acc, out_dtype=y)
        ref.close(got, want, y, 2e-4 * float(P.v.double().nan_to_num(0).abs().max()))
    assert float((scores.double().cpu() - want_scores).abs().max()) <= 2e-4 * group + 2 ** -20


def test_a_captured_call_whose_rows_grow(te, gpu_device):
    """Replays under one bound, from empty rows to full ones, with eager calls between."""
    bound, lengths = 3000, [3000, 2000, 700]
    P = _pages(lengths, bound, 2, 16, 64, seed=5)
    q = torch.randn((3, 8, 64), generator=P.g).half()
    k, v, table, lens, scores, _ = P.to(gpu_device)
    dq, at = q.to(gpu_device), torch.zeros_like(lens)

    def call(acc):
        return te.paged_attention(dq, k, v, table, at, max_len=bound, scores=acc, out_dtype=F32)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(scores.clone())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(scores)
    for now in ([0, 0, 0], [1, 0, 700], [513, 2000, 3], [3000, 1, 0], [3000, 2000, 700]):
        at.copy_(torch.tensor(now, dtype=torch.int32))
        twin = scores.clone()
        graph.replay()
        eager = call(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(scores, twin)
        ref.close(out, ref.attend(q, P, lengths=now)[0], F32, 2e-4 * float(P.v.double().nan_to_num(0).abs().max()))
