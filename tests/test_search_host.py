"""Host-side checks of the operators that carry several hypotheses over a paged cache: status codes of the C entry points
before any launch, and what the binding refuses before it looks at devices (no GPU)."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd


def _cache(te, **kw):
    c = dict(k=256, v=256, scores=256, pos=256, table=256, lens=512, page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64,
             table_stride=4, pages=9, heads=2, page_size=16, head_dim=64, dtype=1, rows=3, width=4, max_len=64)
    c.update(kw)
    return te._capi.TrellisKVCache(**c)


BAD_CACHE = [(dict(k=None), 1), (dict(dtype=0), 9), (dict(head_dim=60), 19), (dict(heads=0), 19), (dict(page_size=24), 20), (dict(pages=0), 20),
             (dict(width=0), 20), (dict(rows=-1), 11), (dict(max_len=-1), 11), (dict(k=264), 8), (dict(slot_stride=68), 8), (dict(slot_stride=1 << 28), 8)]


@pytest.mark.parametrize("kw,status", BAD_CACHE + [(dict(table=None), 1), (dict(lens=None), 1)])
def test_cache_codes(te, kw, status):
    lib, n, c = te.library(), ctypes.c_size_t(0), _cache(te, **kw)
    assert lib.trellis_tree_attention_workspace_bytes(c, 6, 4, 1, 1, n) == status
    assert lib.trellis_tree_attention(c, 16, 256, 64, 1, 6, 4, 16, None, 1.0, 16, 1, None, 0, None) == status
    assert lib.trellis_kv_copy_pages(c, 1, 16, 16, None, 1, None) == status
    assert lib.trellis_kv_keep(c, 1, 16, 16, 4, 4, 16, None) == status


def test_tree_codes(te):
    lib, n = te.library(), ctypes.c_size_t(0)
    def call(c=_cache(te), q=16, qd=1, tokens=6, hq=4, starts=16, out=16, od=1, ws=None, nb=0):
        return lib.trellis_tree_attention(c, q, 256, 64, qd, tokens, hq, starts, None, 1.0, out, od, ws, nb, None)
    assert call(hq=3) == 19 and call(hq=0) == 19 and call(qd=3) == 9 and call(od=-1) == 9 and call(tokens=-1) == 11
    assert call(starts=None, tokens=7) == 11 and call(_cache(te, rows=0), tokens=1) == 11
    assert call(q=None) == 1 and call(out=None) == 1 and call(q=17) == 8 and call(out=24) == 8
    assert call(tokens=0, q=None, out=None) == 0 and call(_cache(te, rows=0), tokens=0) == 0
    size = lib.trellis_tree_attention_workspace_bytes
    assert size(_cache(te), 6, 4, 1, 1, None) == 1 and size(_cache(te), 6, 3, 1, 1, n) == 19 and size(_cache(te), -1, 4, 1, 1, n) == 11
    assert size(_cache(te), 6, 4, 1, 1, n) == 0


def test_beam_codes(te):
    lib, n = te.library(), ctypes.c_size_t(0)
    def call(x=16, dt=1, batch=2, beams=3, vocab=50, scores=16, end=0, k=4, out=16, frm=16, token=16, ws=256, nb=1 << 20):
        return lib.trellis_beam_select(x, 150, 50, dt, batch, beams, vocab, scores, None, end, k, out, frm, token, ws, nb, None)
    assert call(batch=-1) == 11 and call(beams=0) == 22 and call(beams=65) == 22 and call(k=0) == 22 and call(k=65) == 22 and call(vocab=0) == 22
    assert call(dt=3) == 9 and call(end=50) == 12 and call(end=-1) == 12 and call(batch=0, x=None) == 0
    assert call(x=None) == 1 and call(scores=None) == 1 and call(out=None) == 1 and call(frm=None) == 1 and call(token=None) == 1
    assert call(x=17) == 8 and call(scores=18) == 8 and call(out=18) == 8 and call(ws=None) == 10 and call(nb=16) == 10 and call(ws=264) == 8
    size = lib.trellis_beam_workspace_bytes
    assert size(2, 3, 50, 4, None) == 1 and size(2, 65, 50, 4, n) == 22 and size(2, 3, 50, 4, n) == 0 and 0 < n.value < 1 << 16


def test_layer_codes(te):
    lib = te.library()
    both = lambda **kw: (te._capi.TrellisKVCache * 2)(_cache(te), _cache(te, **kw))
    for call in (lambda c, n: lib.trellis_kv_copy_pages(c, n, 16, 16, None, 0, None),
                 lambda c, n: lib.trellis_kv_keep(c, n, 16, 16, 4, -1 if n == 2 else 4, 16, None)):
        assert call(both(), 0) == 23 and call(None, 1) == 1
        for kw in (dict(pages=8), dict(heads=1), dict(head_dim=56), dict(page_size=32), dict(dtype=2), dict(page_stride=4096),
                   dict(head_stride=2048), dict(slot_stride=72)):
            assert call(both(**kw), 2) == 23, kw
        assert call(both(scores=258), 2) == 8 and call(both(pos=259), 2) == 8 and call(both(v=None), 2) == 1
    c = _cache(te)
    assert lib.trellis_kv_copy_pages(both(), 2, None, None, None, 0, None) == 0
    assert lib.trellis_kv_copy_pages(c, 1, None, 16, None, 1, None) == 1 and lib.trellis_kv_copy_pages(c, 1, 16, None, None, 1, None) == 1
    assert lib.trellis_kv_copy_pages(c, 1, 16, 16, None, -1, None) == 11 and lib.trellis_kv_copy_pages(c, 1, 16, 16, None, 2 ** 31 - 1, None) == 11
    keep = lambda c=c, starts=16, path=16, stride=4, width=4, new=16: lib.trellis_kv_keep(c, 1, starts, path, stride, width, new, None)
    assert keep(starts=None) == 1 and keep(path=None) == 1 and keep(new=None) == 1 and keep(width=-1) == 12 and keep(stride=-1) == 12
    assert keep(new=512) == 12 and keep(_cache(te, rows=0, table=None, lens=None), starts=None, new=None) == 0


def test_status_names(te):
    lib = te.library()
    for code in (22, 23):
        assert lib.trellis_strerror(code).decode() != "unknown trellis status" and code in te._capi.STATUS_NAMES


def _calls(te, t):
    p, table, lens = torch.zeros((4, 2, 16, 64), dtype=torch.float16), torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    return [lambda: te.tree_attention(t, p, p, table, lens), lambda: te.tree_attention(torch.zeros((1, 2, 64)), t, p, table, lens),
            lambda: te.beam_select(t, torch.zeros((1, 1)), 1), lambda: te.copy_pages([t], [p], lens, lens),
            lambda: te.copy_pages([p, p], [p, t], lens, lens), lambda: te.keep_kv(p, t, table, lens, lens, table)]


def test_what_the_binding_refuses(te):
    for i, call in enumerate(_calls(te, torch.ones((1, 2, 64), requires_grad=True))):
        with pytest.raises(ValueError, match="forward only|GPU"):
            call()
            pytest.fail(f"call {i} was not refused")
    with fwd.dual_level():
        dual = fwd.make_dual(torch.ones((1, 2, 64)), torch.ones((1, 2, 64)))
        for i, call in enumerate(_calls(te, dual)):
            with pytest.raises(ValueError, match="tangent|GPU"), torch.no_grad():
                call()
                pytest.fail(f"call {i} was not refused")
    for i, call in enumerate(_calls(te, torch.ones((4, 2, 16, 64), dtype=torch.float16))):
        with pytest.raises(ValueError):       # the host's memory
            call()
            pytest.fail(f"call {i} was not refused")
