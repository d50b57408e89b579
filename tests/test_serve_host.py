"""Host-side checks of the operators between the packed linears: status codes of the C entry points before any
launch, and the paged cache's bookkeeping (no GPU)."""
import ctypes

import pytest
import torch


def _cache(te, **kw):
    c = dict(k=256, v=256, scores=256, pos=256, table=256, lens=512, page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64,
             table_stride=4, pages=9, heads=2, page_size=16, head_dim=64, dtype=1, rows=3, width=4, max_len=64)
    c.update(kw)
    return te._capi.TrellisKVCache(**c)


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), 1), (dict(table=None), 1), (dict(lens=None), 1), (dict(dtype=0), 9), (dict(head_dim=60), 19), (dict(head_dim=264), 19),
    (dict(heads=0), 19), (dict(page_size=24), 20), (dict(page_size=8), 20), (dict(page_size=2048), 20), (dict(pages=0), 20),
    (dict(width=0), 20), (dict(rows=-1), 11), (dict(max_len=-1), 11), (dict(k=264), 8), (dict(slot_stride=68), 8),
    (dict(slot_stride=56), 8), (dict(head_stride=-8), 8), (dict(slot_stride=1 << 28), 8)])
def test_cache_codes(te, kw, status):
    lib, n = te.library(), ctypes.c_size_t(0)
    c = _cache(te, **kw)
    assert lib.trellis_attention_workspace_bytes(c, 4, 0, n) == status
    assert lib.trellis_paged_attention(c, 16, 256, 64, 1, 4, 1.0, 0, 16, 1, None, 0, None) == status
    assert lib.trellis_kv_append(c, 16, 256, 64, 16, 128, 64, 16, 128, 64, 1, 3, 4, None, None, None, None, 1e-6, None, None, 0, 0, 16, 1, None) == status
    assert lib.trellis_kv_evict(c, 4, 1, None, None, 0, 0, 16, 256, 1 << 20, None) == status


def test_attention_codes(te):
    lib, n = te.library(), ctypes.c_size_t(0)
    size = lambda c, hq=4, acc=0: lib.trellis_attention_workspace_bytes(c, hq, acc, n)
    call = lambda c=_cache(te), q=16, qd=1, hq=4, acc=0, out=16, od=1, ws=None, nb=0: \
        lib.trellis_paged_attention(c, q, 256, 64, qd, hq, 1.0, acc, out, od, ws, nb, None)
    assert size(_cache(te), 3) == 19 and size(_cache(te), 0) == 19 and size(_cache(te, scores=None), 4, 1) == 1
    assert lib.trellis_attention_workspace_bytes(_cache(te), 4, 0, None) == 1
    assert size(_cache(te, max_len=1 << 20, width=1 << 16)) == 0 and n.value > 0
    assert call(qd=3) == 9 and call(od=-1) == 9 and call(q=None) == 1 and call(out=None) == 1 and call(q=17) == 8 and call(out=24) == 8
    long = _cache(te, max_len=1 << 20, width=1 << 16)
    assert call(long) == 10 and call(long, ws=256, nb=16) == 10 and call(long, ws=264, nb=1 << 40) == 8
    assert call(_cache(te), acc=1) == 10
    assert call(_cache(te, rows=0), q=None, out=None) == 0


def test_workspace_grows_with_the_call(te):
    """Scores need the logits of max_len tokens; splits never make the partial sums large."""
    lib, n = te.library(), ctypes.c_size_t(0)
    for rows, hq, length in ((1, 32, 32768), (64, 32, 8192), (1, 32, 1 << 20), (256, 32, 4096)):
        c = _cache(te, rows=rows, heads=8, head_dim=128, slot_stride=128, width=length // 16, max_len=length)
        assert lib.trellis_attention_workspace_bytes(c, hq, 0, n) == 0 and n.value < 64 << 20
        plain = n.value
        assert lib.trellis_attention_workspace_bytes(c, hq, 1, n) == 0 and plain + 4 * rows * hq * length <= n.value


def test_append_codes(te):
    lib, c = te.library(), _cache(te)
    def call(c=c, q=16, k=16, xd=1, tokens=3, hq=4, starts=None, qw=None, kw=None, cos=None, sin=None, rot=0, npos=0, out=16, qd=1):
        return lib.trellis_kv_append(c, q, 256, 64, k, 128, 64, 16, 128, 64, xd, tokens, hq, starts, None, qw, kw, 1e-6, cos, sin, rot, npos, out, qd, None)
    assert call(xd=5) == 9 and call(qd=5) == 9 and call(hq=5) == 19 and call(tokens=4) == 11 and call(tokens=-1, starts=16) == 11
    assert call(qw=16) == 1 and call(cos=16) == 1 and call(q=None) == 1 and call(out=None) == 1 and call(out=8) == 8 and call(k=17) == 8
    assert call(cos=16, sin=16, rot=24, npos=1) == 19 and call(cos=16, sin=16, rot=80, npos=1) == 19 and call(cos=16, sin=16, rot=64) == 12
    assert call(tokens=0, starts=16, q=None) == 0 and call(_cache(te, rows=0), tokens=2, starts=16) == 11


def test_evict_codes(te):
    lib, n = te.library(), ctypes.c_size_t(0)
    # (up to 64 moves of a row and head need no workspace; here 100 can be, and an out table always needs one)
    call = lambda c=_cache(te, width=32, max_len=512, table_stride=32), keep=100, recent=1, out=None, ow=0, new=16, ws=256, nb=1 << 20: \
        lib.trellis_kv_evict(c, keep, recent, None, out, 0, ow, new, ws, nb, None)
    assert call(keep=0, recent=0) == 21 and call(recent=101) == 21 and call(recent=-1) == 21 and call(_cache(te, scores=None)) == 1
    assert call(_cache(te, pos=None)) == 1 and call(out=16, ow=0) == 20 and call(new=None) == 1 and call(new=512) == 12
    assert call(ws=None) == 10 and call(nb=8) == 10 and call(ws=264) == 8 and call(_cache(te, rows=0), new=None) == 0
    size = lib.trellis_evict_workspace_bytes
    assert size(_cache(te), 0, 0, n) == 21 and size(_cache(te), 4, 0, None) == 1
    assert size(_cache(te), 4, 0, n) == 0 and n.value == 0
    assert size(_cache(te), 4, 1, n) == 0 and n.value > 0


def test_norm_codes(te):
    lib = te.library()
    def call(x=16, ldx=64, xd=0, r=16, ldr=64, rd=0, gate=None, inner=1, w=16, h=16, ldh=64, y=16, ldy=64, yd=0, rows=2, width=64):
        return lib.trellis_residual_norm(x, ldx, xd, r, ldr, rd, gate, 0, inner, None, w, 1.0, 1e-6, h, ldh, y, ldy, yd, rows, width, None)
    assert call(rows=-1) == 11 and call(width=0) == 18 and call(width=32769) == 18 and call(xd=3) == 9 and call(rd=-1) == 9 and call(yd=9) == 9
    assert call(x=None) == 1 and call(w=None) == 1 and call(y=None) == 1 and call(x=18) == 8 and call(y=18) == 8 and call(inner=2) == 8
    assert call(ldy=63) == 8 and call(ldh=63) == 8 and call(rows=1 << 40) == 11 and call(rows=0, x=None) == 0


def test_status_names(te):
    lib = te.library()
    for code in range(18, 22):
        assert lib.trellis_strerror(code).decode() != "unknown trellis status" and code in te._capi.STATUS_NAMES


def test_operators_live_on_a_gpu(te):
    x, w = torch.zeros((2, 64)), torch.ones(64)
    with pytest.raises(ValueError):
        te.rms_norm(x, w)
    p = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError):
        te.paged_attention(torch.zeros((1, 2, 64)), p, p, torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_paged_cache_pages(te):
    c = te.PagedKVCache(2, 1, 8, rows=3, max_len=40, pages=5, page_size=16, device="cpu", evictable=True)
    c.grow([1, 0, 17])
    assert c.lengths == [1, 0, 17] and c.lens.tolist() == [1, 0, 17] and len(c._free) == 2
    assert c._starts.tolist() == [0, 1, 1, 18] and c._positions.tolist() == [0] + list(range(17))
    own = [t for t in c.table.flatten().tolist() if t >= 0]
    assert len(own) == 3 == len(set(own)) and (c.table[1] == -1).all()
    c.grow(1)
    assert c.lengths == [2, 1, 18] and c._starts is None and c._positions.tolist() == [1, 0, 17]
    before = c.table.clone()
    for counts in ([39, 0, 0], [0, 0, 40], [16, 16, 0], [1, 1], [-1, 0, 0]):
        with pytest.raises(ValueError):
            c.grow(counts)
    assert c.lengths == [2, 1, 18] and torch.equal(c.table, before) and len(c._free) == 1
    c.release(2)
    assert c.lengths == [2, 1, 0] and c.seen == [2, 1, 0] and len(c._free) == 3 and (c.table[2] == -1).all()
    with pytest.raises(ValueError):
        c.append(0, *(torch.zeros((3, 1, 8)) for _ in range(3)))
    with pytest.raises(ValueError):
        te.PagedKVCache(1, 1, 8, rows=1, max_len=4, device="cpu").evict(2, 1)
    with pytest.raises(ValueError):
        te.PagedKVCache(0, 1, 8, rows=1, max_len=4, device="cpu")
