"""What the binding of the operators between the packed linears owes torch: version counts of what a call writes into,
torch's own errors, refusals of transforms."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def _cache(dev):
    P = ref.Pages([40, 3], 2, 16, 64, F16, 0, idle=0.0, room=2)
    q, t = torch.zeros((2, 4, 64), dtype=F16, device=dev), torch.zeros((2, 2, 64), dtype=F16, device=dev)
    return P.to(dev), q, t


def test_writes_count(te, gpu_device):
    """Each call adds one to the version of every tensor it writes into, and to no other."""
    (k, v, table, lens, scores, pos), q, t = _cache(gpu_device)
    x, w = torch.zeros((2, 64), device=gpu_device), torch.ones(64, device=gpu_device)
    r, out = torch.zeros_like(x), torch.zeros_like(q)
    own = {"k": k, "v": v, "table": table, "lens": lens, "scores": scores, "pos": pos, "q": q, "t": t, "x": x, "r": r, "w": w, "out": out}

    def counted(call):
        before = {n: u._version for n, u in own.items()}
        call()
        return {n for n, u in own.items() if u._version != before[n]}

    assert counted(lambda: te.rms_norm(x, w)) == set()
    assert counted(lambda: te.residual_norm(x, r, w)) == set()
    assert counted(lambda: te.residual_norm(x, r, w, residual_out=r)) == {"r"}
    assert counted(lambda: te.append_kv(q, t, t, k, v, table, lens)) == {"k", "v"}
    assert counted(lambda: te.append_kv(q, t, t, k, v, table, lens, scores=scores, pos=pos)) == {"k", "v", "scores", "pos"}
    assert counted(lambda: te.paged_attention(q, k, v, table, lens)) == set()
    assert counted(lambda: te.paged_attention(q, k, v, table, lens, scores=scores, out=out)) == {"scores", "out"}
    assert counted(lambda: te.evict_kv(k, v, scores, pos, table, lens, 4, 1)) == {"k", "v", "scores", "pos"}


def test_a_saved_tensor_that_a_call_overwrites_is_noticed(te, gpu_device):
    h = torch.ones((2, 64), device=gpu_device)
    scale = torch.ones((), device=gpu_device, requires_grad=True)
    loss = (scale * h).sum()          # saves h for scale's gradient
    with torch.no_grad():
        te.residual_norm(torch.ones_like(h), h, torch.ones(64, device=gpu_device), residual_out=h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors(te, gpu_device):
    """A cache made under inference_mode is used inside it and outside."""
    with torch.inference_mode():
        (k, v, table, lens, scores, pos), q, t = _cache(gpu_device)
        te.append_kv(q, t, t, k, v, table, lens, scores=scores, pos=pos)
    with torch.no_grad():
        te.append_kv(q, t, t, k, v, table, lens, scores=scores, pos=pos)
        te.paged_attention(q, k, v, table, lens, scores=scores)
        te.evict_kv(k, v, scores, pos, table, lens, 4, 1)
    assert (k[table[0, 2].item(), :, 7] == 0).all()


def test_out_of_memory_is_torchs_error(te, gpu_device):
    """An output or scratch that does not fit raises what torch raises, so that a caller can catch it."""
    big = torch.zeros((1, 32768), dtype=F16, device=gpu_device).expand(1 << 18, 32768)     # 32 GiB of f32 out of 64 KiB
    weight = torch.ones(32768, device=gpu_device)
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(0.05)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            te.rms_norm(big, weight, out_dtype=F32)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert te.rms_norm(big[:2], weight).shape == (2, 32768)


def test_transforms_are_refused(te, gpu_device):
    x, w = torch.ones((2, 64), device=gpu_device), torch.ones(64, device=gpu_device)
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.vmap(lambda t: te.rms_norm(t, w))(x)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda t: te.rms_norm(t, w), (x,), (x,))
