"""The binding of the operators between the packed linears, as far as it goes without a GPU: what it refuses before it
looks at devices."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def _calls(te, t):
    """Every function with `t` among its arguments."""
    p, table, lens = torch.zeros((4, 2, 16, 64), dtype=torch.float16), torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x, w = torch.zeros((2, 64)), torch.ones(64)
    return [lambda: te.rms_norm(t, w), lambda: te.rms_norm(x, t), lambda: te.residual_norm(x, t, w),
            lambda: te.residual_norm(x, x, w, gate=t), lambda: te.residual_norm(x, x, w, post_weight=t),
            lambda: te.paged_attention(t, p, p, table, lens), lambda: te.paged_attention(x, t, p, table, lens),
            lambda: te.append_kv(t, x, x, p, p, table, lens), lambda: te.append_kv(x, x, t, p, p, table, lens),
            lambda: te.evict_kv(p, t, x, x, table, lens, 4, 1)]


def test_tangents_are_refused(te):
    """A dual tensor of forward-mode differentiation would lose its tangent; no_grad does not switch that mode off."""
    with fwd.dual_level():
        for no_grad in (False, True):
            dual = fwd.make_dual(torch.ones((2, 64)), torch.ones((2, 64)))
            for i, call in enumerate(_calls(te, dual)):
                with pytest.raises(ValueError, match="tangent"), torch.set_grad_enabled(not no_grad):
                    call()
                    pytest.fail(f"call {i} was not refused")
        primal = fwd.unpack_dual(dual).primal
        with pytest.raises(ValueError, match="GPU"):
            te.rms_norm(primal, torch.ones(64))


def test_gradients_are_refused(te):
    for i, call in enumerate(_calls(te, torch.ones((2, 64), requires_grad=True))):
        with pytest.raises(ValueError, match="forward only"):
            call()
            pytest.fail(f"call {i} was not refused")


def test_transforms_are_refused(te):
    w, x = torch.ones(64), torch.ones((2, 64))
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda t: te.rms_norm(t, w), (x,), (x,))
    with pytest.raises(ValueError, match="gradient"):
        torch.func.grad(lambda t: te.rms_norm(t, w).sum())(x)
