"""CPU: calls of the attention-conditioning operators that their checks and plans have to take or refuse before anything is launched."""
import ctypes

import pytest
import torch


def _lib():
    from layout2img_amd import _lib as L
    return L.load()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 128])
def test_cross_attention_plans_a_list_without_states(D, dtype):
    """Forward and backward, whatever the number of queries: a plan that divides by the number of the states' tiles would end the process."""
    n = (ctypes.c_longlong * 1)()
    for B, Lq, Hk, G in ((1, 1, 1, 1), (1, 64, 1, 1), (1, 65, 1, 1), (2, 65, 2, 4), (1, 100000, 1, 1), (600, 65, 1, 1)):
        for bwd in (0, 1):
            assert _lib().l2i_cross_attention_scratch(B, Lq, 0, Hk, G, D, dtype, bwd, n) == 0, (B, Lq, Hk, G, bwd)
            assert n[0] == (B * Hk * Lq * G + 3) // 4 * 4 * bwd   # (the rows' D alone: nothing is cut in ranges)
        assert _lib().l2i_cross_attention_wants_lo(B, Lq, 0, Hk, G, D, dtype) in (0, 1)


P = 1 << 20   # an address that is never read: every call below is refused before a launch


def _backward(Lq, Hk, G, D, dtype):
    st = (0, D, 0) * 3   # heads in front of positions: the checks of q, k and v pass whatever the number of heads
    return _lib().l2i_cross_attention_bwd(P, P, P, dtype, None, None, P, None, P, P, P, P, P, 1, Lq, 64, Hk, G, D, *st, 0, 0, 1.0, P, 1 << 50, None)


def _span(Lq, Hk, G, D):
    """values between the first and the last of any 64 rows of a contiguous (Lq, Hk G, D) gradient that belong to one state head"""
    at = lambda r: (r // G) * Hk * G * D + (r % G) * D
    R = Lq * G
    return max(at(min(R - 1, r + 63)) - (r // G) * Hk * G * D + D for r in range(min(R, 64 * G)))


def test_cross_attention_refuses_a_gradient_whose_tiles_pass_32_bits():
    """q and k with heads in front of positions step by D, but the gradient of the result, which is contiguous, by all heads: offsets that are counted in
    32 bits would come round."""
    from layout2img_amd import ops
    for Lq, Hk, G, D, dtype in ((64, 1 << 21, 1, 8, 0), (64, 1 << 18, 1, 128, 1), (2, 1 << 23, 4, 128, 1), (33, 1 << 17, 2, 128, 0), (2, 1 << 22, 1, 128, 0)):
        assert not ops._xa_backward_reaches(Lq, Hk, G, D, 2 if dtype else 4)
        assert _backward(Lq, Hk, G, D, dtype) == -1, (Lq, Hk, G, D, dtype)
    z = torch.zeros(1, 1, 1, 8)
    q, k = z.expand(1, 64, 1 << 21, 8), z.expand(1, 64, 1 << 21, 8)
    with pytest.raises(RuntimeError, match="further apart"):
        ops.cross_attention(q.detach().requires_grad_(), k, k)
    with pytest.raises(RuntimeError, match="GPU"):   # (the forward pass alone does not read it)
        ops.cross_attention(q, k, k)
    for G in (1, 2, 3, 5, 31, 32, 62, 63, 64, 65, 100):
        for Lq in (1, 2, 3, 40, 64, 65, 200):
            for Hk in (1, 7, 1 << 15, 1 << 18, 1 << 20):
                for size in (2, 4):
                    if ops._xa_backward_reaches(Lq, Hk, G, 128, size):
                        assert _span(Lq, Hk, G, 128) * size < 1 << 31, (G, Lq, Hk, size)


def _calls(monkeypatch):
    """The operators as calls of one tensor that carries a derivative, with the launches themselves taken out: what the host layer does around them."""
    from layout2img_amd import ops
    monkeypatch.setattr(ops._lib, "call", lambda *a: 0)
    monkeypatch.setattr(ops, "_same_device", lambda *a: None)
    monkeypatch.setattr(ops, "_scratch_floats", lambda *a: 16)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    q, kv, x, w = torch.randn(1, 2, 2, 16), torch.randn(1, 3, 2, 16), torch.randn(2, 3, 3, 8), torch.randn(8)
    rng, tok = torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int64)
    return [(x, lambda t: ops.group_norm_act(t, 2)), (w, lambda t: ops.group_norm_act(x, 2, t)), (w, lambda t: ops.group_norm_act(x, 2, None, t)),
            (q, lambda t: ops.cross_attention(t, kv, kv)), (kv, lambda t: ops.cross_attention(q, t, kv)), (kv, lambda t: ops.cross_attention(q, kv, t)),
            (torch.randn(4, 8), lambda t: ops.embedding(t, tok)), (x, lambda t: ops.dropout(t, 0.5, rng)), (x, lambda t: ops.dropout(x, 0.5, rng, residual=t))]


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_derivatives_are_refused_not_dropped(monkeypatch, grad_mode):
    fa = torch.autograd.forward_ad
    for i, (t, f) in enumerate(_calls(monkeypatch)):
        with torch.set_grad_enabled(grad_mode):
            with fa.dual_level():
                with pytest.raises(NotImplementedError, match="jvp"):
                    f(fa.make_dual(t, torch.ones_like(t)))
                assert f(t).shape is not None, i                  # (without a tangent the call is an ordinary one)
            with pytest.raises((RuntimeError, NotImplementedError)):
                torch.func.jvp(f, (t,), (torch.ones_like(t),))
            with pytest.raises((RuntimeError, NotImplementedError)):
                torch.func.vmap(f)(t[None])
            assert f(t).shape is not None, i


def test_a_trace_is_refused(monkeypatch):
    for t, f in _calls(monkeypatch):
        for grad in (False, True):
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(f, (t.detach().requires_grad_(grad),), check_trace=False)
