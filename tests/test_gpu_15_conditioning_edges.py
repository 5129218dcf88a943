"""GPU: calls at which the attention-conditioning operators can go wrong: lists without states, numbers that are not finite, means and single values
far from the rest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rnd(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------ group norm
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [(0, 0), (2, 3), (-1, -1)])
@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("B,hw,C,G,dtype", [(2, (4, 4), 1024, 32, F32), (3, (16, 16), 96, 3, BF16), (2, (40, 40), 24, 3, F32), (2, (33, 9), 25, 5, F32), (2, (64, 48), 64, 4, BF16)])
def test_group_norm_of_a_value_that_is_not_finite(B, hw, C, G, dtype, act, at, bad):
    """Its group of its image is not a number as a whole, whatever the activation; every other value is as it was. Both forms."""
    from layout2img_amd import ops
    gen = _gen(C + G)
    x, w, b, dy = _rnd(gen, B, *hw, C, dtype=dtype), 1 + 0.2 * _rnd(gen, C), _rnd(gen, C), _rnd(gen, B, *hw, C, dtype=dtype)
    g, cg = 1, C // G
    broken = x.clone()
    broken[1, at[0], at[1], g * cg + cg // 2] = bad
    runs = []
    for t in (x, broken):
        leaves = [a.detach().requires_grad_() for a in (t, w, b)]
        y = ops.group_norm_act(leaves[0], G, leaves[1], leaves[2], act=act)
        runs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    group = torch.zeros(B, *hw, C, dtype=torch.bool, device=DEV)
    group[1, ..., g * cg:(g + 1) * cg] = True
    channel = torch.zeros(C, dtype=torch.bool, device=DEV)
    channel[g * cg:(g + 1) * cg] = True
    for clean, got, where, what in zip(runs[0], runs[1], (group, group, channel), ("y", "dx", "dw")):
        assert got[where].isnan().all(), what
        assert torch.equal(got[~where], clean[~where]), what
    assert torch.equal(runs[1][3][~channel], runs[0][3][~channel])


# ------------------------------------------------------------------------------------------------ cross attention
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [40, 64, 72, 128])
@pytest.mark.parametrize("Lq", [1, 64, 65, 300])
def test_cross_attention_to_a_list_without_states(Lq, D, dtype):
    from layout2img_amd import ops
    gen = _gen(Lq + D)
    q, g = _rnd(gen, 2, Lq, 4, D, dtype=dtype).requires_grad_(), _rnd(gen, 2, Lq, 4, D, dtype=dtype)
    k, v = (torch.empty(2, 0, 2, D, dtype=dtype, device=DEV).requires_grad_() for _ in range(2))
    mask = torch.empty(2, Lq, 0, dtype=torch.bool, device=DEV)
    lengths = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    for kw in ({}, {"mask": mask}, {"lengths": lengths}):
        y = ops.cross_attention(q, k, v, **kw)
        assert y.shape == q.shape and not y.any()
        dq, dk, dv = torch.autograd.grad(y, (q, k, v), g)
        assert not dq.any() and dk.shape == dv.shape == k.shape
        with torch.no_grad():
            assert not ops.cross_attention(q, k, v, **kw).any()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq,Lk,D", [(1, 20, 40), (40, 20, 40), (40, 20, 128), (1, 50, 40), (40, 50, 40), (40, 130, 128), (200, 130, 64), (1, 5000, 40), (300, 2000, 128)])
def test_cross_attention_of_a_state_that_is_not_finite(Lq, Lk, D, dtype, bad):
    """A key that is not a number makes the weights of every state of its image so: out, dq and the live states' dk and dv; the other image keeps its bits, and
    states behind a length have no gradient. An infinite key does the same where it scores +inf."""
    from layout2img_amd import ops
    gen = _gen(Lq + Lk)
    q, k, v, g = (_rnd(gen, 2, n, 1, D, dtype=dtype) for n in (Lq, Lk, Lk, Lq))
    q[..., 3] = q[..., 3].abs() + 1                          # (an infinite key scores +inf)
    n = torch.tensor([Lk - 3, Lk], dtype=torch.int32, device=DEV)
    shared = (torch.arange(Lk, device=DEV) % 4 > 0)[None, None]
    for mask in (None, shared, shared.expand(1, Lq, Lk).contiguous()):
        runs = []
        for broken in (False, True):
            kk = k.clone()
            if broken:
                kk[0, Lk // 2 + (Lk // 2) % 2 + 1, 0, 3] = bad   # (live under the masks too: an odd state)
            leaves = [a.detach().requires_grad_() for a in (q, kk, v)]
            y = ops.cross_attention(*leaves, lengths=n, mask=mask)
            runs.append([y.detach(), *torch.autograd.grad(y, leaves, g)])
        live = torch.arange(Lk, device=DEV) < Lk - 3
        if mask is not None:
            live = live & mask[0, 0]
        for clean, got, what in zip(runs[0], runs[1], ("out", "dq", "dk", "dv")):
            assert torch.equal(got[1], clean[1]), what
            if what in ("out", "dq"):
                assert got[0].isnan().all(), what
            else:
                assert got[0, live].isnan().all() and not got[0, Lk - 3:].any(), what
