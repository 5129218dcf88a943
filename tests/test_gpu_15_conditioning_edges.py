"""GPU: calls at which the attention-conditioning operators can go wrong: lists without states, numbers that are not finite, means and single values
far from the rest."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rnd(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


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
