"""CPU: what the attention-conditioning operators refuse (in Python and at the C entry points, which check before they launch), the scratch they
ask for, and their references against torch and published values."""
import ctypes
import math

import pytest
import torch

from tests import conditioning_ref as R

F32, BF16 = torch.float32, torch.bfloat16
Z = torch.zeros


def _refused(match, fn, *a, **k):
    with pytest.raises(RuntimeError, match=match):
        fn(*a, **k)


def test_group_norm_refusals():
    from layout2img_amd import ops
    f = ops.group_norm_act
    x = Z(2, 3, 3, 8)
    _refused("tensor expected", f, None, 2)
    _refused("float16", f, x.half(), 2)
    _refused("op_dtype", f, x, 2, op_dtype=torch.float16)
    _refused("contiguous", f, x.transpose(1, 3), 1)
    _refused("contiguous", f, Z(0, 3, 8), 2)
    _refused("contiguous", f, Z(8), 2)
    _refused("groups", f, x, 3)
    _refused("groups", f, x, 0)
    _refused("groups", f, x, 2.0)
    _refused("4096", f, Z(1, 1, 8192), 2)
    _refused("act", f, x, 2, act="gelu")
    _refused("weight", f, x, 2, Z(7))
    _refused("weight", f, x, 2, Z(8, dtype=BF16))
    _refused("bias", f, x, 2, Z(8), Z(16)[::2])
    _refused("GPU", f, x, 2)


def test_cross_attention_refusals():
    from layout2img_amd import ops
    f = ops.cross_attention
    q, k = Z(2, 3, 4, 16), Z(2, 5, 2, 16)
    _refused("tensor expected", f, q, None, k)
    _refused("float64", f, q.double(), k, k)
    _refused("one type", f, q, k.bfloat16(), k.bfloat16())
    _refused("heads, D", f, q[0], k, k)
    _refused("belong together", f, q, k, k[:, :4])
    _refused("belong together", f, q, k[:1], k[:1])
    _refused("belong together", f, q, Z(2, 5, 2, 8), Z(2, 5, 2, 8))
    for d in (4, 12, 136, 0):
        _refused("multiple of 8", f, Z(1, 1, 1, d), Z(1, 1, 1, d), Z(1, 1, 1, d))
    _refused("divide", f, q, Z(2, 5, 3, 16), Z(2, 5, 3, 16))
    one = Z(1, 1, 1, 8)
    for shapes in (((1 << 24, 1, 1, 8), (1 << 24, 1, 1, 8)), ((1, 1, 65537, 8), (1, 1, 1, 8)), ((1 << 14, 1 << 17, 1, 8), (1 << 14, 1, 1, 8)),
                   ((1 << 14, 1, 1, 8), (1 << 14, 1 << 16, 1, 8)), ((1, (1 << 30) + 1, 1, 8), (1, 1, 1, 8))):
        _refused("tiles", f, one.expand(shapes[0]), one.expand(shapes[1]), one.expand(shapes[1]))
    _refused("at least one", f, Z(2, 0, 4, 16), k, k)
    _refused("consecutive", f, Z(2, 3, 16, 4).transpose(2, 3), k, k)
    _refused("16-byte", f, Z(2, 3, 4, 18)[..., :16], k, k)
    _refused("16-byte", f, Z(2 * 3 * 4 * 16 + 1)[1:].view(2, 3, 4, 16), k, k)
    _refused("lengths", f, q, k, k, lengths=Z(3, dtype=torch.int32))
    _refused("lengths", f, q, k, k, lengths=Z(2, dtype=torch.int64))
    _refused("mask", f, q, k, k, mask=Z(2, 3, 5))
    for shape in ((2, 3, 4), (3, 3, 5), (2, 2, 5), (2, 5), (2, 4, 3, 5)):
        _refused("mask", f, q, k, k, mask=Z(shape, dtype=torch.bool))
    _refused("consecutive", f, q, k, k, mask=Z(2, 5, 3, dtype=torch.bool).transpose(1, 2))
    _refused("GPU", f, q, k, k, mask=Z(1, 1, 5, dtype=torch.bool))


def test_embedding_refusals():
    from layout2img_amd import ops
    f = ops.embedding
    w, t = Z(5, 8), Z(3, dtype=torch.int64)
    _refused("float16", f, w.half(), t)
    _refused("op_dtype", f, w, t, op_dtype=torch.int64)
    _refused(r"\(V, D\)", f, w[0], t)
    _refused(r"\(V, D\)", f, Z(0, 8), t)
    _refused(r"\(V, D\)", f, Z(1, 65537), t)
    _refused("contiguous", f, w.t(), t)
    _refused("tokens", f, w, t.float())
    _refused("tokens", f, w, [1, 2])
    _refused("padding_idx", f, w, t, padding_idx=5)
    _refused("padding_idx", f, w, t, padding_idx=-2)
    _refused("padding_idx", f, w, t, padding_idx=None)
    _refused("GPU", f, w, t)


def test_dropout_refusals():
    from layout2img_amd import ops
    f = ops.dropout
    x, r = Z(6), Z(2, dtype=torch.int64)
    _refused("float16", f, x.half(), 0.5, r)
    for p in (-0.1, 1.1, math.nan):
        _refused("p lies", f, x, p, r)
    for layer in (-1, 1 << 31, 0.5):
        _refused("layer", f, x, 0.5, r, layer=layer)
    _refused("rng", f, x, 0.5, Z(3, dtype=torch.int64))
    _refused("rng", f, x, 0.5, Z(2, dtype=torch.int32))
    _refused("rng", f, x, 0.5, Z(4, dtype=torch.int64)[::2])
    _refused("contiguous", f, Z(4, 4).t(), 0.5, r)
    _refused("contiguous", f, Z(4, 4), 0.5, r, residual=Z(4, 4).t())
    _refused("residual", f, x, 0.5, r, residual=Z(5))
    _refused("residual", f, x, 0.5, r, residual=x, op_dtype=BF16)
    _refused("residual", f, x, 0.5, r, residual=1.0)
    _refused("GPU", f, x, 0.5, r)


P = 1 << 20   # an address that is never read: every call below is refused before a launch


def _lib():
    from layout2img_amd import _lib as L
    return L.load()


def _floats(name, *sizes):
    n = (ctypes.c_longlong * 1)()
    rc = getattr(_lib(), name)(*sizes, n)
    return rc, n[0]


def test_entry_points_refuse_before_a_launch():
    lib, big = _lib(), 1 << 40
    gn = lambda x=P, xd=0, y=P, yd=0, m=P, r=P, B=2, HW=9, C=8, G=2, act=0, s=P, n=big: lib.l2i_group_norm_fwd(
        x, xd, None, None, y, yd, m, r, B, HW, C, G, 1e-5, act, s, n, None)
    gb = lambda x=P, dy=P, m=P, C=8, G=2, s=P, n=big: lib.l2i_group_norm_bwd(x, 0, None, None, m, P, dy, 0, P, P, P, 2, 9, C, G, 0, s, n, None)
    for bad in (dict(x=None), dict(y=None), dict(m=None), dict(r=None), dict(xd=2), dict(yd=-1), dict(B=0), dict(B=65536), dict(HW=0), dict(C=4097), dict(G=3),
                dict(G=0), dict(act=3), dict(s=None), dict(s=P + 4), dict(n=0), dict(HW=1 << 40)):
        assert gn(**bad) == -1, bad
    for bad in (dict(x=None), dict(dy=None), dict(m=None), dict(G=5), dict(C=0), dict(s=None), dict(n=1)):
        assert gb(**bad) == -1, bad
    xa = lambda q=P, k=P, v=P, dt=1, o=P, B=2, Lq=3, Lk=5, Hk=2, G=2, D=16, st=(0,) * 9, mb=0, mq=0, s=None, n=0, lo=None: lib.l2i_cross_attention_fwd(
        q, k, v, dt, None, None, o, lo, None, B, Lq, Lk, Hk, G, D, *st, mb, mq, 1.0, s, n, None)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(dt=2), dict(B=0), dict(Lq=0), dict(Lk=-1), dict(Hk=0), dict(G=0), dict(D=0), dict(D=12),
                dict(D=136), dict(q=P + 8), dict(o=P + 2), dict(st=(4,) + (0,) * 8), dict(st=(0,) * 8 + (-8,)), dict(mb=-1), dict(mq=-1), dict(Lq=1 << 30, G=2),
                dict(lo=P, dt=0), dict(lo=P + 8), dict(B=1 << 24), dict(G=65537), dict(B=1 << 14, Lq=1 << 17, G=1), dict(B=1 << 14, Lk=1 << 16), dict(Lk=100000)):   # (the last one needs scratch)
        assert xa(**bad) == -1, bad
    xb = lambda lse=P, g=P, dq=P, dk=P, dv=P, s=P, n=big: lib.l2i_cross_attention_bwd(
        P, P, P, 1, None, None, P, None, lse, g, dq, dk, dv, 2, 3, 5, 2, 2, 16, *(0,) * 11, 1.0, s, n, None)
    for bad in (dict(lse=None), dict(g=None), dict(dk=None), dict(dv=None), dict(dq=P + 8), dict(s=None), dict(s=P + 4), dict(n=1)):
        assert xb(**bad) == -1, bad
    ef = lambda w=P, wd=0, t=P, o=P, od=0, n=3, V=5, D=8: lib.l2i_embedding_fwd(w, wd, t, o, od, n, V, D, 1.0, -1, None)
    for bad in (dict(w=None), dict(t=None), dict(o=None), dict(wd=3), dict(od=2), dict(n=-1), dict(n=1 << 31), dict(V=0), dict(V=0x7fffffff), dict(D=0), dict(D=65537)):
        assert ef(**bad) == -1, bad
    assert ef(n=0) == 0
    eb = lambda t=P, dy=P, dw=P, n=3000, V=5, D=8, s=P, sn=big: lib.l2i_embedding_bwd(t, dy, 0, dw, 0, n, V, D, 1.0, -1, s, sn, None)
    for bad in (dict(t=None), dict(dy=None), dict(dw=None), dict(n=-1), dict(n=0x7fffffff), dict(V=0), dict(D=0), dict(s=None), dict(s=P + 4), dict(sn=3)):
        assert eb(**bad) == -1, bad
    dr = lambda x=P, xd=0, o=P, od=0, r=P, n=5, t=7, layer=0: lib.l2i_dropout(x, xd, None, o, od, r, None, n, t, 1.0, layer, None)
    for bad in (dict(x=None), dict(o=None), dict(r=None), dict(xd=2), dict(od=4), dict(n=-1), dict(n=(1 << 34) + 1), dict(t=-1), dict(t=(1 << 32) + 1), dict(layer=-1)):
        assert dr(**bad) == -1, bad
    assert dr(n=0) == 0


def test_scratch_sizes():
    assert _floats("l2i_group_norm_scratch", 2, 9, 8, 3, 0)[0] == -1
    assert _floats("l2i_cross_attention_scratch", 1, 1, 1, 1, 1, 7, 1, 0)[0] == -1
    assert _floats("l2i_embedding_bwd_scratch", -1, 5, 8)[0] == -1
    for B, HW, C, G in ((1, 1, 1, 1), (32, 16384, 64, 32), (65535, 1, 4096, 1)):
        for bwd in (0, 1):
            rc, n = _floats("l2i_group_norm_scratch", B, HW, C, G, bwd)
            assert rc == 0 and 0 <= n < 1 << 31
    assert _floats("l2i_cross_attention_scratch", 4, 4096, 2048, 4, 4, 128, 1, 0) == (0, 0)   # rows enough: no splits
    lib = _lib()
    assert [lib.l2i_cross_attention_wants_lo(1, 64, lk, 1, 1, 64, dt) for lk, dt in ((31, 1), (33, 1), (33, 0), (-1, 1))] == [0, 1, 0, 0]
    rc, n = _floats("l2i_cross_attention_scratch", 1, 1, 4096, 1, 1, 128, 1, 0)
    assert rc == 0 and n > 0


def test_generator_words_are_the_published_ones():
    assert [hex(int(w)) for w in R.words(0, 0, 0, 0, 1)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_references_against_torch(dtype):
    torch.manual_seed(0)
    q, k, v, g = (torch.randn(2, n, h, 16).to(dtype) for n, h in ((33, 4), (20, 2), (20, 2), (33, 4)))
    n = torch.tensor([20, 7], dtype=torch.int32)
    want, tol = R.cross_attention(q, k, v, n, None, None, g)
    leaves = [t.float().requires_grad_() for t in (q, k, v)]
    s = leaves[0].transpose(1, 2) @ leaves[1].transpose(1, 2).repeat_interleave(2, 1).transpose(2, 3) / 4
    s = s.masked_fill(~(torch.arange(20)[None] < n[:, None])[:, None, None], -1e30)
    y = (torch.softmax(s, -1) @ leaves[2].transpose(1, 2).repeat_interleave(2, 1)).transpose(1, 2)
    for a, w, t, what in zip([y, *torch.autograd.grad(y, leaves, g.float())], want, tol, ("out", "dq", "dk", "dv")):
        R.close(a.to(dtype), w, t, what)
    x, w, b, dy = torch.randn(2, 5, 5, 12) + 3, torch.randn(12), torch.randn(12), torch.randn(2, 5, 5, 12)
    want, tol = R.group_norm_act(x, 3, w, b, 1e-5, "silu", F32, dy)
    ls = [t.requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.silu(torch.nn.functional.group_norm(x.permute(0, 3, 1, 2), 3, w, b)).permute(0, 2, 3, 1)
    for a, r, t, what in zip([y, *torch.autograd.grad(y, ls, dy)], want, tol, ("y", "dx", "dw", "db")):
        R.close(a, r, t, what)
