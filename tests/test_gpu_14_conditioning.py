"""GPU: the attention-conditioning operators (ops.group_norm_act, cross_attention, embedding, dropout) against plain references in 64 bits
(tests/conditioning_ref.py, which states the tolerances), at the sizes, strides and masks where they can go wrong; a run of them together."""
import math

import pytest
import torch

from tests import conditioning_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rnd(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------ group norm
GN = [  # B, spatial, C, G, act, x, y
    (1, (1, 1), 8, 2, None, F32, F32), (2, (3, 5), 12, 4, "silu", F32, F32), (2, (7, 1), 25, 5, "silu", F32, BF16), (3, (4, 4), 1024, 32, "relu", F32, BF16),
    (2, (16, 16), 100, 4, "silu", BF16, BF16), (1, (33, 31), 64, 32, "silu", BF16, F32), (2, (64, 64), 32, 1, None, BF16, BF16),
    (4, (8, 8), 96, 96, "silu", F32, F32), (1, (5,), 4096, 1, "relu", BF16, F32), (1, (2, 3), 1023, 33, "silu", F32, F32), (2, (128, 96), 8, 8, "silu", F32, F32),
    (1, (1, 1), 1, 1, None, F32, F32), (70, (2, 2), 16, 4, "silu", F32, F32),
    (2, (15, 15), 512, 32, "silu", BF16, BF16), (2, (16, 16), 96, 3, "relu", BF16, BF16), (1, (257,), 64, 2, "silu", BF16, BF16), (2, (11, 12), 64, 2, None, BF16, BF16),
]


@pytest.mark.parametrize("B,hw,C,G,act,ti,to", GN)
def test_group_norm_act(B, hw, C, G, act, ti, to):
    from layout2img_amd import ops
    gen = _gen(B + C + G)
    x = (_rnd(gen, B, *hw, C, scale=1.5) + _rnd(gen, B, *(1,) * len(hw), C)).to(ti).requires_grad_()
    w, b = (1 + 0.2 * _rnd(gen, C)).requires_grad_(), (0.2 * _rnd(gen, C)).requires_grad_()
    dy = _rnd(gen, B, *hw, C, dtype=to)
    y = ops.group_norm_act(x, G, w, b, act=act, op_dtype=to)
    assert y.dtype == to
    outs = [y, *torch.autograd.grad(y, (x, w, b), dy)]
    want, tol = R.group_norm_act(x, G, w, b, 1e-5, act, to, dy)
    for got, ref, t, what in zip(outs, want, tol, ("y", "dx", "dw", "db")):
        R.close(got, ref, t, what)
    with torch.no_grad():
        assert torch.equal(ops.group_norm_act(x, G, w, b, act=act, op_dtype=to), y)


def test_group_norm_without_affine_and_a_far_mean():
    from layout2img_amd import ops
    gen = _gen(1)
    x = (_rnd(gen, 2, 40, 40, 24) + 1000.0).requires_grad_()   # the mean is a thousand deviations away
    dy = _rnd(gen, 2, 40, 40, 24)
    y = ops.group_norm_act(x, 3)
    want, tol = R.group_norm_act(x, 3, None, None, 1e-5, None, F32, dy)
    R.close(y, want[0], tol[0], "y")
    R.close(torch.autograd.grad(y, x, dy)[0], want[1], tol[1], "dx")
    const = torch.full((1, 6, 6, 8), 3.25, device=DEV)
    assert torch.equal(ops.group_norm_act(const, 2), torch.zeros_like(const))


def test_group_norm_of_a_map_off_its_alignment():
    from layout2img_amd import ops
    gen = _gen(2)
    flat = _rnd(gen, 2 * 9 * 16 + 1)
    x = flat[1:].view(2, 3, 3, 16)                            # contiguous, four bytes off
    want, tol = R.group_norm_act(x, 4, None, None, 1e-5, "silu", F32)
    R.close(ops.group_norm_act(x, 4, act="silu"), want[0], tol[0], "y")


def test_group_norm_of_maps_past_32_bits():
    """More values than 2^31; the last image is the first one again."""
    from layout2img_amd import ops
    gen = _gen(22)
    x = _rnd(gen, 3, 700, 1024, 1024, dtype=BF16)
    x[2] = x[0]
    x.requires_grad_()
    w = (1 + 0.2 * _rnd(gen, 1024)).requires_grad_()
    y = ops.group_norm_act(x, 32, w, act="silu")
    assert y.numel() > 1 << 31 and torch.equal(y[2], y[0])
    (dx, dw) = torch.autograd.grad(y, (x, w), y.detach())
    assert torch.equal(dx[2], dx[0]) and dw.isfinite().all()


# ------------------------------------------------------------------------------------------------ cross attention
def _xa(B, Lq, Lk, Hk, G, D, dtype, seed, lengths=None, mask=None):
    gen = _gen(seed)
    q, k, v = _rnd(gen, B, Lq, Hk * G, D, dtype=dtype, scale=1.5), _rnd(gen, B, Lk, Hk, D, dtype=dtype), _rnd(gen, B, Lk, Hk, D, dtype=dtype)
    g = _rnd(gen, B, Lq, Hk * G, D, dtype=dtype)
    return q, k, v, g


def _check_xa(q, k, v, g, lengths=None, mask=None, scale=None, what=""):
    from layout2img_amd import ops
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    y = ops.cross_attention(*leaves, lengths=lengths, mask=mask, scale=scale)
    outs = [y, *torch.autograd.grad(y, leaves, g)]
    want, tol = R.cross_attention(q, k, v, lengths, mask, scale, g)
    for got, ref, t, name in zip(outs, want, tol, ("out", "dq", "dk", "dv")):
        R.close(got, ref, t, what + name)
    with torch.no_grad():
        assert torch.equal(ops.cross_attention(*leaves, lengths=lengths, mask=mask, scale=scale), y)
    return outs


XA = [  # B, Lq, Lk, Hk, G, D
    (1, 1, 1, 1, 1, 8), (2, 1, 33, 2, 4, 64), (2, 5, 31, 4, 1, 32), (1, 32, 32, 1, 1, 16), (1, 33, 65, 2, 1, 40), (2, 129, 64, 1, 3, 128),
    (1, 7, 130, 2, 2, 96), (1, 257, 31, 1, 1, 128), (3, 64, 8, 2, 1, 56), (1, 1, 1000, 1, 1, 128), (1, 100, 500, 1, 1, 64), (1, 17, 200, 3, 5, 24),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Lq,Lk,Hk,G,D", XA)
def test_cross_attention(B, Lq, Lk, Hk, G, D, dtype):
    _check_xa(*_xa(B, Lq, Lk, Hk, G, D, dtype, Lq + Lk + D))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq,Lk,D", [(1, 300, 64), (40, 150, 32), (200, 31, 40)])
def test_cross_attention_lengths_of_zero_one_and_all(Lq, Lk, D, dtype):
    q, k, v, g = _xa(6, Lq, Lk, 2, 2, D, dtype, 3)
    n = torch.tensor([0, 1, Lk, Lk // 2, 2 * Lk, -3], dtype=torch.int32, device=DEV)
    bad = torch.arange(Lk, device=DEV)[None, :, None, None] >= n[:, None, None, None]
    k, v = k.masked_fill(bad, math.nan), v.masked_fill(bad, math.inf)   # nothing behind a length is read
    outs = _check_xa(q, k, v, g, lengths=n)
    assert not outs[0][0].any() and not outs[1][0].any() and not outs[2][0].any() and not outs[2].masked_select(bad).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq,Lk,G", [(1, 200, 4), (70, 31, 1), (130, 70, 2), (40, 161, 1)])
def test_cross_attention_masks_and_rows_without_a_state(Lq, Lk, G, dtype):
    q, k, v, g = _xa(3, Lq, Lk, 2, G, 48, dtype, 4)
    gen = _gen(5)
    mask = torch.rand(3, Lq, Lk, generator=gen, device=DEV) < 0.3
    mask[0, ::3] = False                                    # rows that see nothing
    mask[1] = False                                         # an image whose queries all see nothing
    mask[2, :, Lk // 2:] = False                            # keys that nobody sees
    outs = _check_xa(q, k, v, g, mask=mask)
    assert not outs[0][1].any() and not outs[1][1].any() and not outs[2][1].any() and not outs[0][0, ::3].any()
    n = torch.tensor([Lk, Lk, 5], dtype=torch.int32, device=DEV)
    _check_xa(q, k, v, g, lengths=n, mask=mask)
    _check_xa(q, k, v, g, mask=mask[:1].expand(3, Lq, Lk))   # one mask for every image
    _check_xa(q, k, v, g, mask=mask[:1])
    # a mask row that every query shares: its states are not read
    row = mask[:, 1:2] if Lq > 1 else mask
    kk, vv = (t.masked_fill(~row.transpose(1, 2)[..., None], math.nan) for t in (k, v))
    _check_xa(q, kk, vv, g, mask=row, lengths=n)
    _check_xa(q, kk, vv, g, mask=row.expand(3, Lq, Lk), lengths=n)
    wide = torch.zeros(3, Lq, Lk + 7, dtype=torch.bool, device=DEV)
    wide[:, :, 3:3 + Lk] = mask
    _check_xa(q, k, v, g, mask=wide[:, :, 3:3 + Lk])         # rows that start anywhere


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Lq,Hk,G,D", [(1, 1, 1, 1, 40), (2, 1, 2, 4, 128), (1, 2, 1, 9, 64), (1, 60, 1, 1, 64)])
def test_cross_attention_of_few_queries_over_many_ranges(B, Lq, Hk, G, D, dtype):
    """Enough states that they are cut in dozens of ranges, of which a length or a mask leaves many without a state."""
    Lk = 9001
    q, k, v, g = _xa(B, Lq, Lk, Hk, G, D, dtype, 11)
    _check_xa(q, k, v, g)
    n = torch.tensor([700, 0][:B], dtype=torch.int32, device=DEV)
    bad = torch.arange(Lk, device=DEV)[None, :, None, None] >= n[:, None, None, None]
    _check_xa(q, k.masked_fill(bad, math.nan), v.masked_fill(bad, math.inf), g, lengths=n)
    mask = torch.zeros(B, Lq, Lk, dtype=torch.bool, device=DEV)
    mask[:, :, 5000:5003] = True
    mask[:, :, 8999] = True
    _check_xa(q, k, v, g, mask=mask)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq,Lk", [(1, 20), (40, 20), (1, 50), (40, 50), (40, 130), (1, 5000)])
def test_cross_attention_of_a_query_that_is_not_a_number(Lq, Lk, dtype):
    """Its own rows and every live state's gradients are not numbers either; other images and rows are as they were, and a state that a length or a
    mask of all queries takes out has no gradient (one that a query's own mask takes out weighs 0, and 0 times that query is not a number)."""
    from layout2img_amd import ops
    q, k, v, g = _xa(2, Lq, Lk, 1, 1, 40, dtype, 23)
    bad = q.clone()
    bad[0, Lq // 2, 0, 3] = math.nan
    n = torch.tensor([Lk - 3, Lk], dtype=torch.int32, device=DEV)
    shared = (torch.arange(Lk, device=DEV) % 4 > 0)[None, None]
    for mask in (None, shared, shared.expand(1, Lq, Lk).contiguous()):
        runs = []
        for t in (q, bad):
            leaves = [a.detach().requires_grad_() for a in (t, k, v)]
            y = ops.cross_attention(*leaves, lengths=n, mask=mask)
            runs.append([y, *torch.autograd.grad(y, leaves, g)])
        live = torch.arange(Lk, device=DEV) < Lk - 3
        if mask is not None:
            live = live & mask[0, 0]
        for a, b in zip(runs[0][:2], runs[1][:2]):
            assert b[0, Lq // 2].isnan().all() and torch.equal(b[1], a[1]) and torch.equal(b[0, :Lq // 2].isnan(), a[0, :Lq // 2].isnan())
            assert b[0, Lq // 2 + 1:].isfinite().all()
        gone = ~live if mask is None or mask.shape[1] < Lq or Lq == 1 else torch.arange(Lk, device=DEV) >= Lk - 3
        for a, b in zip(runs[0][2:], runs[1][2:]):
            assert b[0, live].isnan().all() and not b[0, gone].any() and torch.equal(b[1], a[1])


def test_cross_attention_with_scores_of_any_size():
    q, k, v, g = _xa(1, 50, 90, 1, 1, 64, F32, 6)
    _check_xa(q * 30, k, v, g, scale=0.5)                    # probabilities of one and zero
    _check_xa(q, k, v, g, scale=-0.25)
    _check_xa(q, k, v, g, scale=0.0)
    k2 = k.clone()
    k2[:, 60:] = torch.finfo(F32).max
    _check_xa(q, k2, v, g, lengths=torch.tensor([60], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq,Lk", [(1, 200), (50, 150), (50, 20)])
def test_cross_attention_of_far_low_scores_beside_dead_states(Lq, Lk, dtype):
    """Every live score lies hundreds below 0, where a state that is not there would score 0 and take the row over (or overflow) if it counted."""
    q, k, v, g = _xa(2, Lq, Lk, 2, 1, 64, dtype, 17)
    q, k = q * 0.1 + 6, k * 0.1 - 6                          # scores about -288 with a scale of 1 / 8
    n = torch.tensor([Lk - 7, Lk // 2], dtype=torch.int32, device=DEV)
    _check_xa(q, k, v, g, lengths=n)
    mask = (torch.arange(Lk, device=DEV) % 3 > 0)[None, None]
    _check_xa(q, k, v, g, mask=mask, lengths=n)
    _check_xa(q, k, v, g, mask=mask.expand(2, Lq, Lk).contiguous())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_attention_strides(dtype):
    """Slices of a grouped projection, heads in front of positions, states expanded over the batch; gradients come in the leaves' own form."""
    from layout2img_amd import ops
    gen = _gen(7)
    B, Lq, Lk, H, D = 2, 37, 50, 4, 32
    kv = _rnd(gen, B, Lk, 2, 2, D, dtype=dtype).requires_grad_()
    q = _rnd(gen, B, H, Lq, D, dtype=dtype).requires_grad_()
    g = _rnd(gen, B, Lq, H, D, dtype=dtype)
    y = ops.cross_attention(q.transpose(1, 2), kv[:, :, 0], kv[:, :, 1])
    dq, dkv = torch.autograd.grad(y, (q, kv), g)
    want, tol = R.cross_attention(q.transpose(1, 2), kv[:, :, 0], kv[:, :, 1], g=g)
    for got, ref, t, n in zip((y, dq.transpose(1, 2), dkv[:, :, 0], dkv[:, :, 1]), want, tol, ("out", "dq", "dk", "dv")):
        R.close(got, ref, t, n)
    k1 = _rnd(gen, 1, Lk, 2, D, dtype=dtype).requires_grad_()
    qq = _rnd(gen, 3, Lq, 2, D, dtype=dtype)
    g = _rnd(gen, 3, Lq, 2, D, dtype=dtype)
    e = k1.expand(3, Lk, 2, D)
    y = ops.cross_attention(qq, e, e)
    (dk1,) = torch.autograd.grad(y, (k1,), g)
    want, tol = R.cross_attention(qq, e, e, g=g)
    R.close(y, want[0], tol[0], "out")
    total, bound = want[2].sum(0, keepdim=True) + want[3].sum(0, keepdim=True), tol[2].sum(0, keepdim=True) + tol[3].sum(0, keepdim=True)
    R.close(dk1, total, bound + 8 * R.u(dtype) * (want[2].abs() + want[3].abs()).sum(0, keepdim=True), "dk of a broadcast input")   # (autograd adds 6 values in the type)
    y = ops.cross_attention(qq, e.detach(), e.detach())
    assert torch.equal(y, ops.cross_attention(qq, e.detach().contiguous(), e.detach().contiguous()))


def test_cross_attention_far_offsets_in_a_long_cache():
    """Rows of a state cache whose offsets pass 32 bits (in values and in bytes)."""
    from layout2img_amd import ops
    gen = _gen(8)
    B, Lk, D, step = 3, 70, 64, (1 << 30) + 1024
    big = torch.zeros(2 * step + Lk * 2 * D, dtype=BF16, device=DEV)
    kv = _rnd(gen, B, Lk, 2, D, dtype=BF16)
    cache = big.as_strided((B, Lk, 2, D), (step, 2 * D, D, 1))
    cache.copy_(kv)
    q = _rnd(gen, B, 3, 1, D, dtype=BF16)
    a = ops.cross_attention(q, cache[:, :, :1], cache[:, :, 1:])
    assert torch.equal(a, ops.cross_attention(q, kv[:, :, :1].contiguous(), kv[:, :, 1:].contiguous()))


def test_cross_attention_of_queries_past_32_bits():
    """More query values than 2^31, a block of 128 rows over and over: its results repeat bit for bit, and dv's rows add up to the number of queries."""
    from layout2img_amd import ops
    gen = _gen(21)
    n, D = (1 << 17) + 1, 128
    block = _rnd(gen, 1, 128, 1, D, dtype=BF16)
    q = block.repeat(1, n, 1, 1).requires_grad_()
    k, v = (_rnd(gen, 1, 40, 1, D, dtype=BF16).requires_grad_() for _ in range(2))
    y = ops.cross_attention(q, k, v)
    assert y.numel() > 1 << 31
    for part in (1, n // 2, n - 1):
        assert torch.equal(y[:, 128 * part:128 * part + 128], y[:, :128]), part
    dq, dk, dv = torch.autograd.grad(y, (q, k, v), torch.ones(1, device=DEV, dtype=BF16).expand_as(y).contiguous())
    for part in (1, n // 2, n - 1):
        assert torch.equal(dq[:, 128 * part:128 * part + 128], dq[:, :128]), part
    # P and dv are rounded to bf16 (2^-9 each), a sum of 4096 steps a range in 32 bits errs by 2^-12: below 2^-7
    assert torch.allclose(dv.double().sum(1), torch.tensor(128.0 * n, dtype=torch.float64, device=DEV), rtol=2.0 ** -7, atol=0.0) and dk.isfinite().all()


def test_cross_attention_no_states():
    from layout2img_amd import ops
    q = torch.randn(2, 3, 2, 16, device=DEV, requires_grad=True)
    k = torch.zeros(2, 0, 2, 16, device=DEV, requires_grad=True)
    y = ops.cross_attention(q, k, k)
    assert not y.any()
    dq, dk = torch.autograd.grad(y.sum(), (q, k))
    assert not dq.any() and dk.shape == k.shape


# ------------------------------------------------------------------------------------------------ embedding
EMB = [  # tokens' shape, V, D, W, y
    ((5, 3), 7, 180, F32, F32), ((1,), 1, 1, F32, F32), ((256,), 184, 180, F32, BF16), ((33, 31), 500, 64, BF16, BF16), ((5000,), 3, 7, F32, F32),
    ((9000,), 300, 20, BF16, F32), ((20000,), 70000, 8, F32, F32), ((100,), 100000, 1, BF16, F32), ((8192,), 256, 4, F32, F32), ((8193,), 255, 4, F32, F32),
    ((12345,), 1, 100, F32, F32), ((64,), 40, 1026, F32, F32), ((1024,), 9, 520, BF16, BF16), ((1025,), 9, 520, BF16, BF16), ((1000,), 17000, 12, F32, F32),
    ((32768,), 300, 6, F32, F32), ((32769,), 66000, 6, BF16, BF16), ((131072,), 1000, 3, F32, F32), ((131073,), 40, 3, F32, F32), ((524289,), 70000, 1, F32, F32), ((300, 1001), 70000, 2, F32, F32),
]


@pytest.mark.parametrize("shape,V,D,ti,to", EMB)
def test_embedding(shape, V, D, ti, to):
    from layout2img_amd import ops
    gen = _gen(V + D)
    w = _rnd(gen, V, D, dtype=ti).requires_grad_()
    tok = torch.randint(-1, V + 1, shape, generator=gen, device=DEV)     # some lie outside the table
    skew = torch.rand(shape, generator=gen, device=DEV) < 0.5
    tok = torch.where(skew, torch.full_like(tok, V // 2), tok)            # half of them the same
    dy = _rnd(gen, *shape, D, dtype=to)
    for pad in (-1, V // 3):
        y = ops.embedding(w, tok, scale=1.7, padding_idx=pad, op_dtype=to)
        (dw,) = torch.autograd.grad(y, (w,), dy)
        want, tol = R.embedding(w, tok, 1.7, pad, to, dy)
        R.close(y, want[0], tol[0], "y")
        R.close(dw, want[1], tol[1], "dw")
        y2 = ops.embedding(w, tok.int(), scale=1.7, padding_idx=pad, op_dtype=to)
        assert torch.equal(y2, y) and torch.equal(torch.autograd.grad(y2, (w,), dy)[0], dw)   # the same bits on every run


def test_embedding_of_nothing_and_of_a_transposed_batch():
    from layout2img_amd import ops
    w = torch.randn(6, 12, device=DEV, requires_grad=True)
    y = ops.embedding(w, torch.zeros(0, 3, dtype=torch.int64, device=DEV))
    assert y.shape == (0, 3, 12) and not torch.autograd.grad(y.sum(), (w,))[0].any()
    tok = torch.randint(0, 6, (4, 5), device=DEV)
    assert torch.equal(ops.embedding(w, tok.t()), w[tok.t()])


def test_embedding_of_more_rows_than_a_launch_has_workgroups():
    from layout2img_amd import ops
    w = torch.arange(1.0, 3 * 255 + 1, device=DEV).view(3, 255).to(BF16)      # a workgroup a row
    n = (1 << 24) + 5
    tok = torch.arange(n, device=DEV) % 3
    y = ops.embedding(w, tok)
    for at in (0, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 1, 1 << 24, n - 1):
        assert torch.equal(y[at], w[at % 3]), at
    assert int((y[:, 254] == w[tok, 254]).sum()) == n
    del y
    for V, toks in (((1 << 23) + 5, [(1 << 23) + 4]), ((1 << 27) + 9, [0, 1 << 26, (1 << 26) - 1, (1 << 27) + 8, 1 << 26]), ((1 << 23) + 5, [])):
        w = torch.zeros(V, 1, device=DEV, requires_grad=True)
        t = torch.tensor(toks, dtype=torch.int64, device=DEV)
        dy = torch.arange(1.0, len(toks) + 1, device=DEV)[:, None]
        (dw,) = torch.autograd.grad(ops.embedding(w, t), (w,), dy)
        want = torch.zeros(V, 1, device=DEV).index_add_(0, t, dy)
        assert torch.equal(dw, want)


def test_embedding_table_past_32_bits():
    from layout2img_amd import ops
    V, D = (1 << 24) + 3, 136                                   # 2.3e9 values
    w = torch.zeros(V, D, dtype=BF16, device=DEV)
    w[-1] = 2.0
    w[5] = 3.0
    w.requires_grad_()
    tok = torch.tensor([V - 1, 5, V - 1], device=DEV)
    y = ops.embedding(w, tok)
    assert torch.equal(y[:, 0].float().cpu(), torch.tensor([2.0, 3.0, 2.0]))
    (dw,) = torch.autograd.grad(y, (w,), torch.ones_like(y))
    assert float(dw[-1].float().sum()) == 2 * D and float(dw[5].float().sum()) == D and float(dw[6:-1].abs().max()) == 0


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("ti,to", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("n,p", [(1, 0.5), (3, 0.1), (4, 0.9), (1027, 0.0), (4096, 0.25), (100003, 0.1), (8, 1.0)])
def test_dropout(n, p, ti, to):
    from layout2img_amd import ops
    gen = _gen(n)
    rng = torch.tensor([(n << 40) + 0xF123456789, (1 << 62) + n], dtype=torch.int64, device=DEV)
    x, dy, res = _rnd(gen, n, dtype=ti).requires_grad_(), _rnd(gen, n, dtype=to), _rnd(gen, n, dtype=to).requires_grad_()
    for layer in (0, (1 << 31) - 1):
        y = ops.dropout(x, p, rng, residual=res, layer=layer)
        dx, dres = torch.autograd.grad(y, (x, res), dy)
        want, tol = R.dropout(x, p, rng, layer, res, to, dy)
        R.close(y, want[0], tol[0], "y")
        R.close(dx, want[1], tol[1], "dx")
        assert torch.equal(dres, dy)
        y = ops.dropout(x.detach(), p, rng, layer=layer, op_dtype=to)
        want, tol = R.dropout(x, p, rng, layer, None, to)
        R.close(y, want[0], tol[0], "y without a residual")


def test_dropout_of_infinities_off_alignment_and_far_elements():
    from layout2img_amd import ops
    rng = torch.tensor([-5, 77], dtype=torch.int64, device=DEV)
    x = torch.full((1001,), math.inf, device=DEV)[1:]
    y = ops.dropout(x, 0.5, rng)
    on = R.keep(2 ** 64 - 5, 77, 0, 1000, 0.5)
    assert torch.equal(y.cpu(), torch.where(on, math.inf, 0.0))
    n = (1 << 31) + 5
    big = torch.ones(n, dtype=BF16, device=DEV)
    y = ops.dropout(big, 0.25, rng)
    first = (n - 4096) // 4
    tail = y[4 * first:].float().cpu()
    on = R.keep(2 ** 64 - 5, 77, 0, len(tail), 0.25, first)
    assert torch.equal(tail != 0, on)


def test_dropout_of_more_elements_than_a_launch_takes():
    from layout2img_amd import ops
    rng = torch.tensor([3, 9], dtype=torch.int64, device=DEV)
    n = (1 << 33) + 9
    x = torch.ones(n, dtype=BF16, device=DEV)
    y = ops.dropout(x, 0.25, rng, layer=2)
    for first in (0, (1 << 31) - 8, 1 << 31):                 # in blocks of four
        part = y[4 * first:4 * first + 64].float().cpu()
        assert torch.equal(part != 0, R.keep(3, 9, 2, len(part), 0.25, first)), first


def test_dropout_keeps_its_share_and_its_mask():
    from layout2img_amd import ops
    rng = torch.tensor([11, 0], dtype=torch.int64, device=DEV)
    x = torch.ones(1 << 20, device=DEV, requires_grad=True)
    y = ops.dropout(x, 0.3, rng)
    rng[1] += 1                                               # the backward pass uses the pair that the forward read
    (dx,) = torch.autograd.grad(y, (x,), torch.ones_like(y))
    assert torch.equal(dx, y.detach())
    share = float((y != 0).double().mean())
    assert abs(share - 0.7) < 6 * math.sqrt(0.3 * 0.7 / (1 << 20))
    other = ops.dropout(x.detach(), 0.3, rng)
    assert abs(float(((y != 0) == (other != 0)).double().mean()) - (0.49 + 0.09)) < 6 * math.sqrt(0.25 / (1 << 20))


# ------------------------------------------------------------------------------------------------ together
def _block(x, table, tok, gw, gb, wq, wkv, rng, mask, lengths, dtype):
    """The conditioning half of a block: the map looks at its layout's states and adds what it read."""
    from layout2img_amd import ops
    B, H, W, C = x.shape
    heads, D = 2, C // 2
    st = ops.embedding(table, tok, scale=math.sqrt(C), padding_idx=0, op_dtype=dtype)
    h = ops.group_norm_act(x, 4, gw, gb, act="silu", op_dtype=dtype)
    q = (h.reshape(-1, C) @ wq.to(dtype)).view(B, H * W, heads, D)
    kv = (st.reshape(-1, C) @ wkv.to(dtype)).view(B, -1, 2, heads, D)
    a = ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1], lengths=lengths, mask=mask)
    return ops.dropout(a.reshape(x.shape), 0.25, rng, residual=x, layer=3)


def _block_inputs(seed, B=2, S=9, C=64, O=13, V=30):
    gen = _gen(seed)
    x = _rnd(gen, B, S, S, C)
    leaves = [x, _rnd(gen, V, C), 1 + 0.1 * _rnd(gen, C), 0.1 * _rnd(gen, C), _rnd(gen, C, C, scale=C ** -0.5), _rnd(gen, C, 2 * C, scale=C ** -0.5)]
    tok = torch.randint(0, V, (B, O), generator=gen, device=DEV)
    mask = torch.rand(B, S * S, O, generator=gen, device=DEV) < 0.6
    return leaves, tok, mask, torch.tensor([9, O], dtype=torch.int32, device=DEV), torch.tensor([3, 4], dtype=torch.int64, device=DEV), _rnd(gen, B, S, S, C)


def _block_ref(leaves, tok, mask, lengths, rng, dy):
    """The same block from elementary operations in 64 bits, under autograd."""
    x, table, gw, gb, wq, wkv = (t.detach().double().cpu().requires_grad_() for t in leaves)
    tok, mask, lengths = tok.cpu(), mask.cpu(), lengths.cpu()
    B, H, W, C = x.shape
    st = table[tok] * math.sqrt(C) * (tok != 0)[..., None]
    xg = x.view(B, H * W, 4, C // 4)
    z = ((xg - xg.mean((1, 3), keepdim=True)) / (xg.var((1, 3), unbiased=False, keepdim=True) + 1e-5).sqrt()).view(B, H * W, C) * gw + gb
    q = ((z * torch.sigmoid(z)) @ wq).view(B, H * W, 2, C // 2).transpose(1, 2)
    kv = (st @ wkv).view(B, -1, 2, 2, C // 2).permute(2, 0, 3, 1, 4)
    live = (mask & (torch.arange(mask.shape[2])[None, None] < lengths[:, None, None]))[:, None]
    s = (q @ kv[0].transpose(2, 3) / math.sqrt(C // 2)).masked_fill(~live, -1e30)
    e = torch.exp(s - s.amax(-1, keepdim=True)) * live
    a = ((e / e.sum(-1, keepdim=True).clamp(min=1e-300)) @ kv[1]).transpose(1, 2).reshape(x.shape)
    on = R.keep(*(int(t) for t in rng.tolist()), 3, x.numel(), 0.25).view(x.shape)
    y = x + torch.where(on, a / 0.75, 0.0)
    return [y, *torch.autograd.grad(y, (x, table, gw, gb, wq, wkv), dy.double().cpu())]


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_operators_together(dtype):
    leaves, tok, mask, lengths, rng, dy = _block_inputs(21)
    leaves = [t.requires_grad_() for t in leaves]
    y = _block(leaves[0], leaves[1], tok, *leaves[2:], rng, mask, lengths, dtype)
    outs = [y, *torch.autograd.grad(y, leaves, dy)]
    # a chain of five products and sums over at most 162 rows; bf16: each of ~10 roundings on the way adds u to the relative error of the whole
    rel = 12 * R.u(BF16) if dtype == BF16 else 4096 * R.U32
    for got, ref, what in zip(outs, _block_ref(leaves, tok, mask, lengths, rng, dy), ("y", "x", "table", "weight", "bias", "wq", "wkv")):
        off = float((got.detach().double().cpu() - ref).norm() / ref.norm())
        assert off < rel, (what, off)


def test_gradients_against_differences():
    leaves, tok, mask, lengths, rng, dy = _block_inputs(22, S=5)
    leaves = [t.requires_grad_() for t in leaves]
    f = lambda ls: float((_block(ls[0], ls[1], tok, *ls[2:], rng, mask, lengths, F32).detach().double() * dy.double()).sum())
    y = _block(leaves[0], leaves[1], tok, *leaves[2:], rng, mask, lengths, F32)
    grads = torch.autograd.grad(y, leaves, dy)
    gen = _gen(23)
    for i, g in enumerate(grads):
        d = _rnd(gen, *g.shape)
        d = d / d.norm() * leaves[i].detach().norm()
        slope = float((g.double() * d.double()).sum())
        h = 2e-3    # truncation h^2 of a smooth function of relative steps, rounding U32 sqrt(n) |y| / h
        with torch.no_grad():
            diff = (f([t + h * d if j == i else t for j, t in enumerate(leaves)]) - f([t - h * d if j == i else t for j, t in enumerate(leaves)])) / (2 * h)
        size = float(g.double().norm() * d.double().norm())
        assert abs(diff - slope) < 2e-3 * size, (i, diff, slope, size)


def test_a_captured_block_replays_what_it_computes_eagerly():
    """Forward and backward in one graph, replayed several times with new inputs, masks and offsets, eager work and waits between the replays."""
    leaves, tok, mask, lengths, rng, dy = _block_inputs(24)
    leaves = [t.requires_grad_() for t in leaves]
    run = lambda: (lambda y: [y.detach(), *torch.autograd.grad(y, leaves, dy)])(_block(leaves[0], leaves[1], tok, *leaves[2:], rng, mask, lengths, F32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                                        # two graphs of the same work: neither may use what the other writes
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(run())
        graphs.append(g)
    for step in range(4):
        with torch.no_grad():
            for t in leaves:
                t.add_(0.01 * (step + 1) * torch.randn_like(t))
            rng[1] += 1
            mask.copy_(torch.rand(mask.shape, device=DEV) < 0.5)
            lengths.copy_(torch.tensor([step, 13 - step], dtype=torch.int32))
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for got in outs:
            for a, b in zip(got, want):
                assert torch.equal(a, b), step


def test_another_stream_and_two_runs_give_the_same_bits():
    leaves, tok, mask, lengths, rng, dy = _block_inputs(25, S=16, O=40)
    leaves = [t.requires_grad_() for t in leaves]
    run = lambda: (lambda y: [y.detach(), *torch.autograd.grad(y, leaves, dy)])(_block(leaves[0], leaves[1], tok, *leaves[2:], rng, mask, lengths, BF16))
    a = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run()
    torch.cuda.synchronize()
    for s, t in zip(a, b):
        assert torch.equal(s, t)


def test_no_second_derivative():
    from layout2img_amd import ops
    x = torch.randn(2, 4, 4, 8, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(ops.group_norm_act(x, 2, act="silu").sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_wide_heads_captured_and_replayed():
    """Kernels that ask for more than 64 KiB of LDS, split ranges and joins, inside a graph; the scratch of a replay is the graph's own."""
    from layout2img_amd import ops
    gen = _gen(31)
    sets = []
    for Lq, Lk in ((1, 3000), (70, 600), (300, 40)):
        q, k, v = (_rnd(gen, 2, n, 2, 128, dtype=BF16).requires_grad_() for n in (Lq, Lk, Lk))
        sets.append((q, k, v, _rnd(gen, 2, Lq, 2, 128, dtype=BF16), torch.tensor([Lk, Lk // 3], dtype=torch.int32, device=DEV)))

    def run():
        out = []
        for q, k, v, g, n in sets:
            y = ops.cross_attention(q, k, v, lengths=n)
            out += [y.detach(), *torch.autograd.grad(y, (q, k, v), g)]
        return out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    for step in range(3):
        with torch.no_grad():
            for q, k, v, g, n in sets:
                q.mul_(0.9), g.neg_()
                n[0] -= 7
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), step


def test_gradients_of_some_inputs_only_and_of_an_expanded_gradient():
    from layout2img_amd import ops
    q, k, v, g = _xa(2, 40, 70, 2, 1, 32, F32, 32)
    want, tol = R.cross_attention(q, k, v, g=torch.ones_like(g))
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        y = ops.cross_attention(*leaves)
        first = torch.autograd.grad(y.sum(), (leaves[i],), retain_graph=True)[0]      # (the gradient of a sum is an expanded one)
        R.close(first, want[1 + i], tol[1 + i], f"input {i}")
        assert torch.equal(torch.autograd.grad(y.sum(), (leaves[i],))[0], first)     # a graph that is used twice
    x, w, b = _rnd(_gen(33), 2, 20, 20, 16), 1 + 0.1 * _rnd(_gen(34), 16), _rnd(_gen(35), 16)
    want, tol = R.group_norm_act(x, 4, w, b, 1e-5, "silu", F32, torch.ones_like(x))
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        R.close(torch.autograd.grad(ops.group_norm_act(leaves[0], 4, leaves[1], leaves[2], act="silu").sum(), (leaves[i],))[0], want[1 + i], tol[1 + i], f"gn {i}")


def test_two_streams_at_once():
    """The same operators on two streams at the same time: no workspace is shared."""
    from layout2img_amd import ops
    gen = _gen(36)
    q, k, v = _rnd(gen, 1, 4, 2, 64, dtype=BF16), _rnd(gen, 1, 5000, 2, 64, dtype=BF16), _rnd(gen, 1, 5000, 2, 64, dtype=BF16)
    x = _rnd(gen, 4, 64, 64, 32)
    w = _rnd(gen, 300, 16).requires_grad_()
    tok = torch.randint(0, 300, (30000,), generator=gen, device=DEV)
    dy = _rnd(gen, 30000, 16)
    run = lambda: [ops.cross_attention(q, k, v), ops.group_norm_act(x, 8, act="silu"), torch.autograd.grad(ops.embedding(w, tok), (w,), dy)[0]]
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for outs in got:
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_a_tensor_of_the_cpu_is_refused():
    from layout2img_amd import ops
    q = torch.zeros(1, 2, 2, 16, device=DEV)
    for bad in (dict(lengths=torch.zeros(1, dtype=torch.int32)), dict(mask=torch.zeros(1, 1, 2, dtype=torch.bool))):
        with pytest.raises(RuntimeError):
            ops.cross_attention(q, q, q, **bad)
    with pytest.raises(RuntimeError):
        ops.embedding(torch.zeros(3, 4, device=DEV), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        ops.dropout(torch.zeros(4, device=DEV), 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        ops.group_norm_act(torch.zeros(1, 2, 2, 8, device=DEV), 2, torch.ones(8))
