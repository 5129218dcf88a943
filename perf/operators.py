"""The operators of a layout-conditioned attention block, as measured cases.

Four operators that stand in one block of a generator which looks at its layout by attention: the feature map is normalised over channel
groups (group_norm_act), its pixels attend to the states of the objects or words (cross_attention), those states start as rows of a table
(embedding), and the block's result is dropped out and added to the stream (dropout). A case names an operator, a direction ("fwd": the
forward alone, "train": the forward and every gradient), types and sizes. `own` False computes the plain form from elementary operations in
32 bits, `own` True calls the framework.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the first map of the generator (4 x 4 x 1024) when one image is sampled: a launch's latency, not its bandwidth
        dict(name="gn_one_image", op="gn", do="fwd", b=1, h=4, w=4, c=1024, g=32, act="relu", tin="f32", tout="bf16"),
        # a middle block of a training step at batch 32 with operands kept in bf16
        dict(name="gn_train_64", op="gn", do="train", b=32, h=64, w=64, c=128, g=32, act="silu", tin="bf16", tout="bf16"),
        # the last block's stream, the largest map of a training step
        dict(name="gn_train_128_f32", op="gn", do="train", b=32, h=128, w=128, c=64, g=32, act="silu", tin="f32", tout="f32"),
        # one new token for each of 32 sequences against cached states of ragged lengths, four query heads to a cached head
        dict(name="xa_one_token", op="xa", do="fwd", b=32, lq=1, lk=4096, hk=4, gq=4, d=128, ragged=True, mask=False, tin="bf16"),
        # the pixels of a 64 x 64 map attend to the boxes they lie in, 31 slots for a scene-graph layout; background pixels lie in none
        dict(name="xa_boxes_train", op="xa", do="train", b=32, lq=4096, lk=31, hk=4, gq=1, d=32, ragged=False, mask=True, tin="bf16"),
        # the pixels of a 64 x 64 map attend to sentences of ragged lengths
        dict(name="xa_words_train", op="xa", do="train", b=16, lq=4096, lk=512, hk=8, gq=1, d=64, ragged=True, mask=False, tin="bf16"),
        # the same on a small odd map in 32 bits, as a parity run would
        dict(name="xa_small_train_f32", op="xa", do="train", b=8, lq=289, lk=77, hk=2, gq=2, d=40, ragged=True, mask=False, tin="f32"),
        # a long encoder result read by a large map, wide heads shared by four query heads: the matrix rate
        dict(name="xa_long", op="xa", do="fwd", b=4, lq=4096, lk=2048, hk=4, gq=4, d=128, ragged=False, mask=False, tin="bf16"),
        # the label table of the COCO layouts: 32 images of 8 objects, 184 classes, 180 columns
        dict(name="emb_labels_train", op="emb", do="train", n=256, v=184, d=180, skew=False, pad=0, tin="f32", tout="f32"),
        # a vocabulary's table under a step's tokens, as skewed as words are
        dict(name="emb_words_train", op="emb", do="train", n=16384, v=32000, d=1024, skew=True, pad=-1, tin="bf16", tout="bf16"),
        # the object latents of a step (256 rows of 308)
        dict(name="drop_latents", op="drop", do="fwd", n=256 * 308, p=0.1, res=False, tin="f32", tout="f32"),
        # a block's result added to its stream at batch 32
        dict(name="drop_stream_train", op="drop", do="train", n=32 * 64 * 64 * 256, p=0.1, res=True, tin="bf16", tout="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("gn", "gn", "xa", "xa", "xa", "emb", "drop"))
    do = rng.choice(("fwd", "train"))
    if op == "gn":
        g = rng.choice((1, 2, 4, 8, 16, 32))
        c = g * rng.choice((1, 2, 3, 4, 5, 8, 16, 25, 32))
        b, h, w = _log(rng, 1, 32), _log(rng, 1, 128), _log(rng, 1, 128)
        while b * h * w * c > 32 * 128 * 128 * 64:
            b, h = max(1, b // 2), max(1, h // 2)
        while h * w * (c // g) < 32:   # (a handful of values per group: their gradient cancels to nothing)
            h, w = 2 * h, 2 * w
        # (relu's gradient jumps at zero, so that two right computations of it differ there by whole values: forward only)
        act = rng.choice(("none", "silu", "relu")) if do == "fwd" else rng.choice(("none", "silu"))
        tin, tout = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")))
        return dict(op="gn", do=do, b=b, h=h, w=w, c=c, g=g, act=act, tin=tin, tout=tout)
    if op == "xa":
        one = do == "fwd" and rng.random() < 0.4
        # (one state alone has weight 1 and passes no gradient to its query: a training step has a few)
        b, lq, lk = _log(rng, 1, 32), 1 if one else _log(rng, 1, 8192), _log(rng, 1 if do == "fwd" else 8, 4096)
        hk, gq, d = rng.choice((1, 2, 4, 8)), rng.choice((1, 1, 2, 3, 4)), 8 * rng.randint(1, 16)
        most = 4 * 16 * 4096 * 2048 if do == "fwd" else 16 * 8 * 4096 * 512
        while b * hk * gq * lq * lk > most:
            b, lq = max(1, b // 2), max(1, lq // 2)
        tin = rng.choice(("bf16", "bf16", "f32"))
        while tin == "f32" and b * hk * gq * lq * lk * d > 16 * 8 * 4096 * 512 * 8:
            b, lq = max(1, b // 2), max(1, lq // 2)
        return dict(op="xa", do=do, b=b, lq=lq, lk=lk, hk=hk, gq=gq, d=d, ragged=rng.random() < 0.5, mask=rng.random() < 0.3, tin=tin)
    if op == "emb":
        v, d, n = _log(rng, 1, 50000), _log(rng, 1, 1024), _log(rng, 1, 32768)
        while v * d > 32000 * 1024:
            v = max(1, v // 2)
        while n * d > 16384 * 1024:
            n = max(1, n // 2)
        tin, tout = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")))
        return dict(op="emb", do=do, n=n, v=v, d=d, skew=rng.random() < 0.5, pad=rng.choice((-1, 0)), tin=tin, tout=tout)
    tin, tout = rng.choice((("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")))
    return dict(op="drop", do=do, n=_log(rng, 1, 32 * 64 * 64 * 256), p=rng.choice((0.0, 0.1, 0.25, 0.5, 0.9)), res=rng.random() < 0.5, tin=tin, tout=tout)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case, gen):
    """ragged: half to all of the states are there; mean three quarters."""
    lk = case["lk"]
    return torch.randint((lk + 1) // 2, lk + 1, (case["b"],), generator=gen, device=DEV, dtype=torch.int32) if case["ragged"] else None


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    train = case["do"] == "train"
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    tin, tout = TYPES[case["tin"]], TYPES[case.get("tout", case["tin"])]
    leaf = lambda t: t.requires_grad_() if train else t
    st = dict(case)
    if case["op"] == "gn":
        shp = (case["b"], case["h"], case["w"], case["c"])
        st["x"] = leaf((rnd(*shp) * 1.5 + rnd(case["b"], 1, 1, case["c"]) * 0.5 + 0.25).to(tin))   # channels with means of their own
        st["weight"], st["bias"] = leaf(1 + 0.2 * rnd(case["c"])), leaf(0.2 * rnd(case["c"]))
        st["dy"] = rnd(*shp).to(tout) if train else None
    elif case["op"] == "xa":
        b, lq, lk, hk, h, d = case["b"], case["lq"], case["lk"], case["hk"], case["hk"] * case["gq"], case["d"]
        st["q"], st["k"], st["v"] = leaf((1.5 * rnd(b, lq, h, d)).to(tin)), leaf(rnd(b, lk, hk, d).to(tin)), leaf(rnd(b, lk, hk, d).to(tin))
        st["dy"] = rnd(b, lq, h, d).to(tin) if train else None
        st["lengths"] = _lengths(case, gen)
        st["mask"] = None
        if case["mask"]:   # boxes over a unit square that the lq places scan: most places lie in some, a few in none
            x, y = torch.rand(b, lq, 1, generator=gen, device=DEV), torch.rand(b, lq, 1, generator=gen, device=DEV)
            x0, y0 = (0.6 * torch.rand(b, 1, lk, generator=gen, device=DEV) for _ in range(2))
            bw, bh = (0.15 + 0.5 * torch.rand(b, 1, lk, generator=gen, device=DEV) for _ in range(2))
            st["mask"] = (x >= x0) & (x < x0 + bw) & (y >= y0) & (y < y0 + bh)
    elif case["op"] == "emb":
        u = torch.rand(case["n"], generator=gen, device=DEV)
        st["tokens"] = ((u ** 4 if case["skew"] else u) * case["v"]).long().clamp_(max=case["v"] - 1)
        st["weight"] = leaf(rnd(case["v"], case["d"]).to(tin))
        st["scale"] = math.sqrt(case["d"])
        st["dy"] = rnd(case["n"], case["d"]).to(tout) if train else None
    else:
        st["x"] = leaf(rnd(case["n"]).to(tin))
        st["residual"] = leaf(rnd(case["n"]).to(tout)) if case["res"] else None
        st["rng"] = torch.randint(0, 1 << 62, (2,), generator=gen, device=DEV, dtype=torch.int64)   # (seed, offset)
        st["dy"] = rnd(case["n"]).to(tout) if train else None
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"gn": _gn, "xa": _xa, "emb": _emb, "drop": _drop}[state["op"]](state)


def _gn(s):
    x, w, b, dy, g, eps, tout = s["x"], s["weight"], s["bias"], s["dy"], s["g"], 1e-5, TYPES[s["tout"]]
    if own:
        from layout2img_amd import ops
        y = ops.group_norm_act(x, g, w, b, eps=eps, act=None if s["act"] == "none" else s["act"], op_dtype=tout)
        return [y] if dy is None else [y, *torch.autograd.grad(y, (x, w, b), dy)]
    with torch.no_grad():
        n, c = x.shape[0], x.shape[-1]
        xf = x.float().view(n, -1, g, c // g)
        d = xf - xf.mean(dim=(1, 3), keepdim=True)
        rstd = 1 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + eps)
        xh = d * rstd
        wf, bf = w.view(1, 1, g, c // g), b.view(1, 1, g, c // g)
        z = xh * wf + bf
        sig = 1 / (1 + torch.exp(-z))
        y = z if s["act"] == "none" else z * (z > 0) if s["act"] == "relu" else z * sig
        y = y.reshape(x.shape).to(tout)
        if dy is None:
            return [y]
        dz = dy.float().view_as(xf)
        if s["act"] == "silu":
            dz = dz * sig * (1 + z * (1 - sig))
        dxh = dz * wf
        dx = rstd * (dxh - dxh.mean(dim=(1, 3), keepdim=True) - xh * (dxh * xh).mean(dim=(1, 3), keepdim=True))
        return [y, dx.reshape(x.shape).to(x.dtype), (dz * xh).sum(dim=(0, 1)).view(c), dz.sum(dim=(0, 1)).view(c)]


def _live(s):
    """(b, 1 or lq, lk) truth values: which states a query may read; None: all of them."""
    live = s["mask"]
    if s["lengths"] is not None:
        inside = (torch.arange(s["lk"], device=DEV)[None, :] < s["lengths"][:, None])[:, None, :]
        live = inside if live is None else live & inside
    return live


def _xa(s):
    q, k, v, dy = s["q"], s["k"], s["v"], s["dy"]
    if own:
        from layout2img_amd import ops
        y = ops.cross_attention(q, k, v, lengths=s["lengths"], mask=s["mask"])
        return [y] if dy is None else [y, *torch.autograd.grad(y, (q, k, v), dy)]
    with torch.no_grad():
        b, lq, h, d = q.shape
        lk, hk = k.shape[1], k.shape[2]
        scale = 1 / math.sqrt(d)
        # (b, hk, rows, d) with the query heads of a state head's group as further rows; states (b, hk, lk, d) and their transposes
        rows = lambda t: t.float().view(b, lq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
        back = lambda t: t.view(b, hk, h // hk, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, h, d)
        qf, kf, vf = rows(q), k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()
        t = torch.matmul(qf, kf.transpose(2, 3).contiguous()).view(b, hk, h // hk, lq, lk) * scale
        live = _live(s)
        if live is not None:
            t = torch.where(live[:, None, None], t, torch.full_like(t, -float("inf")))
            m = t.amax(dim=-1, keepdim=True)
            e = torch.exp(t - torch.where(m == -float("inf"), torch.zeros_like(m), m))
            p = e / e.sum(dim=-1, keepdim=True).clamp_min(1e-37)   # (a row without a state to read: zeros)
        else:
            e = torch.exp(t - t.amax(dim=-1, keepdim=True))
            p = e / e.sum(dim=-1, keepdim=True)
        p = p.view(b, hk, -1, lk)
        y = back(torch.matmul(p, vf)).to(q.dtype)
        if dy is None:
            return [y]
        g = rows(dy)
        dp = torch.matmul(g, vf.transpose(2, 3).contiguous())
        ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) * scale
        dq = back(torch.matmul(ds, kf)).to(q.dtype)
        dk = torch.matmul(ds.transpose(2, 3).contiguous(), qf).transpose(1, 2).contiguous().to(k.dtype)
        dv = torch.matmul(p.transpose(2, 3).contiguous(), g).transpose(1, 2).contiguous().to(v.dtype)
        return [y, dq, dk, dv]


def _emb(s):
    w, tok, dy, tout = s["weight"], s["tokens"], s["dy"], TYPES[s["tout"]]
    if own:
        from layout2img_amd import ops
        y = ops.embedding(w, tok, scale=s["scale"], padding_idx=s["pad"], op_dtype=tout)
        return [y] if dy is None else [y, *torch.autograd.grad(y, (w,), dy)]
    with torch.no_grad():
        there = (tok != s["pad"]).float()[:, None]   # (rows of the padding token are zeros and have no gradient)
        y = (w[tok].float() * s["scale"] * there).to(tout)
        if dy is None:
            return [y]
        dw = torch.zeros(w.shape, device=DEV).index_add_(0, tok, dy.float() * s["scale"] * there)
        return [y, dw.to(w.dtype)]


def _philox(rng, blocks):
    """Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011): key = seed, counter =
    (block, layer 0, offset): (blocks, 4) words of 32 bits, held in int64, whose products keep their 64 bits."""
    lo = 0xFFFFFFFF
    half = lambda t: (t & lo, (t >> 32) & lo)
    k0, k1 = half(rng[0])
    c2, c3 = (t.expand(blocks) for t in half(rng[1]))
    c0 = torch.arange(blocks, device=rng.device, dtype=torch.int64)
    c1 = torch.zeros_like(c0)
    for r in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & lo) ^ c1 ^ k0, p1 & lo, ((p0 >> 32) & lo) ^ c3 ^ k1, p0 & lo
        k0, k1 = (k0 + 0x9E3779B9) & lo, (k1 + 0xBB67AE85) & lo
    return torch.stack((c0, c1, c2, c3), dim=1)


def _drop(s):
    x, res, dy, p, n, tout = s["x"], s["residual"], s["dy"], s["p"], s["n"], TYPES[s["tout"]]
    if own:
        from layout2img_amd import ops
        y = ops.dropout(x, p, s["rng"], residual=res, op_dtype=tout)
        return [y] if dy is None else [y, *torch.autograd.grad(y, (x,) if res is None else (x, res), dy)]
    with torch.no_grad():
        keep = (_philox(s["rng"], (n + 3) // 4).view(-1)[:n] >= round(p * 2.0 ** 32)).float()
        y = x.float() * keep * (1 / (1 - p))
        y = (y if res is None else y + res.float()).to(tout)
        if dy is None:
            return [y]
        dx = (dy.float() * keep * (1 / (1 - p))).to(x.dtype)
        return [y, dx] if res is None else [y, dx, dy]


# ------------------------------------------------------------------------------------------------ what it has to be
def _exact_gn(case, s):
    x, w, b = (s[k].detach().double().requires_grad_() for k in ("x", "weight", "bias"))
    n, c, g = case["b"], case["c"], case["g"]
    groups = x.view(n, -1, g, c // g).transpose(1, 2).reshape(n, g, -1)
    var, mean = torch.var_mean(groups, dim=2, unbiased=False, keepdim=True)
    z = ((groups - mean) / (var + 1e-5).sqrt()).view(n, g, -1, c // g).transpose(1, 2).reshape(n, -1, c) * w + b
    z = {"none": lambda t: t, "relu": lambda t: t.clamp(min=0), "silu": lambda t: t * torch.sigmoid(t)}[case["act"]](z).view(x.shape)
    return [z.detach()] if case["do"] == "fwd" else [z.detach(), *torch.autograd.grad(z, (x, w, b), s["dy"].double())]


def _exact_xa(case, s):
    b, lq, lk, hk, gq, d = (case[k] for k in ("b", "lq", "lk", "hk", "gq", "d"))
    train = case["do"] == "train"
    outs = [torch.zeros(s[k].shape, dtype=torch.float64, device=DEV) for k in (("q", "q", "k", "v") if train else ("q",))]
    for i in range(b):
        n = lk if s["lengths"] is None else int(s["lengths"][i])
        for j in range(hk):
            heads = slice(j * gq, (j + 1) * gq)
            q = s["q"][i, :, heads].detach().double().reshape(lq * gq, d).requires_grad_()
            k, v = (s[t][i, :n, j].detach().double().contiguous().requires_grad_() for t in ("k", "v"))
            t = (q @ k.t()).view(lq, gq, n) * d ** -0.5
            if s["mask"] is not None:
                on = s["mask"][i, :, None, :n]
                t = t.masked_fill(~on, -1e300)
                e = torch.exp(t - t.max(dim=2, keepdim=True).values.detach()) * on
                p = e / e.sum(dim=2, keepdim=True).clamp(min=1e-300)
            else:
                p = torch.softmax(t, dim=2)
            y = p.reshape(lq * gq, n) @ v
            outs[0][i, :, heads] = y.detach().view(lq, gq, d)
            if train:
                dq, dk, dv = torch.autograd.grad(y, (q, k, v), s["dy"][i, :, heads].double().reshape(lq * gq, d))
                outs[1][i, :, heads], outs[2][i, :n, j], outs[3][i, :n, j] = dq.view(lq, gq, d), dk, dv
    return outs


def _exact_emb(case, s):
    tok, w = s["tokens"].cpu().numpy(), s["weight"].detach().double().cpu().numpy()
    there = np.flatnonzero(tok != case["pad"])
    y = np.zeros((case["n"], case["d"]))
    y[there] = w[tok[there]] * math.sqrt(case["d"])
    if case["do"] == "fwd":
        return [y]
    dw = np.zeros_like(w)
    order = there[np.argsort(tok[there], kind="stable")]
    if len(order):
        first = np.flatnonzero(np.r_[True, np.diff(tok[order]) > 0])
        dw[tok[order[first]]] = np.add.reduceat(s["dy"].double().cpu().numpy()[order] * math.sqrt(case["d"]), first, axis=0)
    return [y, dw]


def _exact_drop(case, s):
    n, p = case["n"], case["p"]
    seed, off = (int(t) for t in s["rng"].tolist())
    m = np.uint64(0xFFFFFFFF)
    sh = np.uint64(32)
    a = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [a, np.zeros_like(a), np.full_like(a, off & 0xFFFFFFFF), np.full_like(a, off >> 32)]
    for r in range(10):
        key = [np.uint64((seed + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
        x, y = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(y >> sh) ^ c[1] ^ key[0], y & m, (x >> sh) ^ c[3] ^ key[1], x & m]
    keep = torch.from_numpy(np.stack(c, axis=1).reshape(-1)[:n] >= np.uint64(round(p * 2 ** 32))).to(DEV)
    y = torch.where(keep, s["x"].detach().double() / (1 - p), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].detach().double()
    if case["do"] == "fwd":
        return [y]
    dy = s["dy"].double()
    dx = torch.where(keep, dy / (1 - p), 0.0)
    return [y, dx] if s["residual"] is None else [y, dx, dy]


def exact(case, seed):
    s = prepare(case, seed)
    return {"gn": _exact_gn, "xa": _exact_xa, "emb": _exact_emb, "drop": _exact_drop}[case["op"]](case, s)


def work(case):
    size = {"f32": 4, "bf16": 2}
    i, o = size[case["tin"]], size[case.get("tout", case["tin"])]
    train = case["do"] == "train"
    if case["op"] == "gn":
        n = case["b"] * case["h"] * case["w"] * case["c"]
        return {"bytes": n * (i + o) * (2 if train else 1) + case["c"] * (16 if train else 8), "flops": n * (24 if train else 10)}
    if case["op"] == "xa":
        live = case["lk"] * (0.75 if case["ragged"] else 1.0)
        nq = case["b"] * case["lq"] * case["hk"] * case["gq"] * case["d"]
        nk = case["b"] * case["hk"] * case["d"]
        mask = case["b"] * case["lq"] * live if case["mask"] else 0
        # forward: q, k, v -> y; training: also dy -> dq, dk, dv (whole, with the zeros behind a sequence's end)
        return {"bytes": i * (2 * nq + 2 * nk * live) + mask + (i * (2 * nq + 2 * nk * case["lk"]) if train else 0), "flops": nq * live * (14 if train else 4)}
    if case["op"] == "emb":
        n = case["n"] * case["d"]
        rows = min(case["n"], case["v"]) * case["d"]
        return {"bytes": rows * i + n * o + 8 * case["n"] + (n * o + case["v"] * case["d"] * i if train else 0), "flops": n * (2 if train else 1)}
    n = case["n"]
    return {"bytes": n * (i + o + (o if case["res"] else 0)) + (n * (i + o) if train else 0), "flops": n * 3}
