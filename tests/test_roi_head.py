"""The RoI head's operators against their definitions in 64 bits: attention over an image's boxes (forward, backward), rotary
positions over several axes, log probabilities of labels.

Tolerances.  One rounding to a type moves a value by at most half a step, u = 2^-8 of it in bf16, 2^-11 in fp16, 2^-24 in fp32.
Attention in bf16: p (and ds) is rounded once as an operand, the result once at the end, so an output element is off by at most
u sum |p_ij v_j| + u |o_i|, and the sum itself is held in 32 bits; delta is formed from the rounded out (u |do| |out| per row).
(Without the forward's rest, that is; with it delta is off by 2^-16 of its terms.)
Each bound below is such a sum of magnitudes, formed in 64 bits from the same inputs, plus the 32-bit terms: a product of d
terms is off by at most d 2^-24 sum |q k| scale, which moves p by that factor."""
import math

import numpy as np
import pytest
import torch

# A value below a type's smallest normal one, 2^-14 in fp16 and 2^-126 in the others, stands among values 2^-24 (2^-133, 2^-149)
# apart: its rounding is off by half of that, 2^-25 (2^-134, 2^-150), however small it is.  Flushed to 0 in 32 bits: 2^-126.
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
E32 = 2.0 ** -24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _attn64(q, k, v, qc, kc, mask, scale, do=None):
    """definition in 64 bits on the CPU, with the bounds of the module's text: dict of (value, bound)"""
    u = 2.0 ** -24 if q.dtype == torch.float32 else 2.0 ** -8
    B, Nq, Hq, D = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)     # noqa: E731
    out, lse, dq, dk, dv = z(B, Nq, Hq, D), torch.full((B, Hq, Nq), -math.inf, dtype=torch.float64), z(B, Nq, Hq, D), z(B, Nk, Hk, D), z(B, Nk, Hk, D)
    tout, tlse, tdq, tdk, tdv = z(B, Nq, Hq, D), z(B, Hq, Nq), z(B, Nq, Hq, D), z(B, Nk, Hk, D), z(B, Nk, Hk, D)
    for b in range(B):
        n = Nq if qc is None else min(max(int(qc[b]), 0), Nq)
        m = Nk if kc is None else min(max(int(kc[b]), 0), Nk)
        see = torch.ones(n, m, dtype=torch.bool) if mask is None else mask[b if mask.shape[0] > 1 else 0, :n, :m].bool()
        for h in range(Hq):
            j = h // (Hq // Hk)
            Q, K, V = q[b, :n, h].double(), k[b, :m, j].double(), v[b, :m, j].double()
            s = (Q @ K.T) * scale
            s = torch.where(see, s, torch.full_like(s, -math.inf))
            L = torch.logsumexp(s, 1) if m else torch.full((n,), -math.inf, dtype=torch.float64)
            p = torch.where(see, torch.exp(s - torch.where(torch.isinf(L), torch.zeros_like(L), L)[:, None]), torch.zeros_like(s))
            # relative error of a probability in 32 bits: the product's, the exponent's argument and its statistic, the exponential
            ep = (D + 4) * E32 * (Q.abs() @ K.abs().T) * scale + 8 * E32 * (1 + torch.where(torch.isinf(L), torch.zeros_like(L), L.abs())[:, None]) + \
                8 * E32 * torch.where(see, s.abs(), torch.zeros_like(s)) + m * E32
            o = p @ V
            out[b, :n, h], lse[b, h, :n] = o, L
            eo = (p * (2 * ep + u)) @ V.abs() + u * o.abs()
            tout[b, :n, h] = eo
            tlse[b, h, :n] = torch.where(torch.isinf(L), torch.zeros_like(L), (p * ep).sum(1) + 4 * E32 * (1 + L.abs()))
            if do is not None:
                G = do[b, :n, h].double()
                dp = G @ V.T
                delta = (G * o).sum(1, keepdim=True)
                edp = (D + 4) * E32 * (G.abs() @ V.abs().T) + (G.abs() * eo).sum(1, keepdim=True) + (D + 4) * E32 * (G.abs() * o.abs()).sum(1, keepdim=True)
                ds = p * (dp - delta)
                eds = ds.abs() * (2 * ep + u + 2 * E32) + p * edp
                dv[b, :m, j] += p.T @ G
                tdv[b, :m, j] += (p * (2 * ep + u + n * E32)).T @ G.abs()
                dq[b, :n, h] = ds @ K * scale
                tdq[b, :n, h] = (eds + m * E32 * ds.abs()) @ K.abs() * scale + u * (ds @ K * scale).abs()
                dk[b, :m, j] += ds.T @ Q * scale
                tdk[b, :m, j] += (eds + n * (Hq // Hk) * E32 * ds.abs()).T @ Q.abs() * scale
    tdk += u * dk.abs()
    tdv += u * dv.abs()
    r = dict(out=(out, tout), lse=(lse, tlse))
    if do is not None:
        r.update(dq=(dq, tdq), dk=(dk, tdk), dv=(dv, tdv))
    return r


def _close(got, want, what):
    w, tol = want
    g = got.detach().cpu().double()
    assert g.shape == w.shape, what
    same = (g == w) | (torch.isnan(g) & torch.isnan(w))
    off = torch.where(same, torch.zeros_like(w), (g - w).abs() - (tol + 1e-30))
    assert not torch.isnan(off).any(), (what, "NaN")
    assert float(off.max() if off.numel() else 0.0) <= 0.0, (what, float(off.max()), int((off > 0).sum()), float((g - w).abs().max()))


def _attn_inputs(seed, B, Nq, Nk, Hq, Hk, D, dtype):
    g = _gen(seed)
    q, k, v, do = (torch.randn(s, generator=g).to(dtype) for s in ((B, Nq, Hq, D), (B, Nk, Hk, D), (B, Nk, Hk, D), (B, Nq, Hq, D)))
    return q, k, v, do


ATTN_CASES = [
    # B, Nq, Nk, Hq, Hk, D, counts, mask
    (1, 1, 1, 1, 1, 8, False, None),
    (1, 1, 5000, 8, 2, 128, False, None),        # one query, split over the keys
    (2, 1, 700, 4, 4, 64, True, None),
    (1, 3, 1, 2, 1, 32, False, None),
    (2, 33, 65, 2, 2, 40, False, None),
    (1, 128, 64, 1, 1, 64, False, None),
    (2, 129, 127, 6, 2, 64, True, None),
    (3, 98, 98, 4, 4, 32, True, "pairs"),
    (2, 200, 257, 4, 1, 128, True, "pairs"),
    (1, 5000, 40, 2, 2, 64, False, None),        # few keys, many rows: dk, dv split over the rows
    (1, 700, 900, 2, 2, 72, False, "shared"),
    (2, 64, 100, 2, 1, 104, True, "none"),       # a mask that leaves every row empty
    (1, 90, 700, 2, 1, 24, False, None),         # more keys than those for which ds is cut in two
    (4, 50, 50, 3, 3, 16, "zero", None),         # images with no rows or no keys at all
]


def _attn_masks(case, seed):
    B, Nq, Nk, Hq, Hk, D, counts, mask = case
    g = _gen(seed + 1)
    qc = kc = None
    if counts:
        qc, kc = torch.randint(0, Nq + 1, (B,), generator=g).int(), torch.randint(0, Nk + 1, (B,), generator=g).int()
        qc[0], kc[0] = max(1, Nq - 1), max(1, Nk - 1)
        if counts == "zero":
            qc[1], kc[2], kc[3] = 0, 0, Nk + 5
        else:
            qc[-1] = max(1, int(qc[-1]))
    m = None
    if mask == "pairs":
        m = (torch.rand((B, Nq, Nk), generator=g) < 0.3) & (torch.rand((B, Nq, 1), generator=g) > 0.1)
    elif mask == "shared":
        m = (torch.rand((1, Nq, Nk), generator=g) < 0.5)
    elif mask == "none":
        m = torch.zeros((B, Nq, Nk), dtype=torch.bool)
    return qc, kc, m


def _dev(t):
    return None if t is None else t.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", ATTN_CASES, ids=lambda c: "x".join(map(str, c)))
def test_roi_attention(case, dtype):
    from vision_amd import ops
    q, k, v, do = _attn_inputs(7, *case[:6], dtype)
    qc, kc, m = _attn_masks(case, 7)
    want = _attn64(q, k, v, qc, kc, m, None, do)
    if qc is not None:                           # what lies behind a count is never read
        for b in range(case[0]):
            q[b, max(int(qc[b]), 0):] = math.nan
            do[b, max(int(qc[b]), 0):] = math.inf
            k[b, max(int(kc[b]), 0):] = math.nan
            v[b, max(int(kc[b]), 0):] = math.inf
    Q, K, V, G, QC, KC, M = map(_dev, (q, k, v, do, qc, kc, m))
    out, lse = ops.roi_attention(Q, K, V, QC, KC, M)
    _close(out, want["out"], "out")
    _close(lse, want["lse"], "lse")
    dq, dk, dv = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M)
    _close(dq, want["dq"], "dq")
    _close(dk, want["dk"], "dk")
    _close(dv, want["dv"], "dv")
    out2, lse2 = ops.roi_attention(Q, K, V, QC, KC, M)             # the same bits in every run
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    again = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M)
    assert all(torch.equal(x, y) for x, y in zip((dq, dk, dv), again))
    only_q = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M, need_kv=False)
    only_kv = ops.roi_attention_backward(G, Q, K, V, out, lse, QC, KC, M, need_q=False)
    assert torch.equal(only_q[0], dq) and only_q[1] is None and only_kv[0] is None
    assert torch.equal(only_kv[1], dk) and torch.equal(only_kv[2], dv)


# ------------------------------------------------------------------ rotary positions
def _rope64(x, pos, sections, theta, ladder, pairing, inverse=False):
    """definition in 64 bits: (value, bound).  The bound: one rounding to the type, and in 32 bits sine and cosine (2 units),
    their arguments (half a unit of pi) and two products and a sum."""
    u = U[x.dtype]
    n = sum(sections)
    freq, axis = [], []
    for a, m in enumerate(sections):
        for i in range(m):
            freq.append(theta ** -(i / m if ladder == "axis" else len(freq) / n))
            axis.append(a)
    ang = pos.double()[..., axis] * torch.tensor(freq, dtype=torch.float64)
    ang = (ang if ang.dim() == 3 else ang[None])[:, :, None]
    c, s = torch.cos(ang), torch.sin(ang) * (-1 if inverse else 1)
    X = x.double()
    i, j = (slice(0, n), slice(n, 2 * n)) if pairing == "halves" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    want, tol = X.clone(), torch.zeros_like(X)
    p, q = X[..., i], X[..., j]
    want[..., i], want[..., j] = p * c - q * s, p * s + q * c
    # the 64-bit angles themselves, here and in the kernel, are off by a few units of 2^-53 of their size
    tol[..., i] = tol[..., j] = (p.abs() + q.abs()) * (8 * E32 + 8 * 2.0 ** -53 * ang.abs())
    return want, tol + u * want.abs() + TINY[x.dtype]


ROPE_CASES = [
    # B, N, Hq, Hk, D, sections, ladder, pairing, pos type
    (1, 1, 1, 1, 2, (1,), "axis", "halves", torch.float32),
    (2, 37, 3, 1, 64, (16, 16), "axis", "halves", torch.float32),
    (2, 37, 4, 2, 64, (8, 12, 12), "shared", "halves", torch.float64),
    (1, 130, 2, 2, 80, (16, 16), "axis", "neighbours", torch.float32),
    (3, 19, 5, 1, 22, (3, 4), "axis", "neighbours", torch.int64),       # odd cuts: one pair at a time
    (3, 19, 5, 1, 22, (3, 4), "axis", "halves", torch.float32),
    (1, 1000, 8, 8, 128, (16, 24, 24), "axis", "halves", torch.float32),
    (2, 5, 2, 0, 32, (0, 16), "axis", "halves", torch.float32),
    (2, 16, 4, 2, 64, (8, 8), "axis", "neighbours", torch.float64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", ROPE_CASES, ids=lambda c: "x".join(map(str, c)))
def test_rope_axes(case, dtype):
    from vision_amd import ops
    B, N, Hq, Hk, D, sections, ladder, pairing, pt = case
    g = _gen(3)
    q, k = torch.randn((B, N, Hq, D), generator=g).to(dtype), torch.randn((B, N, Hk, D), generator=g).to(dtype)
    pos = torch.rand((B, N, len(sections)), generator=g, dtype=torch.float64) * 1900
    pos[:, ::3] += 1e6                           # far positions
    pos = pos.to(pt)
    plan = ops.rope_plan(sections, 10000.0, ladder, pairing)
    for inverse in (False, True):
        a, b = ops.rope_axes(q.cuda(), pos.cuda(), plan, k=k.cuda(), inverse=inverse)
        _close(a, _rope64(q, pos, sections, 10000.0, ladder, pairing, inverse), "q")
        _close(b, _rope64(k, pos, sections, 10000.0, ladder, pairing, inverse), "k")
    alone = ops.rope_axes(q.cuda(), pos[0].cuda(), plan)                # one set of positions for all images
    _close(alone, _rope64(q, pos[0], sections, 10000.0, ladder, pairing), "shared positions")
    big = torch.randn((B, N, 2, Hq + 1, D + 1), generator=g).to(dtype).cuda()      # strided, not aligned
    view = big[:, :, 1, 1:, :D]
    _close(ops.rope_axes(view, pos.cuda(), plan), _rope64(view.cpu(), pos, sections, 10000.0, ladder, pairing), "strided")
    t = torch.randn((B, Hq, N, D), generator=g).to(dtype).cuda().transpose(1, 2)
    _close(ops.rope_axes(t, pos.cuda(), plan), _rope64(t.cpu(), pos, sections, 10000.0, ladder, pairing), "heads first")


# ------------------------------------------------------------------ log probabilities
def _logp64(z, y, top, g=None, gh=None):
    """definition in 64 bits on the CPU: dict of (value, bound), and the indexes.  In 32 bits: a difference to the maximum is off
    by one rounding of itself, its exponential by that and two units, a sum of c terms by c / 64 + 64 units (lanes of 64 or more
    add their own), the logarithm by one and two roundings at the end."""
    n, c = z.shape
    Z = z.double()
    m = Z.amax(1, keepdim=True)
    dead = torch.isinf(m[:, 0]) & (m[:, 0] < 0)
    m0 = torch.where(dead[:, None], torch.zeros_like(m), m)
    d = Z - m0
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    ls = torch.where(dead[:, None], torch.zeros_like(s), torch.log(torch.where(dead[:, None], torch.ones_like(s), s)))
    lp = torch.where(dead[:, None], torch.full_like(d, -math.inf), d - ls)
    p = torch.where(dead[:, None], torch.zeros_like(e), e / torch.where(dead[:, None], torch.ones_like(s), s))
    dd = torch.where(torch.isinf(d), torch.zeros_like(d), d.abs())
    terms = c / 64 + 64
    es = (p * (2 * dd + 4) * E32).sum(1, keepdim=True) + terms * E32                 # relative error of the sum, and of log s
    elp = torch.where(torch.isinf(lp), torch.zeros_like(lp), 2 * E32 * (dd + ls.abs() + lp.abs()) + es)
    pl = torch.where(p > 0, p * torch.where(torch.isinf(lp), torch.zeros_like(lp), lp), torch.zeros_like(p))
    H = -pl.sum(1)
    eH = (p * dd * ((2 * dd + 4) * E32 + terms * E32)).sum(1) + (1 + (p * dd).sum(1)) * es[:, 0] + 4 * E32 * (ls[:, 0].abs() + (p * dd).sum(1))
    known = (y >= 0) & (y < c)
    yy = torch.where(known, y, torch.zeros_like(y))[:, None]
    logp = torch.where(known, lp.gather(1, yy)[:, 0], torch.where(y < 0, 0.0, math.nan).double())
    elogp = torch.where(known, elp.gather(1, yy)[:, 0], torch.zeros_like(H))
    index = torch.sort(Z + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    r = dict(logp=(logp, elogp), entropy=(H, eH), best=(lp.gather(1, index), elp.gather(1, index)), index=index)
    if g is not None:
        G = torch.where(known, g.double(), torch.zeros_like(H))
        GH = gh.double()[:, None]
        t = torch.where(p > 0, lp, torch.zeros_like(lp)) + H[:, None]
        dz = -p * (G[:, None] + GH * t)
        at = torch.where(known & ~dead, G, torch.zeros_like(G))
        dz.scatter_add_(1, yy, at[:, None])
        dz[y >= c] = math.nan
        edz = p * (elp + 4 * E32) * (G.abs()[:, None] + GH.abs() * t.abs()) + p * GH.abs() * (elp + eH[:, None] + 2 * E32 * t.abs()) + \
            2 * E32 * (p * G.abs()[:, None] + (at[:, None].abs()))
        r["dz"] = (dz, torch.where(torch.isnan(dz), torch.zeros_like(dz), edz + U[z.dtype] * dz.abs() + TINY[z.dtype]))
    return r


LOGP_CASES = [(1, 1, 1), (1, 2, 2), (5, 21, 3), (300, 81, 5), (20, 200, 6), (257, 33, 32), (64, 512, 8), (33, 513, 8), (7, 1000, 32), (40, 4096, 4), (3, 4097, 8),
              (2, 20011, 5), (1, 131072, 8), (600, 5003, 1), (1, 70001, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,c,top", LOGP_CASES)
def test_class_logprobs(n, c, top, dtype):
    from vision_amd import ops
    rng = _gen(n + c)
    z = (torch.randn((n, c), generator=rng) * 3).to(dtype)
    if c > 2:
        z[torch.rand((n, c), generator=rng) < 0.1] = -math.inf            # masked classes
        z[:, 0] = 0.5
    if n > 4:
        z[1] = -math.inf                         # nothing to choose from
        z[2] = torch.finfo(dtype).min            # masked by the type's lowest value throughout: equal odds
        z[3] = torch.finfo(dtype).min
        z[3, c // 2] = 1.0
        z[4] = z[4].clamp(min=-1) * 0 + 2.0      # all equal: the lowest indexes
    y = torch.randint(0, c, (n,), generator=rng)
    if n > 6:
        y[5], y[6] = -1, c
    g, gh = torch.randn((n,), generator=rng), torch.randn((n,), generator=rng)
    want = _logp64(z, y, top, g, gh)
    Z, Y = z.cuda(), y.cuda()
    logp, entropy, norm, best, index = ops.class_logprobs(Z, Y, top)
    _close(logp, want["logp"], "logp")
    _close(entropy, want["entropy"], "entropy")
    _close(best, want["best"], "best")
    assert torch.equal(index.cpu(), want["index"])
    dz = ops.class_logprobs_backward(g.cuda(), gh.cuda(), Z, Y, norm, entropy)
    _close(dz, want["dz"], "dz")
    again = ops.class_logprobs(Z, Y, top)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip((logp, entropy, norm, best, index), again))
    wide = torch.zeros((n, c + 3), dtype=dtype, device="cuda")            # rows apart, not aligned
    wide[:, 1:c + 1] = Z
    strided = ops.class_logprobs(wide[:, 1:c + 1], Y, top)
    _close(strided[0], want["logp"], "strided logp")
    assert torch.equal(strided[4].cpu(), want["index"])
    _close(ops.class_logprobs_backward(g.cuda(), None, wide[:, 1:c + 1], Y, strided[2], strided[1]),
           _logp64(z, y, 0, g, torch.zeros_like(gh))["dz"], "dz of logp alone")
    none = ops.class_logprobs(Z, None, top)
    assert none[0] is None and torch.equal(none[4], index) and torch.equal(none[1].nan_to_num(7.0), entropy.nan_to_num(7.0))


# ------------------------------------------------------------------ layouts, offsets, streams, graphs
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_roi_attention_layouts(dtype):
    """Heads first, one fused buffer of q, k and v, odd offsets (copied), expanded batches: the bits of the dense call."""
    from vision_amd import ops
    B, N, H, D = 2, 77, 4, 64
    q, k, v, do = (t.cuda() for t in _attn_inputs(11, B, N, N, H, H, D, dtype))
    out, lse = ops.roi_attention(q, k, v)
    grads = ops.roi_attention_backward(do, q, k, v, out, lse)
    views = []
    views.append([t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)])
    fused = torch.stack([q, k, v, do], 2)
    views.append([fused[:, :, i] for i in range(4)])
    odd = [torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v, do)]
    views.append(odd)
    wide = [torch.zeros((B, N, H, D + 3), dtype=dtype, device="cuda") for _ in range(4)]
    for w, t in zip(wide, (q, k, v, do)):
        w[..., :D] = t
    views.append([w[..., :D] for w in wide])
    for a, b, c, g in views:
        o, s = ops.roi_attention(a, b, c)
        assert torch.equal(o, out) and torch.equal(s, lse)
        assert all(torch.equal(x, y) for x, y in zip(ops.roi_attention_backward(g, a, b, c, out, lse), grads))
    o, _ = ops.roi_attention(q, k[:1].expand(B, N, H, D), v[:1].expand(B, N, H, D))
    o2, _ = ops.roi_attention(q, k[:1].repeat(B, 1, 1, 1), v[:1].repeat(B, 1, 1, 1))
    assert torch.equal(o, o2)
    one = do[:, :, :, :1].expand(B, N, H, D)                              # what sum().backward() hands over
    assert all(torch.equal(x, y) for x, y in zip(ops.roi_attention_backward(one, q, k, v, out, lse),
                                                 ops.roi_attention_backward(one.contiguous(), q, k, v, out, lse)))


@pytest.mark.gpu
def test_roi_attention_far_rows():
    """Keys and values whose rows lie so far apart that offsets pass 2^32 bytes and 2^31 values; one more stride and the call
    goes by a copy."""
    from vision_amd import ops
    q, k, v, do = (t.cuda() for t in _attn_inputs(12, 1, 5, 520, 1, 1, 64, torch.bfloat16))
    out, lse = ops.roi_attention(q, k, v)
    want = ops.roi_attention_backward(do, q, k, v, out, lse)
    for step in (1 << 22, (1 << 22) + 8):
        big = torch.empty((2, 520, step), dtype=torch.bfloat16, device="cuda")
        K, V = big[0, None, :, None, :64], big[1, None, :, None, :64]
        K.copy_(k)
        V.copy_(v)
        o, s = ops.roi_attention(q, K, V)
        assert torch.equal(o, out) and torch.equal(s, lse)
        assert all(torch.equal(x, y) for x, y in zip(ops.roi_attention_backward(do, q, K, V, out, lse), want))
        del big, K, V


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_roi_attention_nan_behind_mask(dtype):
    """What a mask hides from a row does not reach it, whatever it holds; what a row does see and is not finite makes it NaN."""
    from vision_amd import ops
    B, N, M, H, D = 1, 70, 90, 2, 64
    q, k, v, do = _attn_inputs(13, B, N, M, H, H, D, dtype)
    g = _gen(14)
    mask = torch.rand((B, N, M), generator=g) < 0.5
    bad_keys, bad_rows = [3, 40, 88], [7, 33]
    mask[:, :35, bad_keys] = False               # the first half sees none of them
    mask[:, 35:, bad_keys[0]] = True
    clean = mask.clone()
    clean[:, 35:] = False                        # the rows that stay finite, for the reference
    clean[:, bad_rows] = False
    K, V, Q, G = k.clone(), v.clone(), q.clone(), do.clone()
    K[:, 3, 0, 5], V[:, 3, 1, 6] = math.nan, math.inf
    K[:, 40] = math.inf
    V[:, 88] = math.nan
    Q[:, 7] = math.nan
    G[:, 33, :, 2] = math.inf
    want = _attn64(q, k, v, None, None, mask, None, do)
    Qc, Kc, Vc, Gc, Mc = map(_dev, (Q, K, V, G, mask))
    out, lse = ops.roi_attention(Qc, Kc, Vc, mask=Mc)
    rows = [i for i in range(35) if i != 7]
    _close(out[:, rows], tuple(t[:, rows] for t in want["out"]), "rows that see no bad key")
    assert torch.isnan(out[:, 7]).all() and torch.isnan(out[:, 35:]).all()
    dq, dk, dv = ops.roi_attention_backward(Gc, Qc, Kc, Vc, out, lse, mask=Mc)
    rows = [i for i in rows if i != 33]
    _close(dq[:, rows], tuple(t[:, rows] for t in want["dq"]), "dq of those rows")
    # keys that only good rows see
    seen_bad = mask[0, 35:].any(0) | mask[0, bad_rows].any(0)
    good = [j for j in range(M) if not bool(seen_bad[j])]
    mask[:, :, :5] = mask[:, :, :5]
    only = torch.zeros_like(mask)
    only[:, rows] = mask[:, rows]
    ref = _attn64(q, k, v, None, None, only, None, do)
    if good:
        _close(dk[:, good], tuple(t[:, good] for t in ref["dk"]), "dk")
        _close(dv[:, good], tuple(t[:, good] for t in ref["dv"]), "dv")
    # the same with every later row masked off for every key: all good rows' gradients, none of the bad ones'
    Mc[:, 35:] = False
    Mc[:, bad_rows] = False
    out, lse = ops.roi_attention(Qc, Kc, Vc, mask=Mc)
    dq, dk, dv = ops.roi_attention_backward(Gc, Qc, Kc, Vc, out, lse, mask=Mc)
    keys = [j for j in range(M) if j not in bad_keys]
    _close(dk[:, keys], tuple(t[:, keys] for t in ref["dk"]), "dk, bad rows off")
    _close(dv, ref["dv"], "dv, bad rows off")
    assert float(dk[:, bad_keys].abs().max()) == 0.0 and float(dq[:, bad_rows].abs().max()) == 0.0 and float(out[:, bad_rows].abs().max()) == 0.0


@pytest.mark.gpu
def test_roi_attention_scale_and_large_scores():
    """Scores far apart and far from zero: the running maximum follows, nothing overflows; a scale of one's own."""
    from vision_amd import ops
    q, k, v, do = _attn_inputs(15, 1, 40, 300, 1, 1, 32, torch.float32)
    k = k * torch.linspace(0.1, 30.0, 300)[None, :, None, None]          # the largest scores come last
    for scale in (None, 1.0, 1e-3):
        want = _attn64(q, k, v, None, None, None, scale, do)
        out, lse = ops.roi_attention(q.cuda(), k.cuda(), v.cuda(), scale=scale)
        _close(out, want["out"], "out")
        _close(lse, want["lse"], "lse")
        for n, g in zip(("dq", "dk", "dv"), ops.roi_attention_backward(do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, scale=scale)):
            _close(g, want[n], n)


@pytest.mark.gpu
def test_streams_and_graphs():
    """Every operator on a stream of its own, and captured into two graphs that are replayed in turn with eager work between."""
    from vision_amd import ops
    g = _gen(16)
    B, N, H, D, C = 2, 150, 4, 64, 1000
    plan = ops.rope_plan((16, 16))
    ins = [[torch.randn((B, N, H, D), generator=g).bfloat16().cuda() for _ in range(4)] + [torch.rand((B, N, 2), generator=g).cuda() * 40,
           torch.tensor([N, N - 40 - i]).int().cuda(), torch.randn((B * N, C), generator=g).cuda(), torch.randint(0, C, (B * N,), generator=g).cuda(),
           torch.rand((B, N, N), generator=g).cuda() < 0.5] for i in range(2)]

    def work(q, k, v, do, pos, counts, z, y, mask):
        a, b = ops.rope_axes(q, pos, plan, k=k)
        out, lse = ops.roi_attention(a, b, v, counts, counts, mask)
        grads = ops.roi_attention_backward(do, a, b, v, out, lse, counts, counts, mask)
        logp, h, norm, best, index = ops.class_logprobs(z, y, 5)
        dz = ops.class_logprobs_backward(logp, h, z, y, norm, h)
        return [a, b, out, lse, *grads, logp, h, best, index, dz]

    eager = [[t.clone() for t in work(*i)] for i in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = work(*ins[0])
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(on_side, eager[0]))
    graphs, outs = [], []
    for i in ins:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(work(*i))
        graphs.append(gr)
    for r in range(3):
        for i in (0, 1):
            for t in outs[i]:
                t.zero_()
            graphs[i].replay()
            work(*ins[1 - i])                    # eager work between
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(outs[i], eager[i])), (r, i)
    graphs[0].replay()                           # both at once, on two streams
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for i in (0, 1) for x, y in zip(outs[i], eager[i]))


# ------------------------------------------------------------------ gradients through autograd
def _slope(f, xs, ds, h=1e-6):
    """central difference of a 64-bit function along ds"""
    up, down = f(*[x + h * d for x, d in zip(xs, ds)]), f(*[x - h * d for x, d in zip(xs, ds)])
    return float((up - down) / (2 * h))


@pytest.mark.gpu
def test_roi_attention_gradient_against_differences():
    """The gradient's product with a direction against the difference quotient of the 64-bit definition.  The quotient's own error
    is h^2 / 6 times a third derivative plus 2^-52 |f| / h: below 1e-6 of the sum of magnitudes here; the rest is the bound of
    each gradient's elements."""
    from vision_amd import fast_rcnn
    B, N, M, H, Hk, D = 2, 20, 30, 4, 2, 16
    q, k, v, do = _attn_inputs(21, B, N, M, H, Hk, D, torch.float32)
    mask = torch.rand((B, N, M), generator=_gen(22)) < 0.6
    qc, kc = torch.tensor([20, 11]), torch.tensor([30, 25])
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    out = fast_rcnn.roi_attention(*leaves, q_counts=qc, k_counts=kc, mask=mask)
    assert out.is_cuda and out.requires_grad
    grads = torch.autograd.grad(out, leaves, do.cuda())
    want = _attn64(q, k, v, qc, kc, mask, None, do)
    f = lambda a, b, c: (_attn64(a, b, c, qc, kc, mask, None)["out"][0] * do.double()).sum()    # noqa: E731
    g = _gen(23)
    for i, name in enumerate(("dq", "dk", "dv")):
        _close(grads[i], want[name], name)
        d = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v)]
        d[i] = torch.randn(d[i].shape, generator=g, dtype=torch.float64)
        slope, mine = _slope(f, (q.double(), k.double(), v.double()), d), float((grads[i].cpu().double() * d[i]).sum())
        size = float((want[name][0].abs() * d[i].abs()).sum())
        assert abs(slope - mine) <= float((want[name][1] * d[i].abs()).sum()) + 1e-6 * size, name
    cpu = [t.clone().requires_grad_(True) for t in (q, k, v)]              # tensors on the CPU go in and come back
    o = fast_rcnn.roi_attention(*cpu, q_counts=qc, k_counts=kc, mask=mask)
    assert not o.is_cuda and torch.equal(o, out.detach().cpu())
    (o * do).sum().backward()
    assert all(torch.equal(t.grad, x.cpu()) for t, x in zip(cpu, grads))
    only_v = v.cuda().requires_grad_(True)
    (dv,) = torch.autograd.grad(fast_rcnn.roi_attention(q.cuda(), k.cuda(), only_v, qc, kc, mask), (only_v,), do.cuda())
    assert torch.equal(dv, grads[2])


@pytest.mark.gpu
def test_rope_and_logprobs_gradient():
    from vision_amd import fast_rcnn, ops
    g = _gen(31)
    q, k = torch.randn((2, 9, 3, 32), generator=g).cuda().requires_grad_(True), torch.randn((2, 9, 1, 32), generator=g).cuda().requires_grad_(True)
    pos = torch.rand((2, 9, 3), generator=g).cuda() * 50
    plan = ops.rope_plan((4, 6, 6))
    a, b = fast_rcnn.rope_axes(q, k, pos, plan)
    da, db = torch.randn(a.shape, generator=g).cuda().requires_grad_(True), torch.randn(b.shape, generator=g).cuda()
    dq, dk = torch.autograd.grad((a, b), (q, k), (da, db), create_graph=True)
    assert torch.equal(dq.detach(), ops.rope_axes(da.detach(), pos, plan, inverse=True)) and torch.equal(dk.detach(), ops.rope_axes(db, pos, plan, inverse=True))
    (twice,) = torch.autograd.grad(dq, (da,), q.detach())                  # linear: its second derivative is the turn itself
    assert torch.equal(twice, a.detach())
    (only,) = torch.autograd.grad(fast_rcnn.rope_axes(q, k, pos, plan)[1], (k,), db)
    assert torch.equal(only, dk.detach())
    z = torch.randn((12, 37), generator=g)
    y = torch.randint(0, 37, (12,), generator=g)
    y[3] = -1
    w, wh = torch.randn(12, generator=g), torch.randn(12, generator=g)
    Z = z.cuda().requires_grad_(True)
    r = fast_rcnn.class_logprobs(Z, y, top=4)
    assert not r.top_logp.requires_grad and r.top_index.dtype == torch.int64
    (dz,) = torch.autograd.grad((r.logp, r.entropy), (Z,), (w.cuda(), wh.cuda()), retain_graph=True)
    want = _logp64(z, y, 4, w, wh)
    _close(dz, want["dz"], "dz")
    f = lambda x: (_logp64(x, y, 0)["logp"][0] * w.double()).sum() + (_logp64(x, y, 0)["entropy"][0] * wh.double()).sum()    # noqa: E731
    d = torch.randn(z.shape, generator=g, dtype=torch.float64)
    # the quotient's own error: below 1e-6 of the sum of magnitudes, as above
    assert abs(_slope(f, (z.double(),), (d,)) - float((dz.cpu().double() * d).sum())) <= float((want["dz"][1] * d.abs()).sum()) + 1e-6 * float((want["dz"][0] * d).abs().sum())
    (one,) = torch.autograd.grad(r.entropy, (Z,), wh.cuda())
    _close(one, _logp64(z, y, 0, torch.zeros(12), wh)["dz"], "dz of the entropy alone")


@pytest.mark.gpu
def test_head_together():
    """Boxes of two frames turned by their positions, related to each other where they overlap, classified, and a training loss
    back through all of it: the chain's gradients are the operators' own, one after the other, and its loss and its gradient agree
    with the definitions in 64 bits.  Every stage is exact to 2^-15 of the magnitudes that it sums (checked above: at most 64 values
    a product, 60 keys, 30 classes); through three stages forward and back, each norm-preserving up to a factor of 4 (logits by a
    projection of norm below 4), the loss's slope along a direction stays within 2^-15 x 6 x 4^3 < 2^-6 of its magnitudes."""
    from tools import workloads as wl
    from vision_amd import fast_rcnn, ops
    B, N, H, D, C = 2, 60, 4, 64, 30
    boxes = torch.stack([torch.from_numpy(wl.random_boxes(50 + i, N)) for i in range(B)])
    pos = torch.stack([torch.tensor([5.0, 6.0])[:, None].expand(B, N), (boxes[..., 1] + boxes[..., 3]) * 10, (boxes[..., 0] + boxes[..., 2]) * 10], 2)
    counts = torch.tensor([N, 41]).int()
    over = torch.stack([ops.iou_pairwise(b.cuda(), b.cuda()) > 0.05 for b in boxes])
    g = _gen(41)
    q, k, v = (torch.randn((B, N, H, D), generator=g) for _ in range(3))
    proj = torch.randn((H * D, C), generator=g) / math.sqrt(H * D)
    y = torch.randint(0, C, (B, N), generator=g)
    y[1, 41:] = -1                               # padded rows carry no label
    plan = ops.rope_plan((8, 12, 12))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    a, b = fast_rcnn.rope_axes(leaves[0], leaves[1], pos, plan)
    out = fast_rcnn.roi_attention(a, b, leaves[2], counts, counts, over)
    z = out.reshape(B * N, H * D) @ proj.cuda()
    r = fast_rcnn.class_logprobs(z, y.reshape(-1), top=3)
    loss = -r.logp.sum() / int((y >= 0).sum()) - 0.01 * r.entropy.sum()
    grads = torch.autograd.grad(loss, leaves)
    # the same by hand
    ones = torch.full((B * N,), -1.0 / int((y >= 0).sum()), device="cuda")
    logp, h, norm, best, index = ops.class_logprobs(z.detach(), y.reshape(-1), 3)
    assert torch.equal(logp, r.logp.detach()) and torch.equal(index, r.top_index)
    dz = ops.class_logprobs_backward(ones, torch.full_like(ones, -0.01), z.detach(), y.reshape(-1), norm, h)
    dout = (dz @ proj.cuda().T).view(B, N, H, D)
    o, lse = ops.roi_attention(a.detach(), b.detach(), leaves[2].detach(), counts, counts, over)
    da, db, dv = ops.roi_attention_backward(dout, a.detach(), b.detach(), leaves[2].detach(), o, lse, counts, counts, over)
    dq, dk = ops.rope_axes(da, pos.cuda(), plan, k=db, inverse=True)
    assert all(torch.equal(x, w) for x, w in zip(grads, (dq, dk, dv)))
    # and in 64 bits
    mask = over.cpu()

    def f(Q, K, V):
        ang = pos.double()[..., plan.axis.cpu().long()] * plan.turns.cpu() * 2 * math.pi
        c, s = torch.cos(ang)[:, :, None], torch.sin(ang)[:, :, None]
        turn = lambda t: torch.cat([t[..., :32] * c - t[..., 32:] * s, t[..., :32] * s + t[..., 32:] * c], -1)   # noqa: E731
        w = _attn64(turn(Q), turn(K), V, counts, counts, mask, None)["out"][0].reshape(B * N, H * D) @ proj.double()
        lp = _logp64(w, y.reshape(-1), 0)
        return -lp["logp"][0].sum() / int((y >= 0).sum()) - 0.01 * lp["entropy"][0].sum()
    xs = [t.double() for t in (q, k, v)]
    exact = float(f(*xs))
    assert abs(float(loss.detach()) - exact) <= 2.0 ** -6 * abs(exact)
    for i in range(3):
        d = [torch.zeros_like(t) for t in xs]
        d[i] = torch.randn(xs[i].shape, generator=g, dtype=torch.float64)
        mine = grads[i].cpu().double() * d[i]
        assert abs(_slope(f, xs, d) - float(mine.sum())) <= 2.0 ** -6 * float(mine.abs().sum()), i


# ------------------------------------------------------------------ refusals
def test_refusals_of_the_library():
    """On the host, before any launch."""
    import ctypes as C
    from vision_amd import _abi
    lib = _abi.load()

    def shape(**kw):
        s = _abi.AttnShape(2, 8, 8, 4, 2, 64)
        for t, heads in (("q", 4), ("k", 2), ("v", 2), ("g", 4)):
            for a, n in (("batch", 8 * heads * 64), ("row", heads * 64), ("head", 64)):
                setattr(s, f"{t}_stride_{a}", n)
        s.scale, s.dtype = 0.125, _abi.BF16
        for a, b in kw.items():
            setattr(s, a, b)
        return s
    p = C.c_void_p(4096)                         # never touched: every call below ends before a launch

    def fwd(s, q=p, ws=None, n=0):
        return lib.dg_roi_attn_fwd(s, q, p, p, None, None, None, p, p, None, ws, n, None)
    for kw, word in ((dict(d=12), "head size"), (dict(d=136), "head size"), (dict(q_heads=3), "multiple of k_heads"), (dict(k_heads=0), "multiple of k_heads"),
                     (dict(dtype=_abi.F16), "type"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                     (dict(batch=-1), "negative"), (dict(nq=1 << 40), "2^28"), (dict(masks=3), "masks"), (dict(masks=1), "null"),
                     (dict(q_stride_row=33), "16 bytes"), (dict(k_stride_row=-64), "16 bytes"), (dict(v_stride_row=1 << 23), "2^22")):
        assert fwd(shape(**kw)) == _abi.EINVAL, kw
        assert word in _abi.last_error(), (kw, _abi.last_error())
    assert fwd(shape(), q=C.c_void_p(4098)) == _abi.EINVAL and "16 bytes" in _abi.last_error()
    assert fwd(shape(), q=None) == _abi.EINVAL and "null" in _abi.last_error()
    long = shape(nk=100000)
    need = lib.dg_roi_attn_workspace_bytes(long, 0)
    assert need > 0 and fwd(long, ws=p, n=need - 1) == _abi.ENOMEM and "workspace" in _abi.last_error()
    assert fwd(shape(batch=0)) == _abi.OK and fwd(shape(nq=0)) == _abi.OK
    assert lib.dg_roi_attn_workspace_bytes(shape(d=12), 1) == 0
    assert lib.dg_roi_attn_bwd(shape(), p, p, p, p, p, p, None, None, None, None, p, p, None, p, 1 << 30, None) == _abi.EINVAL     # dk without dv

    def rope(**kw):
        s = _abi.RopeShape(1, 4, 2, 1, 64, 16, 2)
        s.pos_dtype = _abi.F32
        for a, b in kw.items():
            setattr(s, a, b)
        return lib.dg_rope_axes(s, p, p, p, p, p, 0, p, p, None)
    for kw, word in ((dict(pairs=33), "do not fit"), (dict(pairs=0), "do not fit"), (dict(d=7), "even"), (dict(axes=17), "axes"), (dict(pairing=2), "pairing"),
                     (dict(dtype=_abi.F64), "type"), (dict(pos_dtype=_abi.BF16), "positions"), (dict(n=-1), "token"), (dict(q_heads=0, k_heads=0), "head count")):
        assert rope(**kw) == _abi.EINVAL, kw
        assert word in _abi.last_error(), (kw, _abi.last_error())
    assert rope(n=0) == _abi.OK

    def logp(n=4, c=10, top=2, dtype=_abi.F32, z=p, y=p, logp_=p, ws=None, nbytes=0):
        return lib.dg_class_logprobs(z, dtype, y, n, c, c, top, logp_, p, p, p, p, p, ws, nbytes, None)
    for kw, word in ((dict(top=11), "alternatives"), (dict(c=100, top=33), "alternatives"), (dict(c=0, top=0), "classes"), (dict(dtype=_abi.F64), "type"),
                     (dict(n=-1), "row count"), (dict(z=None), "null"), (dict(logp_=None), "null"), (dict(z=C.c_void_p(4097)), "aligned")):
        assert logp(**kw) == _abi.EINVAL, kw
        assert word in _abi.last_error(), (kw, _abi.last_error())
    need = lib.dg_class_logprobs_workspace_bytes(1, 131072, 8)
    assert need > 0 and logp(n=1, c=131072, top=8, ws=p, nbytes=need - 1) == _abi.ENOMEM
    assert logp(n=0) == _abi.OK and logp(n=0, y=None) == _abi.OK
    assert lib.dg_class_logprobs_bwd(p, _abi.F32, None, 4, 10, 10, p, p, p, None, p, None) == _abi.EINVAL     # a gradient of logp without labels


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful on a host without a GPU")
def test_no_cpu_fallback_of_the_head():
    from vision_amd import _abi, fast_rcnn, ops
    t = torch.zeros((1, 4, 2, 32))
    for call in (lambda: ops.roi_attention(t, t, t), lambda: fast_rcnn.roi_attention(t, t, t), lambda: ops.rope_plan((8, 8)),
                 lambda: ops.class_logprobs(torch.zeros((2, 5)), torch.zeros(2, dtype=torch.int64)), lambda: fast_rcnn.class_logprobs(torch.zeros((2, 5)))):
        with pytest.raises(_abi.DetGeomError):
            call()


@pytest.mark.gpu
def test_refusals_of_the_front_end():
    from vision_amd import fast_rcnn, ops
    t = torch.zeros((2, 6, 4, 32), device="cuda")
    k = torch.zeros((2, 9, 2, 32), device="cuda")
    out, lse = ops.roi_attention(t, k, k)
    bad = [
        lambda: ops.roi_attention(t[0], k, k), lambda: ops.roi_attention(t, k, k[:, :5]), lambda: ops.roi_attention(t, k[:1], k[:1]),
        lambda: ops.roi_attention(t.half(), k.half(), k.half()), lambda: ops.roi_attention(t, k.bfloat16(), k), lambda: ops.roi_attention(t[:, :, :3], k, k),
        lambda: ops.roi_attention(t[..., :12], k[..., :12], k[..., :12]), lambda: ops.roi_attention(t, k, k, scale=0.0), lambda: ops.roi_attention(t, k, k, scale=-1.0),
        lambda: ops.roi_attention(t, k, k, q_counts=torch.zeros(3)), lambda: ops.roi_attention(t, k, k, k_counts=torch.zeros((2, 1))),
        lambda: ops.roi_attention(t, k, k, mask=torch.zeros((2, 6, 9))), lambda: ops.roi_attention(t, k, k, mask=torch.zeros((3, 6, 9), dtype=torch.bool)),
        lambda: ops.roi_attention(t, k, k, mask=torch.zeros((6, 8), dtype=torch.bool)),
        lambda: ops.roi_attention_backward(t[:, :5], t, k, k, out, lse), lambda: ops.roi_attention_backward(t, t, k, k, out, lse.transpose(1, 2)),
        lambda: ops.roi_attention_backward(t.bfloat16(), t, k, k, out, lse),
        lambda: ops.rope_plan(()), lambda: ops.rope_plan((0, 0)), lambda: ops.rope_plan((8, -1)), lambda: ops.rope_plan((8,), theta=0.0),
        lambda: ops.rope_plan((8,), ladder="x"), lambda: ops.rope_plan((8,), pairing="x"),
        lambda: ops.rope_axes(t, torch.zeros((2, 6, 3)), ops.rope_plan((8, 8))), lambda: ops.rope_axes(t, torch.zeros((2, 6, 2)), ops.rope_plan((8, 9))),
        lambda: ops.rope_axes(t, torch.zeros((2, 6, 2)), ops.rope_plan((8, 8)), k=k), lambda: ops.rope_axes(t.double(), torch.zeros((2, 6, 2)), ops.rope_plan((8, 8))),
        lambda: ops.rope_axes(t, torch.zeros((2, 6, 2), device="cuda", requires_grad=True), ops.rope_plan((8, 8))),
        lambda: fast_rcnn.rope_axes(t, t, torch.zeros((2, 6, 2), requires_grad=True), ops.rope_plan((8, 8))),
        lambda: ops.class_logprobs(t, torch.zeros(2)), lambda: ops.class_logprobs(t[0, 0], torch.zeros(3, dtype=torch.int64)),
        lambda: ops.class_logprobs(t[0, 0], torch.zeros(4, dtype=torch.int64), top=33), lambda: ops.class_logprobs(t[0, 0], torch.zeros(4, dtype=torch.int64), top=-1),
        lambda: ops.class_logprobs(t[0, 0].double()), lambda: ops.class_logprobs_backward(None, torch.zeros(3), t[0, 0], None, torch.zeros((4, 2)), torch.zeros(4)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)
    # nothing to do is no error
    assert ops.roi_attention(t[:0], k[:0], k[:0])[0].shape == (0, 6, 4, 32)
    o, s = ops.roi_attention(t, k[:, :0], k[:, :0])
    assert float(o.abs().max()) == 0.0 and bool(torch.isinf(s).all())
    dq, dk, dv = ops.roi_attention_backward(t, t, k[:, :0], k[:, :0], o, s)
    assert float(dq.abs().max()) == 0.0 and dk.shape == (2, 0, 2, 32)
    o, s = ops.roi_attention(t[:, :0], k, k)
    dq, dk, dv = ops.roi_attention_backward(t[:, :0], t[:, :0], k, k, o, s)
    assert dq.shape == (2, 0, 4, 32) and float(dk.abs().max()) == 0.0 and float(dv.abs().max()) == 0.0
    assert ops.rope_axes(t[:, :0], torch.zeros((2, 0, 2)), ops.rope_plan((8, 8))).shape == (2, 0, 4, 32)
    assert ops.class_logprobs(t[0, 0, :0], torch.zeros(0, dtype=torch.int64), 3)[4].shape == (0, 3)
    assert ops.class_logprobs_backward(torch.zeros(0), None, t[0, 0, :0], torch.zeros(0, dtype=torch.int64), torch.zeros((0, 2)), torch.zeros(0)).shape == (0, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_class_logprobs_large_gradient(dtype):
    """2^24 scores and more, dense, rows apart, and a gradient that starts off its 16 bytes."""
    import ctypes as C
    from vision_amd import _abi, ops
    n, c = 520, 32771
    rng = torch.Generator(device="cuda").manual_seed(9)
    z = (torch.randn((n, c), generator=rng, device="cuda") * 3).to(dtype)
    y = torch.randint(0, c, (n,), generator=rng, device="cuda")
    g, gh = torch.randn((n,), generator=rng, device="cuda"), torch.randn((n,), generator=rng, device="cuda")
    want = _logp64(z, y, 2, g, gh)
    cpu = lambda t: tuple(x.cpu() for x in t)      # noqa: E731
    logp, entropy, norm, best, index = ops.class_logprobs(z, y, 2)
    _close(logp, cpu(want["logp"]), "logp")
    _close(entropy, cpu(want["entropy"]), "entropy")
    assert torch.equal(index, want["index"])
    dz = ops.class_logprobs_backward(g, gh, z, y, norm, entropy)
    _close(dz, cpu(want["dz"]), "dz")
    wide = torch.zeros((n, c + 5), dtype=dtype, device="cuda")
    wide[:, 2:c + 2] = z
    assert torch.equal(ops.class_logprobs_backward(g, gh, wide[:, 2:c + 2], y, norm, entropy), dz)
    m = 40                                        # the first rows once more through the C ABI, one value off
    off = torch.full((m * c + 2,), 7.0, dtype=dtype, device="cuda")
    rc = _abi.load().dg_class_logprobs_bwd(z.data_ptr(), _abi.TYPES[dtype], y.data_ptr(), m, c, c, norm.data_ptr(), entropy.data_ptr(), g.data_ptr(), gh.data_ptr(),
                                           off[1:].data_ptr(), C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == _abi.OK
    torch.cuda.synchronize()
    assert torch.equal(off[1:-1].view(m, c), dz[:m]) and float(off[0]) == 7.0 and float(off[-1]) == 7.0


@pytest.mark.gpu
def test_class_logprobs_status_and_bad_rows():
    """A label outside the classes is told by the status word and by NaN; a NaN or +inf makes its row NaN and no other."""
    import ctypes as C
    from vision_amd import _abi, ops
    for c in (10, 700):
        z = torch.randn((6, c), generator=_gen(3)).cuda()
        z[1, 4], z[2, 5] = math.nan, math.inf
        y = torch.tensor([0, 1, 2, -5, c, 3]).cuda()
        logp, entropy, norm, best, index = ops.class_logprobs(z, y, 3)
        assert torch.isnan(logp[[1, 2, 4]]).all() and torch.isfinite(logp[[0, 3, 5]]).all() and float(logp[3]) == 0.0
        assert torch.isnan(entropy[[1, 2]]).all() and torch.isfinite(entropy[[0, 3, 4, 5]]).all()
        assert torch.equal(index[1], torch.sort(torch.where(torch.isnan(z[1]), -math.inf, z[1]), descending=True, stable=True).indices[:3])     # NaN last
        dz = ops.class_logprobs_backward(torch.ones(6), torch.ones(6), z, y, norm, entropy)
        assert torch.isnan(dz[[1, 2, 4]]).all() and torch.isfinite(dz[[0, 3, 5]]).all()
        out = [torch.empty(6, device="cuda"), torch.empty(6, device="cuda"), torch.empty((6, 2), device="cuda")]
        for labels, bit in ((y, 1), (y.clamp(max=c - 1), 0)):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            rc = _abi.load().dg_class_logprobs(z.data_ptr(), _abi.F32, labels.data_ptr(), 6, c, c, 0, *(t.data_ptr() for t in out), None, None, status.data_ptr(), None, 0,
                                               C.c_void_p(torch.cuda.current_stream().cuda_stream))
            assert rc == _abi.OK and int(status.item()) == bit


@pytest.mark.gpu
@pytest.mark.parametrize("n,c,first", [(3, 4000, 2500), (300, 20000, 9000)])
def test_class_logprobs_best_behind_nan(n, c, first):
    """The classes of a row that begins with more NaN than are looked at in one turn are still ranked before the NaN."""
    from vision_amd import ops
    z = torch.randn(n, c, generator=_gen(61))
    z[:, :first] = math.nan
    z[:, first::7] = -math.inf
    index = ops.class_logprobs(_dev(z), None, 5)[4].cpu()
    assert torch.equal(index, torch.sort(torch.where(torch.isnan(z), -math.inf, z), dim=1, descending=True, stable=True).indices[:, :5])
    z[:, first:] = -math.inf
    z[:, first + 100:] = math.nan
    index = ops.class_logprobs(_dev(z), None, 5)[4].cpu()
    assert torch.equal(index, first + torch.arange(5).expand(n, 5))


def test_attention_refuses_what_no_launch_holds():
    """On the host: a launch has fewer than 2^32 threads, and a scale times log2 e has to be a 32-bit number."""
    from vision_amd import _abi
    lib = _abi.load()
    for kw, word in ((dict(scale=2.5e38), "scale"), (dict(batch=1 << 23), "too many tiles"), (dict(batch=1 << 20, nq=2000), "too many tiles"),
                     (dict(batch=1 << 20, nk=2000), "too many tiles")):
        s = _abi.AttnShape(2, 8, 8, 4, 2, 64)
        s.scale, s.dtype = 0.125, _abi.BF16
        for a, b in kw.items():
            setattr(s, a, b)
        assert lib.dg_roi_attn_workspace_bytes(s, 1) == 0 and word in _abi.last_error(), (kw, _abi.last_error())


@pytest.mark.gpu
def test_more_blocks_than_one_axis_of_a_launch_holds():
    """2^32 threads and more: the tokens and rows behind them are computed as those before."""
    from vision_amd import ops
    n, d = (1 << 28) + 37, 2                     # 16 tokens a block
    plan = ops.rope_plan((1,), device="cuda")
    q = torch.empty(1, n, 1, d, dtype=torch.bfloat16, device="cuda")
    q[..., 0], q[..., 1] = 1.0, -2.0
    pos = torch.zeros(n, 1, device="cuda")
    pos[:, 0] = torch.arange(n, device="cuda") % 1021
    out = ops.rope_axes(q, pos, plan)
    for a in (0, (1 << 28) - 50, n - 60):
        assert torch.equal(out[:, a:a + 60], ops.rope_axes(q[:, a:a + 60], pos[a:a + 60], plan))
    del q, pos, out
    for c, top in ((300, 1), (600, 0)):          # 4 rows a block
        n = (1 << 26) + 9
        z = torch.randn(1, c, generator=_gen(62)).bfloat16().cuda()
        one = ops.class_logprobs(z, torch.full((1,), 7, device="cuda"), top)
        y = torch.full((n,), 7, dtype=torch.int64, device="cuda")
        y[-1] = -1
        many = ops.class_logprobs(z.expand(n, c), y, top)
        assert bool((many[0][:-1] == one[0]).all()) and float(many[0][-1]) == 0.0
        assert all(bool((a == b).all()) for a, b in zip(many[1:], one[1:]))


@pytest.mark.gpu
def test_roi_attention_empty_views():
    """No rows or no keys, cut from tensors whose strides are no multiples of 16 bytes."""
    from vision_amd import ops
    x = torch.randn(3, 5, 2, 13, dtype=torch.float32, device="cuda")
    full, none = x[..., 5:13], x[:, :0, :, 5:13]
    out, lse = ops.roi_attention(full, none, none)
    assert out.shape == full.shape and bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, dv = ops.roi_attention_backward(full, full, none, none, out, lse)
    assert bool((dq == 0).all()) and dk.shape == dv.shape == none.shape
    out, lse = ops.roi_attention(none, full, full)
    assert out.shape == none.shape and lse.shape == (3, 2, 0)
    dq, dk, dv = ops.roi_attention_backward(none, none, full, full, out, lse)
    assert dq.shape == none.shape and bool((dk == 0).all()) and bool((dv == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_roi_attention_largest_values_behind_mask(dtype, D):
    """Keys and rows that a mask hides from all, filled with a type's largest and lowest value: as if they held zeros."""
    from vision_amd import ops
    B, N, M, H = 2, 70, 90, 2
    q, k, v, do = _attn_inputs(71, B, N, M, H, H, D, dtype)
    mask = torch.rand((B, N, M), generator=_gen(72)) < 0.5
    keys, rows = [0, 17, 63, 89], [5, 31, 69]
    mask[:, :, keys] = False
    mask[:, rows] = False
    got = []
    for fill in ((0.0, 0.0), (torch.finfo(dtype).max, torch.finfo(dtype).min)):
        Q, K, V, G = q.clone(), k.clone(), v.clone(), do.clone()
        K[:, keys, 0], K[:, keys, 1], V[:, keys, 0], V[:, keys, 1] = fill[0], fill[1], fill[1], fill[0]
        Q[:, rows, 0], Q[:, rows, 1], G[:, rows, 0], G[:, rows, 1] = fill[0], fill[1], fill[1], fill[0]
        Q, K, V, G, m = map(_dev, (Q, K, V, G, mask))
        out, lse = ops.roi_attention(Q, K, V, mask=m)
        got.append((out, lse, *ops.roi_attention_backward(G, Q, K, V, out, lse, mask=m)))
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), *got):
        assert torch.equal(a, b), name


@pytest.mark.gpu
def test_roi_attention_keeps_the_bits_of_float32():
    """Values that differ in their last bits only: products of 32-bit operands in three parts keep them.  v is 1 + j 2^-20 for key j and
    one key is seen by each row, so that out is that v exactly; with two keys of equal score it is their mean, rounded once or twice."""
    from vision_amd import ops
    n, d = 96, 64
    q = torch.zeros(1, n, 1, d, device="cuda")
    v = (1.0 + torch.arange(n, dtype=torch.float32)[:, None] * 2.0 ** -20 + torch.arange(d) * 2.0 ** -23).view(1, n, 1, d).cuda()
    eye = torch.eye(n, dtype=torch.bool, device="cuda")
    out, _ = ops.roi_attention(q, q, v, mask=eye)
    assert torch.equal(out, v)
    out, _ = ops.roi_attention(q, q, v, mask=eye | eye.roll(1, 1))
    want = (v.double() + v.double().roll(-1, 1)) / 2
    assert float((out.double() - want).abs().max()) <= 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,D", [(1, 64), (2, 32), (3, 64), (5, 128), (7, 64)])
def test_roi_attention_gradient_of_few_keys(n, D, masked):
    """n keys of equal score: p is 1 / n (1 before it is divided, so without a rounding to bf16), the sum of ds over them 0, and dq, the
    sum of ds k over equal k, 0 too; ds is what is left of dp - delta.  delta comes from out and its rest, 2^-16 of |do| |out| apart, ds
    goes into its products as two parts, 2^-16 of it, and 32-bit sums of D terms add D 2^-24 of their magnitudes."""
    from vision_amd import fast_rcnn, ops
    N, u2 = 150, 2.0 ** -16
    q, k, v, do = (t.double() for t in _attn_inputs(81, 2, N, 40 if masked else n, 2, 1, D, torch.bfloat16))
    k[:] = k[:, :1]
    mask = None
    if masked:
        mask = torch.zeros((2, N, 40), dtype=torch.bool)
        mask[:, :, torch.randperm(40, generator=_gen(82))[:n]] = True
    seen = slice(None) if mask is None else mask[0, 0].nonzero()[:, 0]
    V = v[:, seen, 0]                             # (2, n, D)
    o = V.mean(1)[:, None, None]                  # (2, 1, 1, D)
    dp = torch.einsum("bihd,bjd->bihj", do, V)
    ds = (dp - (do * o).sum(-1, keepdim=True)) / n
    mag = torch.einsum("bihd,bjd->bihj", do.abs(), V.abs()) + (do.abs() * o.abs()).sum(-1, keepdim=True)
    eds = ds.abs() * (u2 + 16 * E32) + ((do.abs() * o.abs()).sum(-1, keepdim=True) * u2 + (D + 8) * E32 * mag) / n + 8 * E32 * dp.abs() / n
    sc = D ** -0.5
    dk = torch.einsum("bihj,bihd->bjd", ds, q) * sc
    edk = torch.einsum("bihj,bihd->bjd", eds + 2 * N * E32 * ds.abs(), q.abs()) * sc + 2.0 ** -8 * dk.abs()
    edq = (eds + n * E32 * ds.abs()).sum(-1, keepdim=True) * k[:, :1, :1].abs() * sc
    Q, K, W, G = (t.to(torch.bfloat16).cuda() for t in (q, k, v, do))
    out, lse, rest = ops.roi_attention(Q, K, W, mask=_dev(mask), rest=True)
    a = ops.roi_attention_backward(G, Q, K, W, out, lse, mask=_dev(mask), rest=rest)
    Q, K, W = (t.requires_grad_(True) for t in (Q, K, W))
    b = torch.autograd.grad(fast_rcnn.roi_attention(Q, K, W, mask=_dev(mask)), (Q, K, W), G)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    _close(a[0], (torch.zeros_like(q), edq), "dq")
    _close(a[1][:, seen, 0], (dk, edk), "dk")


@pytest.mark.gpu
def test_roi_attention_rest():
    """out + rest is the output in 16 bits, also where splits are joined; rows that see nothing have none; float32 has none."""
    from vision_amd import ops
    for case in ((2, 100, 70, 4, 2, 64, True, None), (1, 3, 5000, 2, 1, 128, True, None), (1, 70, 3000, 2, 2, 40, False, "shared")):
        q, k, v, _ = _attn_inputs(91, *case[:6], torch.bfloat16)
        qc, kc, m = _attn_masks(case, 91)
        one = ops.roi_attention(*map(_dev, (q, k, v, qc, kc, m)), rest=True)
        two = ops.roi_attention(*map(_dev, (q, k, v, qc, kc, m)))
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1]) and len(two) == 2
        out, rest = one[0].cpu().double(), one[2].cpu().double()
        assert bool((rest.abs() <= 2.0 ** -8 * out.abs()).all()) and float(rest.abs().max()) > 0.0
        if qc is not None:
            assert all(float(rest[b, int(qc[b]):].abs().sum()) == 0.0 for b in range(case[0]))
        want = _attn64(q, k, v, qc, kc, m, None)["out"]
        p_only = want[1] - 2.0 ** -8 * want[0].abs() + 2.0 ** -16 * want[0].abs()       # without the rounding of out
        _close(torch.from_numpy((out + rest).numpy()), (want[0], p_only), "out + rest")
    q = torch.randn(1, 4, 1, 8, device="cuda")
    assert ops.roi_attention(q, q, q, rest=True)[2] is None
    with pytest.raises(ValueError, match="rest"):
        ops.roi_attention_backward(q, q, q, q, *ops.roi_attention(q, q, q), rest=q)


@pytest.mark.gpu
def test_gradients_of_gradients_and_of_broadcast_inputs():
    """A second derivative that is not there is refused, not wrong; a key set expanded over the batch gets the sum of its gradients; a
    gradient that comes expanded (of a sum) is taken like a dense one."""
    from vision_amd import fast_rcnn
    g = _gen(95)
    q = torch.randn((3, 40, 2, 32), generator=g).cuda().requires_grad_(True)
    k, v = (torch.randn((1, 50, 2, 32), generator=g).cuda().requires_grad_(True) for _ in range(2))
    out = fast_rcnn.roi_attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1))
    wide = [t.detach().expand(3, -1, -1, -1).contiguous().requires_grad_(True) for t in (k, v)]
    ref = fast_rcnn.roi_attention(q, *wide)
    assert torch.equal(out, ref)
    a = torch.autograd.grad(out.sum(), (q, k, v))
    b = torch.autograd.grad(ref, (q, *wide), torch.ones_like(ref))
    assert torch.equal(a[0], b[0])
    for x, y in zip(a[1:], b[1:]):                # a sum of three terms of 32 bits, in any order
        assert bool(((x - y.double().sum(0, keepdim=True)).abs() <= 4 * E32 * y.abs().sum(0, keepdim=True)).all())
    z = torch.randn((6, 9), generator=g).cuda().requires_grad_(True)
    r = fast_rcnn.class_logprobs(z, torch.arange(6), 2)
    for y, x in ((fast_rcnn.roi_attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1)), q), (r.logp, z)):
        w = torch.ones_like(y).requires_grad_(True)
        (dx,) = torch.autograd.grad(y, (x,), w, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            dx.sum().backward()
