"""The RoI head's operators against their definitions in 64 bits: attention over an image's boxes (forward, backward), rotary
positions over several axes, log probabilities of labels.

Tolerances.  One rounding to a type moves a value by at most half a step, u = 2^-8 of it in bf16, 2^-11 in fp16, 2^-24 in fp32.
Attention in bf16: p (and ds) is rounded once as an operand, the result once at the end, so an output element is off by at most
u sum |p_ij v_j| + u |o_i|, and the sum itself is held in 32 bits; delta is formed from the rounded out (u |do| |out| per row).
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


LOGP_CASES = [(1, 1, 1), (1, 2, 2), (5, 21, 3), (300, 81, 5), (257, 33, 32), (64, 512, 8), (33, 513, 8), (7, 1000, 32), (40, 4096, 4), (3, 4097, 8),
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
